"""GPU tests of the 8-bit key/value cache: kv8_append and kv8_read give exactly the codes, scales and
values of the 64-bit implementation (kv8_ref.py); attn_fwd_kv8 stays within the bound that is derived
there for its arithmetic."""
import numpy as np
import pytest
import torch

import b200lab
import kv8_ref
from helpers import assert_close, to_np

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prefix(v):
    return _ints(np.concatenate([[0], np.cumsum(v)]).tolist())


def _normal(shape, seed, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


class Setup:
    """A cache with random contents, its blocks in random order, on the GPU and as the reference's."""

    def __init__(self, lens, Hkv, D, P, seed=0, spare=2, exps=(-8, -4), garbage=False):
        rng = np.random.default_rng(seed)
        used = [-(-n // P) for n in lens]
        self.n_blocks, self.width = sum(used) + spare, max(1, max(used))
        order = rng.permutation(self.n_blocks).tolist()
        self.table, at = [], 0
        for u in used:
            self.table.append(order[at:at + u] + [self.n_blocks + 7] * (self.width - u))  # not to be read
            at += u
        shape = (self.n_blocks, Hkv, P, D)
        self.codes = []
        for _ in range(2):
            x = np.clip(rng.standard_normal(shape) * 80, -448, 448).astype(np.float32)
            c = torch.from_numpy(x).to(E4M3).view(torch.uint8).numpy().copy()
            if garbage:  # NaN wherever no token lies
                own = np.zeros((self.n_blocks, P), dtype=bool)
                for b, n in enumerate(lens):
                    for i, blk in enumerate(self.table[b][:used[b]]):
                        own[blk, :min(P, n - i * P)] = True
                c[~np.broadcast_to(own[:, None, :, None], shape)] = 0x7f
            self.codes.append(c)
        self.scales = [np.exp2(rng.integers(exps[0], exps[1] + 1, shape[:2])).astype(np.float32) for _ in range(2)]
        self.lens, self.P, self.Hkv, self.D = list(lens), P, Hkv, D
        self.k, self.v = (torch.from_numpy(c).cuda().view(E4M3) for c in self.codes)
        self.ks, self.vs = (torch.from_numpy(s).cuda() for s in self.scales)
        self.t, self.l = _ints(self.table), _ints(self.lens)
        self.rk, self.rv = (kv8_ref.Cache(c, s) for c, s in zip(self.codes, self.scales))

    @property
    def cache(self):
        return self.k, self.v, self.ks, self.vs, self.t

    def same(self):
        """The GPU's cache is the reference's: every code's value, every scale."""
        for x, s, r in ((self.k, self.ks, self.rk), (self.v, self.vs, self.rv)):
            assert np.array_equal(s.double().cpu().numpy(), r.scales)
            assert np.array_equal(kv8_ref.TABLE[x.view(torch.uint8).cpu().numpy()], r.values, equal_nan=True)


def _check_attend(s, q, new, causal=True, gate=None, scale=None, total=None, **kw):
    scale = 1 / np.sqrt(s.D) if scale is None else scale
    one = all(n == 1 for n in new) and kw.pop("plain_step", True)
    o = b200lab.attn_fwd_kv8(q, *s.cache, s.l, cu_seqlens_q=None if one else _prefix(new), max_seqlen_q=max(new + [1]),
                             gate=gate, scale=scale, causal=causal, **kw)
    assert b200lab.device_status() == b200lab.OK
    n = sum(new)
    ref, bound = kv8_ref.attend(q[:n].double().cpu().numpy(), s.rk, s.rv, s.table, s.lens, new, scale, causal,
                                None if gate is None else gate[:n].double().cpu().numpy(), UNIT[q.dtype])
    got = o[:n].double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    over = np.abs(got - ref)[fine] - bound[fine]
    assert over.size == 0 or over.max() <= 0, f"{over.max():.3e} over its bound, error {np.abs(got - ref)[fine].max():.3e}"
    return o


# ---- writing ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,P,Hkv", [(64, 16, 3), (128, 64, 2), (256, 128, 1), (128, 32, 1), (256, 16, 2)])
def test_append_exact(cuda, dtype, D, P, Hkv):
    """Sequences of every phase against the blocks, one to some hundred new tokens; twice in a row."""
    lens, new = [1, P, P + 1, 2 * P + 5, 3 * P, 7, 300], [1, P, P + 1, 3, 2 * P, 0, 150]
    s = Setup(lens, Hkv, D, P, seed=D + P)
    total = sum(new)
    k, v = _normal((total, Hkv, D), 1, dtype, 3.0), _normal((total, Hkv, D), 2, dtype)
    v[::7] *= 40  # some tokens need a larger scale than their block has
    b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, s.l, cu_seqlens=_prefix(new), max_seqlen=max(new))
    assert b200lab.device_status() == b200lab.OK
    s.rk.append(k.double().numpy(), s.table, lens, new)
    s.rv.append(v.double().numpy(), s.table, lens, new)
    s.same()


@pytest.mark.parametrize("D,P", [(128, 64), (64, 16), (256, 32)])
def test_append_steps_grow_the_scale(cuda, D, P):
    """One token at a time through several blocks, of magnitudes that rise and fall by powers of ten: the
    codes of a begun block are rounded to each larger scale.  A padding entry writes nothing."""
    steps, B, Hkv = P + 9, 3, 2
    s = Setup([steps + 5, 0, steps], Hkv, D, P, seed=5)
    for i in range(steps):
        lens = [6 + i, 0, i + 1]
        k = _normal((B, Hkv, D), 10 + i, torch.bfloat16, 10.0 ** ((i * 7) % 9 - 4))
        v = _normal((B, Hkv, D), 500 + i, torch.bfloat16, 10.0 ** (i % 5))
        b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, _ints(lens))
        live = [0, 2]
        for r, x in ((s.rk, k), (s.rv, v)):
            r.append(x.double().numpy()[live], [s.table[0], s.table[2]], [lens[0], lens[2]], [1, 1])
    assert b200lab.device_status() == b200lab.OK
    s.same()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append_special_values(cuda, dtype):
    """Zeros, subnormals, the type's largest and smallest values, infinities and NaN."""
    P, D = 16, 64
    big = torch.finfo(dtype).max
    rows = [torch.zeros(D), torch.full((D,), torch.finfo(dtype).smallest_normal), torch.full((D,), big),
            torch.full((D,), float("nan")), torch.tensor([float("inf"), -float("inf"), 1.0, -2.0] * (D // 4)),
            torch.tensor([float("nan"), 3.5, -0.0, 1e-3] * (D // 4)), torch.full((D,), 448.0), torch.full((D,), 449.0),
            torch.full((D,), torch.finfo(dtype).tiny / 4)]
    x = torch.stack(rows)[:, None].to(dtype)
    lens = [P * i + 1 for i in range(1, len(rows) + 1)]
    for new in ([1] * len(rows), None):
        s = Setup(lens if new else [len(rows)], 1, D, P, seed=3)
        n = new or [len(rows)]
        b200lab.kv8_append(x.cuda(), -x.cuda(), *s.cache, s.l, cu_seqlens=_prefix(n), max_seqlen=max(n))
        assert b200lab.device_status() == b200lab.OK
        s.rk.append(x.double().numpy(), s.table, s.lens, n)
        s.rv.append(-x.double().numpy(), s.table, s.lens, n)
        s.same()


def test_append_strided_views_and_rows_behind(cuda):
    """K and V as slices of one fused projection, more rows than the sequences have tokens: the rows
    behind the last sequence are not written anywhere."""
    Hq, Hkv, D, P = 4, 2, 128, 32
    lens, new = [40, 70], [40, 3]
    s = Setup(lens, Hkv, D, P, seed=8)
    total = sum(new) + 5
    qkv = _normal((total, (Hq + 2 * Hkv) * D), 4, torch.bfloat16).cuda()
    k = qkv[:, Hq * D:(Hq + Hkv) * D].view(total, Hkv, D)
    kv = _normal((total, Hkv, 2, D), 6, torch.bfloat16).cuda()
    v = kv[:, :, 1]  # heads are not contiguous either
    b200lab.kv8_append(k, v, *s.cache, s.l, cu_seqlens=_prefix(new), max_seqlen=max(new))
    assert b200lab.device_status() == b200lab.OK
    s.rk.append(k.double().cpu().numpy(), s.table, lens, new)
    s.rv.append(v.double().cpu().numpy(), s.table, lens, new)
    s.same()


def test_append_in_parts_equals_at_once_up_to_subnormals(cuda):
    """The scales do not depend on how a text is cut; codes only where they became subnormal on the way."""
    P, D, Hkv, n = 64, 128, 2, 200
    x = _normal((n, Hkv, D), 9, torch.bfloat16)
    a, b = Setup([n], Hkv, D, P, seed=1), Setup([n], Hkv, D, P, seed=1)
    b200lab.kv8_append(x.cuda(), x.cuda(), *a.cache, a.l, cu_seqlens=_prefix([n]), max_seqlen=n)
    at = 0
    for c in (1, 62, 2, 70, 65):
        part = x[at:at + c].cuda()
        at += c
        b200lab.kv8_append(part, part, *b.cache, _ints([at]), cu_seqlens=_prefix([c]), max_seqlen=c)
    assert b200lab.device_status() == b200lab.OK
    assert torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs)
    ka, kb = a.rk.__class__(a.k.view(torch.uint8).cpu().numpy(), a.ks.cpu().numpy()), \
        b.rk.__class__(b.k.view(torch.uint8).cpu().numpy(), b.ks.cpu().numpy())
    normal = np.abs(ka.values) >= 2.0 ** -6
    assert np.array_equal(ka.values[normal], kb.values[normal])
    assert np.abs(ka.values - kb.values).max() <= 2.0 ** -9


# ---- reading back ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,P,Hkv", [(64, 16, 3), (128, 64, 2), (256, 128, 1), (128, 128, 5)])
def test_read_exact(cuda, dtype, D, P, Hkv):
    lens = [1, P, 0, P + 1, 333, 2 * P - 1]
    s = Setup(lens, Hkv, D, P, seed=D, exps=(-14, 9), garbage=True)
    total = sum(lens) + 3
    kw = {n: torch.full((total, Hkv, D), 77.0, dtype=dtype, device="cuda") for n in ("k_out", "v_out")}
    k, v = b200lab.kv8_read(*s.cache, _prefix(lens), max(lens), total, **kw)
    assert b200lab.device_status() == b200lab.OK
    for got, r in ((k, s.rk), (v, s.rv)):
        want = np.concatenate([r.tokens(row, n) for row, n in zip(s.table, lens)])
        want = torch.from_numpy(want).to(dtype)  # the one rounding there may be (fp16)
        assert torch.equal(got[:sum(lens)].cpu(), want)
        assert bool((got[sum(lens):] == 77.0).all())


def test_read_part_of_the_sequences(cuda):
    s = Setup([200, 100], 2, 128, 64, seed=2)
    k, v = b200lab.kv8_read(*s.cache, _prefix([70, 0]), 70, 70, out_dtype=torch.float32)
    assert b200lab.device_status() == b200lab.OK
    assert np.array_equal(k.double().cpu().numpy(), s.rk.tokens(s.table[0], 70))
    assert np.array_equal(v.double().cpu().numpy(), s.rv.tokens(s.table[0], 70))


# ---- attention -------------------------------------------------------------------------------------------------------
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 1000]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8, 16, 20])
@pytest.mark.parametrize("P,dtype", [(16, torch.bfloat16), (64, torch.float16)])
def test_attend_step(cuda, D, group, P, dtype):
    """One query token a sequence, lengths around every border; NaN wherever no token lies."""
    s = Setup(LENS, 2, D, P, seed=D + group, garbage=True)
    q = _normal((len(LENS), 2 * group, D), 3, dtype).cuda()
    o = _check_attend(s, q, [1] * len(LENS))
    assert bool((o[0] == 0).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D,group", [(128, 4), (64, 1), (256, 6), (128, 8), (64, 5)])
def test_attend_several_tokens(cuda, D, group, P, causal):
    """Ragged query counts, some of them more than the sequence has keys (rows that see none), and more
    rows than one pass over the keys takes."""
    lens, new = [5, 64, 100, 17, 333, 2, 0], [5, 1, 9, 0, 7, 4, 2]
    s = Setup(lens, 2, D, P, seed=D + group, garbage=True)
    q = _normal((sum(new) + 2, 2 * group, D), 5, torch.bfloat16).cuda()
    out = torch.full_like(q, 55.0)
    _check_attend(s, q, new, causal=causal, out=out)
    assert bool((out[sum(new):] == 55.0).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_long_queries(cuda, D):
    """A prompt's worth of queries: many row tiles."""
    s = Setup([150, 90], 1, D, 64, seed=D, garbage=True)
    q = _normal((220, 3, D), 5, torch.float16).cuda()
    _check_attend(s, q, [150, 70])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_gate_and_strides(cuda, D):
    """The gated layer's projection: q and gate interleaved by head, taken as views."""
    lens = [70, 1, 400]
    s = Setup(lens, 2, D, 64, seed=D)
    qg = _normal((3, 12, 2, D), 6, torch.bfloat16, 2.0).cuda()
    _check_attend(s, qg[:, :, 0], [1, 1, 1], gate=qg[:, :, 1])
    odd = _normal((3, 12, D + 3), 7, torch.bfloat16, 2.0).cuda()[:, :, 3:]  # a gate on no boundary
    _check_attend(s, qg[:, :, 0], [1, 1, 1], gate=odd)


def test_attend_one_sequence_cut_over_all_ctas(cuda):
    """One long sequence and one kv-head: every CTA has a part of it, one kernel joins them all."""
    s = Setup([40001], 1, 128, 128, seed=3)
    q = _normal((2, 8, 128), 7, torch.bfloat16).cuda()
    _check_attend(s, q, [2])


def test_attend_scales_far_apart(cuda):
    """Blocks whose scales differ by up to 2^80: the largest values of V can have the smallest weights."""
    lens = [300, 64, 500]
    s = Setup(lens, 2, 128, 16, seed=4, exps=(-40, 40))
    s.ks.fill_(2.0 ** -7)
    s.rk.scales[:] = 2.0 ** -7
    q = _normal((3, 8, 128), 8, torch.float16).cuda()
    # fp16 holds no value above 65504: bf16 here
    _check_attend(s, q.to(torch.bfloat16), [1, 1, 1])


@pytest.mark.parametrize("dtype,std", [(torch.bfloat16, 1e30), (torch.bfloat16, 1e-30), (torch.float16, 3e-6), (torch.float16, 5e3)])
def test_attend_magnitudes_of_q(cuda, dtype, std):
    """Rows of q far outside fp16's comfortable range, with a scale that brings the scores back."""
    s = Setup([100, 33], 2, 128, 16, seed=4)
    q = _normal((2, 4, 128), 8, torch.float32, std).to(dtype).cuda()
    _check_attend(s, q, [1, 1], scale=float(0.09 / std))


def test_attend_sharp_scores(cuda):
    """Scores of some hundreds: one key takes all the weight, the running maximum moves again and again."""
    s = Setup([700], 1, 128, 64, seed=11)
    q = _normal((1, 8, 128), 9, torch.bfloat16, 6.0).cuda()
    _check_attend(s, q, [1], scale=1.0)


def test_attend_nan(cuda):
    """NaN in q reaches its row, NaN in K the rows that see the key, NaN in V that channel of the rows
    that see the key - and nothing else, though they lie in one product."""
    lens, new = [40, 90, 20], [6, 5, 3]
    s = Setup(lens, 2, 128, 16, seed=12)
    def poison(codes, ref, t, b, pos, h, d):
        blk, slot = s.table[b][pos // 16], pos % 16
        t.view(torch.uint8)[blk, h, slot, d] = 0x7f
        ref.values[blk, h, slot, d] = np.nan
    poison(s.k, s.rk, s.k, 0, 37, 0, 5)    # a new token: seen by queries 3.. of sequence 0
    poison(s.v, s.rv, s.v, 0, 38, 1, 100)  # seen by queries 4..
    poison(s.v, s.rv, s.v, 1, 3, 0, 64)    # an old token: seen by all
    poison(s.v, s.rv, s.v, 2, 19, 1, 7)    # the last token: seen by the last query
    q = _normal((sum(new), 8, 128), 10, torch.bfloat16)
    q[12, 3, 9] = float("nan")
    q[13, 1, 0] = float("inf")
    q = q.cuda()
    # the outputs reach 14 here, where half a step of bf16 alone is 2^-5: held to the bound of kv8_ref,
    # whose rows are computed from the keys they see, so that a masked NaN is really not there
    o = _check_attend(s, q, new)
    got = np.isnan(o.double().cpu().numpy())
    assert got[12, 3].all() and got[13, 1].all() and got[3:6, :4].all() and not got[:3].any()
    assert got[4:6, 4:, 100].all() and got[4:6, 4:].sum() == 8 and got[6:11, :4, 64].all() and got[6:11].sum() == 20
    assert got[13, 4:, 7].all() and got[11].sum() == 0


# ---- what a batch may bring ------------------------------------------------------------------------------------------
def test_bad_offsets_and_blocks_are_reported_not_followed(cuda):
    P, D, Hkv = 16, 128, 2
    lens = [40, 30, 20]
    q = _normal((3, 4, D), 1, torch.bfloat16).cuda()
    x = _normal((3, Hkv, D), 2, torch.bfloat16).cuda()
    good = Setup(lens, Hkv, D, P, seed=1)
    want = b200lab.attn_fwd_kv8(q, *good.cache, good.l)
    assert b200lab.device_status() == b200lab.OK

    for bad in (good.n_blocks, -1, 2 ** 31 - 1, -2 ** 31):
        s = Setup(lens, Hkv, D, P, seed=1)
        s.t[1, 1] = bad
        before = [a.clone() for a in (s.k.view(torch.uint8), s.v.view(torch.uint8))]
        o = b200lab.attn_fwd_kv8(q, *s.cache, s.l)
        assert b200lab.device_status() == b200lab.ERR_INVALID
        assert torch.equal(o[0], want[0]) and torch.equal(o[2], want[2])
        b200lab.kv8_append(x, x, *s.cache, s.l)  # sequence 1's new token lies in the bad block
        assert b200lab.device_status() == b200lab.ERR_INVALID
        mine = [s.table[0][2], s.table[2][1]]
        rest = [i for i in range(s.n_blocks) if i not in mine]
        for a, c in zip(before, (s.k, s.v)):
            assert torch.equal(a[rest], c.view(torch.uint8)[rest])
        k, v = b200lab.kv8_read(*s.cache, _prefix(lens), 40, 90)
        assert b200lab.device_status() == b200lab.ERR_INVALID
    s = Setup(lens, Hkv, D, P, seed=1)
    out = torch.full_like(q, 9.0)
    cases = [dict(lens=[40, 10 ** 6, 20]), dict(lens=[40, -5, 20]), dict(cu=[0, 1, 900, 901]), dict(cu=[0, 1, -3, 3]),
             dict(cu=[-2, 1, 2, 3]), dict(cu=[0, 3, 3, 3])]
    for c in cases:
        cu = None if "cu" not in c else _ints(c["cu"])
        out.fill_(9.0)
        most = 2 if cu is not None else 1
        b200lab.attn_fwd_kv8(q, *s.cache, _ints(c.get("lens", lens)), cu_seqlens_q=cu, max_seqlen_q=most, out=out)
        assert b200lab.device_status() == b200lab.ERR_INVALID, c
        if "lens" in c:
            assert bool((out[1] == 9.0).all()) and torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
    # more new tokens than max_seqlen, than the sequence holds; a read longer than its table
    before = s.k.view(torch.uint8).clone()
    b200lab.kv8_append(x, x, *s.cache, s.l, cu_seqlens=_ints([0, 0, 3, 3]), max_seqlen=2)
    assert b200lab.device_status() == b200lab.ERR_INVALID
    assert torch.equal(before, s.k.view(torch.uint8))
    before = s.k.view(torch.uint8).clone()
    b200lab.kv8_append(x, x, *s.cache, _ints([2, 30, 20]), cu_seqlens=_ints([0, 3, 3, 3]), max_seqlen=3)
    assert b200lab.device_status() == b200lab.ERR_INVALID
    assert torch.equal(before, s.k.view(torch.uint8))
    b200lab.kv8_read(*s.cache, _ints([0, 60, 60, 60]), 60, 60)
    assert b200lab.device_status() == b200lab.ERR_INVALID
    assert b200lab.device_status() == b200lab.OK


def test_shared_blocks_of_a_common_prefix(cuda):
    """Two sequences whose first blocks are the same ones."""
    s = Setup([80, 80], 2, 128, 16, seed=6)
    s.table[1][:4] = s.table[0][:4]
    s.t = _ints(s.table)
    _check_attend(s, _normal((2, 8, 128), 4, torch.bfloat16).cuda(), [1, 1])


def test_offsets_beyond_32_bits(cuda):
    """A cache of over 2^31 bytes a side, the sequence's blocks at its end."""
    Hkv, P, D = 8, 128, 256
    n_blocks = (1 << 31) // (Hkv * P * D) + 16
    k = torch.empty((n_blocks, Hkv, P, D), dtype=E4M3, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty((n_blocks, Hkv), device="cuda")
    vs = torch.empty_like(ks)
    n = 300
    ids = [n_blocks - 1, n_blocks - 9, n_blocks - 4]
    x = _normal((n, Hkv, D), 2, torch.bfloat16).cuda()
    y = _normal((n, Hkv, D), 3, torch.bfloat16).cuda()
    t = _ints([ids])
    b200lab.kv8_append(x, y, k, v, ks, vs, t, _ints([n]), cu_seqlens=_ints([0, n]), max_seqlen=n)
    a, b = b200lab.kv8_read(k, v, ks, vs, t, _ints([0, n]), n, n, out_dtype=torch.float32)
    # each value within half a step of e4m3 (2^-4 of it, or half a subnormal step of the block's scale)
    for got, want, sc in ((a, x, ks), (b, y, vs)):
        want = want.float()
        step = torch.maximum(want.abs() * 2.0 ** -4, sc[ids].max() * 2.0 ** -10)
        assert bool(((got - want).abs() <= step).all())
    q = _normal((1, 16, D), 4, torch.bfloat16).cuda()
    o = b200lab.attn_fwd_kv8(q, k, v, ks, vs, t, _ints([n]))
    assert b200lab.device_status() == b200lab.OK
    p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[0].double().view(8, 2, D), a.double()) / 16, -1)
    ref = torch.einsum("hgn,nhd->hgd", p, b.double()).reshape(1, 16, D)
    assert_close(to_np(o), ref.cpu().numpy())


def test_captured_graphs_and_streams(cuda):
    """append + attend captured once and replayed over a growing sequence, on a stream of their own, while
    another stream attends over another cache; each replay is what the same calls give outside a graph."""
    Hkv, D, P, B, steps = 2, 128, 16, 3, 20
    lens = [5, 60, 31]
    a = Setup([n + steps for n in lens], Hkv, D, P, seed=3)
    b = Setup([n + steps for n in lens], Hkv, D, P, seed=3)
    other = Setup([2000, 700], Hkv, D, P, seed=9)
    q2 = _normal((2, 8, D), 11, torch.bfloat16).cuda()
    want2 = b200lab.attn_fwd_kv8(q2, *other.cache, other.l)
    k, v, q = (torch.zeros((B, h, D), dtype=torch.bfloat16, device="cuda") for h in (Hkv, Hkv, 8))
    a.l.copy_(_ints(lens))
    side, noise = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.l += 1
        b200lab.kv8_append(k, v, *a.cache, a.l)
        o = b200lab.attn_fwd_kv8(q, *a.cache, a.l)
    for i in range(steps):
        for x, seed in ((k, 1), (v, 2), (q, 3)):
            x.copy_(_normal(x.shape, 100 * i + seed, torch.bfloat16))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        o2 = b200lab.attn_fwd_kv8(q2, *other.cache, other.l, stream=noise)
        torch.cuda.synchronize()
        now = _ints([n + i + 1 for n in lens])
        assert torch.equal(a.l, now)
        b200lab.kv8_append(k, v, *b.cache, now)
        assert torch.equal(o, b200lab.attn_fwd_kv8(q, *b.cache, now))
        assert torch.equal(o2, want2)
    assert b200lab.device_status() == b200lab.OK
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.vs, b.vs)


def test_capture_with_joined_streams(cuda):
    """The calls behind an event of another captured stream, as the last of two branches."""
    s, u = Setup([50, 7], 2, 64, 16, seed=5), Setup([50, 7], 2, 64, 16, seed=5)
    x, y, q = (_normal((2, h, 64), i, torch.bfloat16).cuda() for i, h in enumerate((2, 2, 4)))
    b200lab.kv8_append(x, y + 1, *u.cache, u.l)
    want = b200lab.attn_fwd_kv8(q, *u.cache, u.l)
    z, other = torch.empty_like(y), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        other.wait_stream(main)
        with torch.cuda.stream(other):
            torch.add(y, 1, out=z)
        w = x * 1
        main.wait_stream(other)
        b200lab.kv8_append(w, z, *s.cache, s.l)
        other.wait_stream(main)
        with torch.cuda.stream(other):
            o = b200lab.attn_fwd_kv8(q, *s.cache, s.l)
        main.wait_stream(other)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert b200lab.device_status() == b200lab.OK
    assert torch.equal(o, want) and torch.equal(s.v.view(torch.uint8), u.v.view(torch.uint8))


def test_same_call_twice_gives_the_same_bits(cuda):
    s = Setup([3000, 17, 911, 64], 4, 128, 64, seed=2)
    q = _normal((4, 16, 128), 4, torch.bfloat16).cuda()
    first = b200lab.attn_fwd_kv8(q, *s.cache, s.l)
    for _ in range(5):
        assert torch.equal(first, b200lab.attn_fwd_kv8(q, *s.cache, s.l))


def test_calls_share_the_library_of_the_other_entries(cuda):
    """The extension module calls the library that ctypes has loaded: one launch count, one status."""
    s = Setup([40], 2, 128, 16, seed=1)
    n = b200lab.launch_count()
    b200lab.attn_fwd_kv8(_normal((1, 8, 128), 1, torch.bfloat16).cuda(), *s.cache, s.l)
    n, before = b200lab.launch_count(), n
    assert n > before
    b200lab.kv8_append(_normal((1, 2, 128), 1, torch.bfloat16).cuda(), _normal((1, 2, 128), 2, torch.bfloat16).cuda(), *s.cache, s.l)
    assert b200lab.launch_count() == n + 1
    assert b200lab.device_status() == b200lab.OK


def test_many_sequences(cuda):
    """More sequences than a CTA has threads, most of them short or padding."""
    lens = [(i * 37) % 90 if i % 3 else 0 for i in range(700)]
    s = Setup(lens, 1, 64, 16, seed=7, garbage=True)
    _check_attend(s, _normal((700, 2, 64), 4, torch.bfloat16).cuda(), [1] * 700)


@pytest.mark.parametrize("D,Hkv,group,B,new", [(128, 8, 2, 230, 1), (64, 8, 1, 300, 1), (256, 8, 1, 150, 1),
                                               (128, 4, 4, 300, 3), (64, 8, 5, 225, 2)])
def test_many_segments(cuda, D, Hkv, group, B, new):
    """So many (sequence, kv-head) pairs that each warp takes segments of its own; a long sequence
    among them, which many warps share, and padding."""
    lens = [3000] + [(i * 29) % 71 if i % 5 else 0 for i in range(1, B)]
    counts = [new] + [(i * 7) % (new + 1) if new > 1 else 1 for i in range(1, B)]
    s = Setup(lens, Hkv, D, 16, seed=D + B, garbage=True)
    q = _normal((sum(counts), Hkv * group, D), 5, torch.bfloat16).cuda()
    _check_attend(s, q, counts)


def test_empty_batch_and_binding_refusals(cuda):
    s = Setup([20, 30], 2, 128, 16, seed=1)
    x = torch.zeros((0, 2, 128), dtype=torch.bfloat16, device="cuda")
    zero = _ints([0, 0, 0])
    b200lab.kv8_append(x, x, *s.cache, s.l, cu_seqlens=zero, max_seqlen=1)
    q = torch.zeros((0, 8, 128), dtype=torch.bfloat16, device="cuda")
    assert b200lab.attn_fwd_kv8(q, *s.cache, s.l, cu_seqlens_q=zero).shape == (0, 8, 128)
    k, v = b200lab.kv8_read(*s.cache, zero, 1, 0)
    assert k.shape == v.shape == (0, 2, 128)
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")  # no sequences at all
    b200lab.kv8_append(x, x, *s.cache[:4], none, none[:, 0].contiguous())
    assert b200lab.attn_fwd_kv8(q, *s.cache[:4], none, none[:, 0].contiguous()).shape == (0, 8, 128)
    s.same()
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        b200lab.attn_fwd_kv8(q[:, :, :64], *s.cache, s.l)
    with pytest.raises(ValueError):
        b200lab.attn_fwd_kv8(q, *s.cache, s.l.long())
    with pytest.raises(ValueError):
        b200lab.attn_fwd_kv8(q.transpose(1, 2).contiguous().transpose(1, 2), *s.cache, s.l)
    with pytest.raises(b200lab.B200LabError):
        b200lab.attn_fwd_kv8(q[:, :7], *s.cache, s.l)
    with pytest.raises(b200lab.B200LabError):
        b200lab.attn_fwd_kv8(q.float(), *s.cache, s.l)
    with pytest.raises(b200lab.B200LabError):
        b200lab.attn_fwd_kv8(q, *s.cache, s.l, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(TypeError):
        b200lab.kv8_append(q[:, :2], q[:, :2].float(), *s.cache, s.l)
    with pytest.raises(TypeError):
        b200lab.attn_fwd_kv8(q, s.k.view(torch.uint8), s.v.view(torch.uint8), s.ks, s.vs, s.t, s.l)
    with pytest.raises(b200lab.B200LabError):
        b200lab.kv8_append(q[:1, :2], q[:1, :2], *s.cache, s.l)  # one token a sequence, but one token for two


# ---- a serving loop --------------------------------------------------------------------------------------------------
def test_prompt_then_steps(cuda):
    """Prompts are appended and attended over by way of kv8_read and the packed attention, then tokens
    one at a time through the cache; both agree with the 64-bit attention over the codes, and the two
    ways with each other."""
    Hq, Hkv, D, P = 8, 2, 128, 32
    lens = [70, 1, 33, 129]
    extra = 3
    s = Setup([n + extra for n in lens], Hkv, D, P, seed=20)
    total = sum(lens)
    k, v, q = (_normal((total, h, D), i, torch.bfloat16) for i, h in enumerate((Hkv, Hkv, Hq)))
    cu, now = _prefix(lens), _ints(lens)
    b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, now, cu_seqlens=cu, max_seqlen=max(lens))
    s.rk.append(k.double().numpy(), s.table, lens, lens)
    s.rv.append(v.double().numpy(), s.table, lens, lens)
    kr, vr = b200lab.kv8_read(*s.cache, cu, max(lens), total)
    o = b200lab.attn_fwd_varlen(q.cuda(), kr, vr, cu, cu, max(lens), causal=True)
    assert b200lab.device_status() == b200lab.OK
    ref, _ = kv8_ref.attend(q.double().numpy(), s.rk, s.rv, s.table, lens, lens, 1 / np.sqrt(D), True)
    assert_close(to_np(o), ref, "prompt")
    s.lens, s.l = lens, now
    direct = _check_attend(s, q.cuda(), lens)
    assert_close(to_np(direct), to_np(o), "both ways")
    for i in range(extra):
        s.lens = [n + i + 1 for n in lens]
        s.l = _ints(s.lens)
        k, v, q = (_normal((4, h, D), 50 + 3 * i + j, torch.bfloat16) for j, h in enumerate((Hkv, Hkv, Hq)))
        b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, s.l)
        s.rk.append(k.double().numpy(), s.table, s.lens, [1] * 4)
        s.rv.append(v.double().numpy(), s.table, s.lens, [1] * 4)
        _check_attend(s, q.cuda(), [1] * 4)
    s.same()


def test_first_call_inside_a_capture(cuda):
    """A process whose first calls of all are recorded into a graph."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = %r
import b200lab
b200lab.lib()
c = [torch.zeros((4, 2, 16, 128), dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
s = [torch.zeros((4, 2), device="cuda") for _ in range(2)]
t = torch.tensor([[2, 1]], dtype=torch.int32, device="cuda")
n = torch.tensor([3], dtype=torch.int32, device="cuda")
x = torch.randn((3, 2, 128), device="cuda").to(torch.bfloat16)
cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b200lab.kv8_append(x, x, *c, *s, t, n, cu_seqlens=cu, max_seqlen=3)
    k, v = b200lab.kv8_read(*c, *s, t, cu, 3, 3)
    o = b200lab.attn_fwd_kv8(x, *c, *s, t, n, cu_seqlens_q=cu, max_seqlen_q=3)
g.replay()
torch.cuda.synchronize()
assert b200lab.device_status() == 0
assert torch.equal(o[0], v[0]) and float((k - x).abs().max()) < 0.5
print("fine")
""" % [p for p in sys.path if p]
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=dict(os.environ))
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


# ---- both ways of the attention --------------------------------------------------------------------------------------
class Wide(Setup):
    """The same with a block table for 9000 tokens: the attention then goes by its plan, where a table that is
    no wider than the lengths mostly gives a cluster of CTAs a segment."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        spare = torch.full((len(self.lens), 9000 // self.P), self.n_blocks + 7, dtype=torch.int32, device="cuda")
        self.t = torch.cat([self.t, spare], 1).contiguous()


@pytest.mark.parametrize("test,kw", [
    *((test_attend_step, dict(D=D, group=g, P=16, dtype=torch.bfloat16)) for D in (64, 128, 256) for g in (1, 8, 20)),
    *((test_attend_several_tokens, dict(D=D, group=g, P=P, causal=c))
      for D, g in ((128, 4), (64, 1), (256, 6), (64, 5)) for P in (16, 128) for c in (True, False)),
    *((test_attend_gate_and_strides, dict(D=D)) for D in (64, 128, 256)),
    *((test_attend_long_queries, dict(D=D)) for D in (64, 128, 256)),
    (test_attend_scales_far_apart, {}), (test_attend_sharp_scores, {}), (test_attend_nan, {}),
], ids=lambda x: x.__name__[5:] if callable(x) else "-".join(str(v) for v in x.values()))
def test_by_the_plan(cuda, monkeypatch, test, kw):
    monkeypatch.setitem(globals(), "Setup", Wide)
    test(cuda, **kw)


@pytest.mark.parametrize("D,group", [(64, 4), (64, 12), (128, 8), (128, 9), (256, 6), (256, 11)])
@pytest.mark.parametrize("B,longest", [(2, 900), (7, 500), (12, 950), (20, 260), (26, 990), (40, 500), (48, 130), (70, 40)])
def test_clusters_of_every_size(cuda, D, group, B, longest):
    """From one CTA a segment to eight, of four warps or eight, of which some have no keys; padding, several tokens, a gate, NaN wherever
    no token lies."""
    lens = [longest] + [(i * 53) % longest if i % 4 else 0 for i in range(1, B)]
    new = [(i * 5) % 4 for i in range(B)]
    s = Setup(lens, 2, D, 32, seed=D + B, garbage=True)
    q = _normal((sum(new) + 1, 2 * group, D), 6, torch.bfloat16).cuda()
    gate = _normal(tuple(q.shape), 7, torch.bfloat16, 2.0).cuda()
    out = torch.full_like(q, 55.0)
    _check_attend(s, q, new, gate=gate, out=out)
    assert bool((out[sum(new):] == 55.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_both_ways_agree(cuda, dtype):
    """A call by clusters and one by the plan on the same cache: each within its bound, so both together
    within twice that; and a call by clusters gives the same bits every time."""
    narrow, wide = (C([1000, 333, 64, 1], 4, 128, 32, seed=5) for C in (Setup, Wide))
    q = _normal((4, 16, 128), 8, dtype).cuda()
    a = _check_attend(narrow, q, [1] * 4)
    _check_attend(wide, q, [1] * 4)
    for _ in range(3):
        assert torch.equal(a, b200lab.attn_fwd_kv8(q, *narrow.cache, narrow.l))
