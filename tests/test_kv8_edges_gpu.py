"""GPU tests of calls at the edge of what the 8-bit key/value cache documents: blocks outside the pool between
good ones, padding entries, weights far below a row's largest."""
import numpy as np
import pytest
import torch

import b200lab
import kv8_ref
from test_kv8_gpu import UNIT, Setup, Wide, _check_attend, _ints, _normal, _prefix

pytestmark = pytest.mark.gpu


def _within(got, ref, bound):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    over = np.abs(got - ref)[fine] - bound[fine]
    assert over.size == 0 or over.max() <= 0, f"{over.max():.3e} over its bound, error {np.abs(got - ref)[fine].max():.3e}"


@pytest.mark.parametrize("kind", [Setup, Wide], ids=["narrow", "wide"])
@pytest.mark.parametrize("D,Hkv,B", [(64, 2, 3), (128, 2, 3), (256, 2, 3), (64, 8, 300), (128, 8, 230), (256, 8, 150)])
def test_attend_bad_blocks_between_good_ones(cuda, kind, D, Hkv, B):
    """Blocks of 16 keys, every other one outside the pool: a piece of keys that a warp takes at a time has a
    group of each sort, and the next piece in its place the other way round.  The good blocks' keys count, with
    their own scales; by clusters, by the plan, and with a warp a segment."""
    lens = [(37 * i) % 300 + 1 if B > 3 else n for i, n in zip(range(B), [40, 333, 1000] * B)]
    s = kind(lens, Hkv, D, 16, seed=D + B, exps=(-12, -3))
    good, left = [], []
    for b, n in enumerate(lens):
        used = -(-n // 16)
        bad = [i for i in range(used - 1) if (i + i // 4) % 2]  # never the last one, which may not be full
        for i in bad:
            s.t[b, i] = (-1, s.n_blocks)[i % 3 == 0]
        good.append([s.table[b][i] for i in range(used) if i not in bad])
        left.append(n - 16 * len(bad))
    q = _normal((B, 2 * Hkv, D), 3, torch.bfloat16).cuda()
    o = b200lab.attn_fwd_kv8(q, *s.cache, s.l)
    assert b200lab.device_status() == (b200lab.ERR_INVALID if good != [t[:-(-n // 16)] for t, n in zip(s.table, lens)]
                                       else b200lab.OK)
    ref, bound = kv8_ref.attend(q.double().cpu().numpy(), s.rk, s.rv, good, left, [1] * B, 1 / np.sqrt(D), True,
                                unit=UNIT[q.dtype])
    _within(o, ref, bound)


# ---- weights far below a row's largest -------------------------------------------------------------------------------
def _attend_tight(s, q, scale):
    """(o, bound) of one query token a sequence, where the weights' fp16 range may cost little.

    A warp takes the keys in pieces of at most 32, from multiples of 32 on.  Its weights 2^(x - m), x with the log of
    V's scale, are held to at most 2^15 (below fp16's end, 2^16), and a piece's largest to at least 2^-8, unless the
    row's sums, moved to such an m, pass 2^60.  Rounded to fp16 they are off by 2^-11 of themselves, or by 2^-25 where
    they are subnormal: 2^-17 of the piece's largest.  So beside the relative roundings (kv8_ref.attend), each
    piece adds 2^-17 (its largest w sV) sum |codes|, and a weight beyond the sums' range is under 2^-25 / 2^58 of a
    unit of l: 448 2^-83 a key.  Nothing here grows with the distance between a weight and the row's largest.
    The output's own rounding is off by half a step: of the value, or, for an fp16 value below 2^-14, of the steps of
    2^-24 that its subnormal numbers have: 2^-25."""
    B, Hq, D = q.shape
    unit, least = UNIT[q.dtype], 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -32
    qd = q.double().cpu().numpy()
    o, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(s.lens):
        k, v = s.rk.tokens(s.table[b], n), s.rv.tokens(s.table[b], n)
        sv = s.rv.token_scales(s.table[b], n)
        for hq in range(Hq):
            h = hq // (Hq // s.Hkv)
            x = scale * (k[:, h] @ qd[b, hq])
            p = np.exp(x - x.max())
            w = p / p.sum()
            o[b, hq] = w @ v[:, h]
            size = w @ np.abs(v[:, h])
            dx = (D + 4) * 2.0 ** -22 * scale * (np.abs(k[:, h]) @ np.abs(qd[b, hq])).max()
            at = np.arange(0, n, 32)
            largest = np.maximum.reduceat(w * sv[:, h], at)
            codes = np.add.reduceat(np.abs(v[:, h]) / sv[:, h][:, None], at)
            bound[b, hq] = ((2 * (dx + 2.0 ** -20 + n * 2.0 ** -24) + 2.0 ** -11) * size + 2.0 ** -17 * (largest @ codes)
                            + n * 448 * 2.0 ** -83 + unit * np.abs(o[b, hq]) * (1 + 2.0 ** -6) + least)
    return o, bound


def _check_tight(s, q, scale, copies=1):
    """A call with the cache as the reference has it.  copies: that many sequences of the same blocks and queries,
    so that a warp has a whole sequence, or a quarter of one, not the few keys that it has of a lone one."""
    for t, ts, r in ((s.k, s.ks, s.rk), (s.v, s.vs, s.rv)):
        t.copy_(torch.from_numpy(r.values).float().to(t.dtype))
        ts.copy_(torch.from_numpy(r.scales).float())
    table, lens = s.t.repeat(copies, 1), s.l.repeat(copies)
    o = b200lab.attn_fwd_kv8(q.repeat(copies, 1, 1), s.k, s.v, s.ks, s.vs, table, lens, scale=scale)
    assert b200lab.device_status() == b200lab.OK
    ref, bound = _attend_tight(s, q, scale)
    for x in o.view(copies, *q.shape):
        _within(x, ref, bound)


def _sink(s, b, pos, h, D):
    """Makes every score of sequence b's head h zero but that of the key at `pos`: q's channel 0 times 448 sK."""
    for i in range(-(-s.lens[b] // s.P)):
        s.rk.values[s.table[b][i], h] = 0
    s.rk.values[s.table[b][pos // s.P], h, pos % s.P, 0] = 448


def _q_of_bits(bits, D, sk, dtype):
    """Rows whose score with the sink (scale 1) lies that many powers of two above the others'."""
    q = torch.zeros((1, len(bits), D), dtype=torch.float32)
    q[0, :, 0] = torch.tensor(bits) * float(np.log(2)) / (448 * sk)
    return q.to(dtype).cuda()


BITS = [0.0, 13.0, 16.5, 20.3, 24.5, 25.5, 29.0, 36.0]


# one segment cut over all CTAs, one in a cluster, CTAs of four warps with a segment each, warps with one each
FORMS = [(Setup, 128, 131072, 1), (Setup, 128, 900, 1), (Wide, 128, 2000, 450), (Wide, 128, 3000, 1800), (Setup, 128, 500, 450),
         (Setup, 64, 700, 1), (Wide, 64, 2000, 600), (Wide, 64, 2000, 2400), (Setup, 64, 250, 580),
         (Setup, 256, 500, 1), (Wide, 256, 2000, 300), (Wide, 256, 2000, 1200), (Setup, 256, 250, 300)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,D,n,copies", FORMS)
def test_attend_one_sharp_key_and_a_long_even_tail(cuda, kind, D, n, copies, dtype):
    """One key takes most of the weight, of values 0; all the others share the rest evenly, and make the output.
    The rows differ by how far below the sharp key's the others' weights are."""
    s = kind([n], 1, D, 64, seed=n + D, exps=(-6, -6))
    s.rk.scales[:] = 2.0 ** -7
    pos = n // 20
    _sink(s, 0, pos, 0, D)
    s.rv.values[:] = np.abs(s.rv.values)  # of one sign: what is lost of the tail is not noise
    # nothing but the tail in the output: the sharp key's 31 neighbours would be a term of the bound
    s.rv.values[s.table[0][pos // 64], 0, pos % 64 // 32 * 32:][:32] = 0
    _check_tight(s, _q_of_bits(BITS, D, 2.0 ** -7, dtype), 1.0, copies)


@pytest.mark.parametrize("kind,D,n,copies", FORMS)
@pytest.mark.parametrize("far", [9, 11, 20, 44])
def test_attend_sharp_key_in_a_block_of_large_values(cuda, kind, D, n, copies, far):
    """The sharp key's block has a V scale 2^far times the others', and codes of 0 in all channels but one: the
    other channels are made by the small weights alone."""
    s = kind([n], 1, D, 16, seed=far, exps=(-12, -12))
    s.rk.scales[:] = 2.0 ** -7
    pos = n // 20
    _sink(s, 0, pos, 0, D)
    s.rv.values[:] = np.abs(s.rv.values)
    block = s.table[0][pos // 16]
    s.rv.scales[block] = 2.0 ** (far - 12)
    for i in (pos // 32 * 2, pos // 32 * 2 + 1):  # and its neighbours' in a piece of 32
        s.rv.values[s.table[0][i]] = 0
    s.rv.values[block, 0, pos % 16, 9] = 448
    _check_tight(s, _q_of_bits(BITS, D, 2.0 ** -7, torch.bfloat16), 1.0, copies)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,D,n,copies", FORMS[:1] + FORMS[2:5] + FORMS[6:])
def test_attend_references_that_move_at_every_piece(cuda, kind, D, n, copies, dtype):
    """Every other 32 keys take nearly all of the weight, of values 0; the others make the output."""
    s = kind([n], 1, D, 32, seed=n + D, exps=(-6, -6))
    s.rk.scales[:] = 2.0 ** -7
    s.rk.values[:] = 0
    s.rv.values[:] = np.abs(s.rv.values)
    for block in s.table[0][:-(-n // 32)][::2]:
        s.rk.values[block, :, :, 0] = 448
        s.rv.values[block] = 0
    _check_tight(s, _q_of_bits([0.0, 13.0, 19.0, 24.5, 25.5, 30.0, 36.0, 47.0], D, 2.0 ** -7, dtype), 1.0, copies)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,B,Hkv", [(Setup, 20, 2), (Wide, 20, 2), (Setup, 300, 8), (Wide, 300, 8)])
@pytest.mark.parametrize("D,group", [(64, 3), (128, 4), (128, 12), (256, 6)])
def test_attend_the_largest_weight_is_exact(cuda, kind, B, Hkv, D, group, dtype):
    """A row whose first key has all of the weight gives that key's values, to the bit: the reference stands at a whole
    number of powers of two below it, so fp16 holds its weight as it is (off by 2^-21 of the exponential, far from
    half a step of the output).  A lone key's, and one's 60 powers of two above the others'."""
    lens = [1 + 40 * (i % 2) for i in range(B)]
    s = kind(lens, Hkv, D, 16, seed=D + group, exps=(-8, -5))
    s.rk.scales[:] = 2.0 ** -7
    q = _normal((B, Hkv * group, D), 7, torch.float32)
    q[..., 0] = q[..., 0].abs() + 17  # scores of 17 * 3.5 = 59 and more with the first key, of 0 with the others
    for b in range(1, B, 2):
        for i in range(3):
            s.rk.values[s.table[b][i]] = 0
        s.rk.values[s.table[b][0], :, 0, 0] = 448
    s.rv.values[s.rv.values == 0] = 1  # where the first key's were 0, the others' 2^-60 would be the answer
    for t, r in ((s.k, s.rk), (s.v, s.rv)):
        t.copy_(torch.from_numpy(r.values).float().to(t.dtype))
    s.ks.copy_(torch.from_numpy(s.rk.scales).float())
    o = b200lab.attn_fwd_kv8(q.to(dtype).cuda(), *s.cache, s.l, scale=1.0)
    assert b200lab.device_status() == b200lab.OK
    want = np.stack([s.rv.tokens(s.table[b], 1)[0] for b in range(B)]).repeat(group, axis=1)
    off = (o.cpu() != torch.from_numpy(want).to(dtype)).nonzero().tolist()
    assert not off, f"{len(off)} differ, the first at {off[0]}"


@pytest.mark.parametrize("copies", [1, 60, 240])
@pytest.mark.parametrize("kind", [Setup, Wide], ids=["narrow", "wide"])
@pytest.mark.parametrize("D,group,P", [(64, 8, 16), (128, 4, 16), (128, 12, 32), (256, 6, 128), (64, 20, 64)])
def test_attend_scales_far_apart_tight(cuda, kind, D, group, P, copies):
    """V scales of 2^-40 to 2^40 in no order, scores some tens apart: rows' references go up and down all the time."""
    s = kind([900, 64, 333, 1, 40], 2, D, P, seed=D + P, exps=(-40, 40))
    s.rk.scales[:] = np.exp2(np.random.default_rng(3).integers(-8, -3, s.rk.scales.shape))
    _check_tight(s, _normal((5, 2 * group, D), 6, torch.bfloat16, 2.0).cuda(), 0.09, copies)


@pytest.mark.parametrize("copies", [1, 450, 1800])
def test_attend_tail_beyond_the_sums_range(cuda, copies):
    """Blocks of zeros have the smallest scale; here all have it, and the tail lies up to 2^-300 below the sharp key:
    nothing overflows, and what is lost is below any value that the cache can hold."""
    s = Wide([3000], 1, 128, 16, seed=1, exps=(-40, -40))
    s.rk.scales[:] = 2.0 ** -7
    _sink(s, 0, 700, 0, 128)
    _check_tight(s, _q_of_bits([1.0, 20.0, 45.0, 70.0, 100.0, 120.0, 126.0, 300.0], 128, 2.0 ** -7, torch.bfloat16), 1.0,
                 copies)


# ---- rows that see no key --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,D,Hkv,group,lens,new", [
    (Setup, 128, 2, 4, [0, 70, 0, 5], [1, 1, 1, 1]),                          # clusters
    (Setup, 64, 2, 5, [3, 0, 200], [7, 2, 2]),
    (Wide, 128, 2, 4, [0, 70, 0, 5], [1, 1, 1, 1]),                           # the plan, four warps a CTA
    (Wide, 256, 2, 3, [3, 0, 200], [7, 2, 2]),
    (Wide, 64, 8, 2, [(i * 7) % 40 if i % 3 else 0 for i in range(300)], [1] * 300),  # a warp a CTA
    (Setup, 128, 8, 2, [(i * 7) % 40 if i % 3 else 0 for i in range(300)], [1] * 300),
    (Wide, 128, 1, 4, [300], [310]),                                          # cut segments, a warp a row joins them
    (Wide, 128, 1, 1, [129], [130]),                                          # cut segments, a block a row
    (Wide, 256, 1, 1, [129], [133])])
def test_rows_without_keys_are_zero_whatever_their_gate(cuda, kind, D, Hkv, group, lens, new):
    """A padded batch's unwritten activations: q and the gate are NaN or infinite in the rows that see no key."""
    s = kind(lens, Hkv, D, 16, seed=D, garbage=True)
    q, gate = (_normal((sum(new), Hkv * group, D), i, torch.bfloat16) for i in (5, 6))
    none = torch.tensor([n - m + i < 0 for n, m in zip(lens, new) for i in range(m)])
    assert bool(none.any())
    ref, bound = kv8_ref.attend(q.double().numpy(), s.rk, s.rv, s.table, lens, new, 1 / np.sqrt(D), True,
                                gate.double().numpy(), UNIT[q.dtype])
    assert not ref[none.numpy()].any()
    q[none] = float("nan")
    gate[none] = float("nan")
    gate[none, 0, 1] = float("inf")
    one = max(new) == 1
    out = torch.full(q.shape, 55.0, dtype=q.dtype, device="cuda")
    b200lab.attn_fwd_kv8(q.cuda(), *s.cache, s.l, cu_seqlens_q=None if one else _prefix(new), max_seqlen_q=max(new),
                         gate=gate.cuda(), out=out)
    assert b200lab.device_status() == b200lab.OK
    assert bool((out[none.cuda()] == 0).all())
    _within(out, ref, bound)


# ---- padding entries -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [-1, -5, -2 ** 31])
def test_append_reports_a_negative_length(cuda, bad):
    """A padding entry of a step has length 0; the step's append and its attention both report a negative one."""
    s = Setup([20, 30, 40], 2, 128, 16, seed=1)
    k, v = (_normal((3, 2, 128), i, torch.bfloat16) for i in (1, 2))
    lens = _ints([20, bad, 40])
    b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, lens)
    assert b200lab.device_status() == b200lab.ERR_INVALID
    for r, x in ((s.rk, k), (s.rv, v)):
        r.append(x.double().numpy()[[0, 2]], [s.table[0], s.table[2]], [20, 40], [1, 1])
    s.same()
    b200lab.attn_fwd_kv8(_normal((3, 4, 128), 3, torch.bfloat16).cuda(), *s.cache, lens)
    assert b200lab.device_status() == b200lab.ERR_INVALID
    b200lab.kv8_append(k.cuda(), v.cuda(), *s.cache, _ints([0, 0, 0]))
    assert b200lab.device_status() == b200lab.OK
    s.same()


# ---- the host's side -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [Setup, Wide], ids=["narrow", "wide"])
def test_calls_after_a_failed_call_of_the_program(cuda, kind):
    """The runtime remembers the last error of a thread, here that of selecting a device that there is not; it
    is not the following calls'."""
    import ctypes
    s, t = kind([900, 33], 2, 128, 16, seed=1), kind([900, 33], 2, 128, 16, seed=1)
    x = _normal((2, 2, 128), 1, torch.bfloat16).cuda()
    q = _normal((2, 8, 128), 2, torch.bfloat16).cuda()
    cu = _ints([0, 900, 933])
    b200lab.kv8_append(x, x, *t.cache, t.l)
    want, (wk, wv) = b200lab.attn_fwd_kv8(q, *t.cache, t.l), b200lab.kv8_read(*t.cache, cu, 900, 933)
    runtime = ctypes.CDLL("libcudart.so.12")
    # every buffer given: torch's allocator looks at the last error, too, where it takes new memory
    out, k, v = torch.empty_like(want), torch.empty_like(wk), torch.empty_like(wv)
    ws = torch.empty(b200lab.attn_fwd_kv8_workspace_bytes(8, 2, 1, 128), dtype=torch.uint8, device="cuda")
    calls = (lambda: b200lab.kv8_append(x, x, *s.cache, s.l),
             lambda: b200lab.attn_fwd_kv8(q, *s.cache, s.l, out=out, workspace=ws),
             lambda: b200lab.kv8_read(*s.cache, cu, 900, 933, k_out=k, v_out=v))
    got = []
    try:
        for call in calls:
            assert runtime.cudaSetDevice(4096) != 0
            got.append(call())
    finally:
        runtime.cudaGetLastError()
    assert b200lab.device_status() == b200lab.OK
    assert torch.equal(got[1], want) and torch.equal(got[2][0], wk) and torch.equal(got[2][1], wv)


# ---- strides ---------------------------------------------------------------------------------------------------------
def test_strides_of_dimensions_of_one(cuda):
    """One token, or one kv-head, cut out of rows of any length: the stride that is never taken does not matter."""
    D = 128
    wide = torch.zeros((1, 3 * 2 * D + 4), dtype=torch.bfloat16, device="cuda")  # a projection with four values more
    wide.copy_(_normal(tuple(wide.shape), 3))
    st = (3 * 2 * D + 4, D, 1)
    q, k, v = (wide.as_strided((1, 2, D), st, i * 2 * D) for i in range(3))
    s, t = (Setup([40], 2, D, 16, seed=1) for _ in range(2))
    for c, args in ((s, (q, k, v, q)), (t, tuple(x.clone(memory_format=torch.contiguous_format) for x in (q, k, v, q)))):
        b200lab.kv8_append(args[1], args[2], *c.cache, c.l)
        c.o = b200lab.attn_fwd_kv8(args[0], *c.cache, c.l, gate=args[3])
    assert torch.equal(s.o, t.o) and torch.equal(s.k.view(torch.uint8), t.k.view(torch.uint8))
    rows = _normal((3, D + 8), 4, torch.bfloat16).cuda()
    one = rows.as_strided((3, 1, D), (D + 8, 5, 1))
    s, t = (Setup([40, 7, 19], 1, D, 16, seed=2) for _ in range(2))
    for c, x in ((s, one), (t, one.clone(memory_format=torch.contiguous_format))):
        b200lab.kv8_append(x, x, *c.cache, c.l)
        c.o = b200lab.attn_fwd_kv8(x, *c.cache, c.l, gate=x)
    assert b200lab.device_status() == b200lab.OK
    assert torch.equal(s.o, t.o) and torch.equal(s.v.view(torch.uint8), t.v.view(torch.uint8))


# ---- NaN that some rows do not see -----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,D,group,B", [(Setup, 64, 4, 3), (Setup, 256, 4, 3), (Wide, 64, 4, 3), (Wide, 256, 4, 3),
                                            (Wide, 128, 4, 3), (Setup, 64, 12, 3), (Wide, 128, 12, 3),
                                            (Wide, 64, 2, 300), (Wide, 128, 2, 230), (Wide, 256, 2, 150), (Wide, 128, 5, 230)])
def test_attend_masked_nan_in_every_channel(cuda, kind, D, group, B):
    """NaN in V at new tokens, each in channels of its own (all of them over the batch, and over the tokens of the
    first sequence): it reaches those channels of the rows that see the key, and no other."""
    new = [4 if B < 100 else 2] * B
    lens = [(b * 31) % 90 + 8 for b in range(B)]
    s = kind(lens, 2 if B < 100 else 8, D, 16, seed=D + group, garbage=True)
    for b in range(B):
        for i in range(1, new[b]):
            pos = lens[b] - new[b] + i
            blk, slot = s.table[b][pos // 16], pos % 16
            for d in range((b * 5 + i) % 7, D, 7):
                s.v.view(torch.uint8)[blk, 1, slot, d] = 0x7f if d % 2 else 0xff
                s.rv.values[blk, 1, slot, d] = np.nan
    q = _normal((sum(new), s.Hkv * group, D), 9, torch.bfloat16)
    o = b200lab.attn_fwd_kv8(q.cuda(), *s.cache, s.l, cu_seqlens_q=_prefix(new), max_seqlen_q=max(new))
    assert b200lab.device_status() == b200lab.OK
    ref, bound = kv8_ref.attend(q.double().numpy(), s.rk, s.rv, s.table, lens, new, 1 / np.sqrt(D), True,
                                unit=UNIT[q.dtype])
    assert np.isnan(ref).any() and not np.isnan(ref[::new[0]]).any()
    _within(o, ref, bound)


# ---- one long sequence among short ones ------------------------------------------------------------------------------
@pytest.mark.parametrize("D,Hkv,group,B,new", [(128, 1, 1, 64, 1), (128, 1, 3, 64, 1), (128, 1, 4, 64, 1), (128, 1, 8, 64, 1),
                                               (64, 1, 2, 64, 1), (64, 2, 5, 40, 3), (128, 1, 4, 40, 5), (256, 1, 6, 64, 1),
                                               (256, 1, 4, 30, 3), (128, 8, 2, 230, 1), (64, 8, 1, 300, 1)])
def test_attend_one_long_sequence_among_short_ones(cuda, D, Hkv, group, B, new):
    """Nearly all parts are one segment's, of one to sixteen rows: the warps of its join share them.  The largest
    values lie in one part, rows that see no key and padding in the short ones."""
    lens = [(i * 13) % 29 for i in range(B)]
    lens[B // 3] = 20000
    counts = [(i * 7) % (new + 1) if new > 1 else 1 for i in range(B)]
    counts[B // 3] = new
    s = Wide(lens, Hkv, D, 32, seed=D + B, garbage=True)
    s.rv.scales[s.table[B // 3][400]] *= 64
    s.vs.copy_(torch.from_numpy(s.rv.scales).float())
    q = _normal((sum(counts), Hkv * group, D), 5, torch.bfloat16).cuda()
    gate = _normal(tuple(q.shape), 6, torch.bfloat16).cuda()
    _check_attend(s, q, counts, gate=gate)
    first = b200lab.attn_fwd_kv8(q, *s.cache, s.l, cu_seqlens_q=_prefix(counts), max_seqlen_q=new, gate=gate)
    assert torch.equal(first, b200lab.attn_fwd_kv8(q, *s.cache, s.l, cu_seqlens_q=_prefix(counts), max_seqlen_q=new, gate=gate))
