"""The operators of the 8-bit key/value cache, as a serving program calls them, with plain forms to measure against.

The cache is paged.  k_cache and v_cache are [n_blocks][Hkv][block_size][D] in 8 bits (e4m3: 4 bits of exponent, 3 of
mantissa, largest value 448); k_scale and v_scale are [n_blocks][Hkv], one power of two for each block of tokens and
head; a sequence's token at position p lies in block block_table[b][p // block_size], slot p % block_size, and stands
for code * scale.

* append  writes a batch's new tokens: a block's scale is the smallest power of two 2^e, -40 <= e <= 40, with
          max |x| <= 448 * 2^e over the finite values written to it (one that was begun earlier keeps its scale where
          that is larger, and has its codes rounded to the new one where it is smaller); codes are rounded to nearest
          even, what is larger than 448 becomes 448.
* read    gives the tokens of sequences back in 16 bits, packed one sequence after the other.
* attend  softmax attention of a batch's last tokens over the cache, each of them seeing the keys up to its own
          position, with an optional sigmoid gate.
"""
import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_E = 40
LARGEST = 64 * 16384 * 8 * 128  # the listed cases' largest cache: values of K (or of V) in it


# ---- cases -----------------------------------------------------------------------------------------------------------
def _attend(name, B, length, spread, Hq, Hkv, D, block, dtype, new=1, gate=False):
    return {"name": name, "op": "attend", "B": B, "length": length, "spread": spread, "Hq": Hq, "Hkv": Hkv, "D": D,
            "block": block, "dtype": dtype, "new": new, "gate": gate}


def _append(name, B, length, spread, new, Hkv, D, block, dtype):
    return {"name": name, "op": "append", "B": B, "length": length, "spread": spread, "new": new, "Hkv": Hkv, "D": D,
            "block": block, "dtype": dtype}


def _read(name, B, length, spread, Hkv, D, block, dtype):
    return {"name": name, "op": "read", "B": B, "length": length, "spread": spread, "Hkv": Hkv, "D": D, "block": block,
            "dtype": dtype}


def listed():
    return [
        # one user's next token after a short prompt: latency alone
        _attend("attend one short", 1, 1000, 0.0, 32, 8, 128, 64, "bf16"),
        # one user's next token far into a long text
        _attend("attend one long", 1, 16384, 0.0, 32, 8, 128, 64, "bf16"),
        # an ordinary batch of conversations of every length
        _attend("attend batch ragged", 64, 8192, 0.95, 32, 8, 128, 64, "bf16"),
        # a full batch of long texts: bandwidth
        _attend("attend batch long", 64, 16384, 0.0, 32, 8, 128, 64, "bf16"),
        # four drafted tokens a sequence, verified at once
        _attend("attend drafts", 16, 4099, 0.5, 32, 8, 128, 32, "fp16", new=4),
        # the gated layer: 24 q-heads on 4 kv-heads of 256, gate after the softmax
        _attend("attend gated d256", 32, 4000, 0.5, 24, 4, 256, 64, "bf16", gate=True),
        # small heads, one q-head to a kv-head, blocks of 16 tokens
        _attend("attend d64", 48, 2500, 0.9, 8, 8, 64, 16, "fp16"),
        # the step of a batch: one new token a sequence
        _append("append step", 64, 4096, 0.5, 1, 8, 128, 64, "bf16"),
        # prompts of every length, some of them the next turn of a conversation
        _append("append prompts", 8, 8192, 0.9, 6001, 8, 128, 64, "bf16"),
        # a few tokens of the gated layer, kept in fp32 by the program until here
        _append("append few d256", 7, 1111, 0.5, 5, 4, 256, 32, "fp32"),
        # the context of a few sequences, for the attention of a long prompt's next part
        _read("read ragged", 8, 16384, 0.8, 8, 128, 64, "bf16"),
        _read("read short d64", 3, 333, 0.5, 8, 64, 16, "fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "read"])
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    block = rng.choice([16, 32, 64, 128])
    spread = round(rng.uniform(0.0, 0.98), 2)
    B = _log(rng, 1, 128)
    length = _log(rng, 1, 20000)
    while B * length * Hkv * D > LARGEST // 4:
        length = max(1, length // 2)
    dtype = rng.choice(["bf16", "fp16"])
    if op == "attend":
        new = min(length, rng.choice([1, 1, 1, rng.randint(2, 8)]))
        c = _attend("", B, length, spread, Hkv * rng.choice([1, 2, 4, 5, 6, 8]), Hkv, D, block, dtype, new,
                    rng.random() < 0.3)
    elif op == "append":
        new = min(length, rng.choice([1, rng.randint(2, 16), _log(rng, 16, 8192)]))
        c = _append("", B, length, spread, new, Hkv, D, block, rng.choice(["bf16", "fp16", "fp32"]))
    else:
        c = _read("", B, length, spread, Hkv, D, block, dtype)
    del c["name"]
    return c


def _power(e):
    """2^e in 32 bits, exactly, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _fraction(b, a):
    return (b * a) % 1.0


def _lengths(c):
    """Tokens of each sequence, the batch's new ones among them, and how many of them are new: from the case alone."""
    lens = [max(1, int(round(c["length"] * (1 - c["spread"] * _fraction(b, 0.6180339887))))) for b in range(c["B"])]
    new = c.get("new", 1)
    return lens, [min(n, max(1, int(round(new * (1 - 0.8 * _fraction(b, 0.3819660113)))))) for b, n in enumerate(lens)]


def work(c):
    lens, new = _lengths(c)
    row = c["Hkv"] * c["D"]
    size = 4 if c["dtype"] == "fp32" else 2
    blocks = [-(-n // c["block"]) for n in lens]
    if c["op"] == "attend":
        seen = sum(sum(range(n - m + 1, n + 1)) for n, m in zip(lens, new))  # keys, over all queries
        rows = (3 if c["gate"] else 2) * sum(new) * c["Hq"] * c["D"]
        return {"bytes": 2 * sum(lens) * row + 8 * sum(blocks) * c["Hkv"] + size * rows,
                "flops": 4 * c["Hq"] * c["D"] * seen}
    if c["op"] == "append":
        touched = sum(n // c["block"] - (n - m) // c["block"] + (n % c["block"] != 0) for n, m in zip(lens, new))
        return {"bytes": 2 * sum(new) * row * (size + 1) + 8 * touched * c["Hkv"], "flops": 4 * sum(new) * row}
    return {"bytes": 2 * sum(lens) * row * (1 + size) + 8 * sum(blocks) * c["Hkv"], "flops": 2 * sum(lens) * row}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(c, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    lens, new = _lengths(c)
    B, Hkv, D, P = c["B"], c["Hkv"], c["D"], c["block"]
    used = [-(-n // P) for n in lens]
    width = max(used)
    n_blocks = sum(used) + 3  # a few blocks that no sequence has
    # the blocks of a pool after some use: in no order; entries past a sequence's last block are 0
    order = list(range(n_blocks))
    random.Random(seed).shuffle(order)
    rows, at = [], 0
    for u in used:
        rows.append(order[at:at + u] + [0] * (width - u))
        at += u
    dtype = DTYPES[c["dtype"]]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def prefix(v):
        return ints([0] + [sum(v[:i + 1]) for i in range(len(v))])

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32)

    def codes():
        x = torch.empty((n_blocks, Hkv, P, D), device=dev, dtype=E4M3)
        step = max(1, (1 << 26) // (Hkv * P * D))
        for i in range(0, n_blocks, step):
            x[i:i + step] = (normal(min(step, n_blocks - i), Hkv, P, D) * 80).clamp(-448, 448).to(E4M3)
        return x

    def scales():  # values of about 1, as of keys and values behind a norm
        return _power(torch.randint(-8, -4, (n_blocks, Hkv), generator=g, device=dev))

    s = dict(c, k_cache=codes(), v_cache=codes(), k_scale=scales(), v_scale=scales(), table=ints(rows))
    if c["op"] == "read":
        return dict(s, cu=prefix(lens), total=sum(lens), longest=max(lens), out_dtype=dtype)
    s["lens"] = ints(lens)
    s["cu"] = prefix(new) if c["new"] > 1 else None
    s["most"] = max(new)
    total = sum(new)
    if c["op"] == "append":
        # K and V as a fused projection leaves them: slices of one row a token
        kv = normal(total, 2 * Hkv * D).to(dtype)
        return dict(s, k=kv[:, :Hkv * D].view(total, Hkv, D), v=kv[:, Hkv * D:].view(total, Hkv, D))
    s["q"] = normal(total, c["Hq"], D).to(dtype)
    s["g"] = normal(total, c["Hq"], D).to(dtype) if c["gate"] else None
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"attend": _plain_attend, "append": _plain_append, "read": _plain_read}[s["op"]](s)


def _own(s):
    import os
    import sys
    root = os.path.join(os.getcwd(), "turing-sm75_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import b200lab
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"])
    if s["op"] == "attend":
        return b200lab.attn_fwd_kv8(s["q"], *cache, s["lens"], cu_seqlens_q=s["cu"], max_seqlen_q=s["most"], gate=s["g"])
    if s["op"] == "append":
        b200lab.kv8_append(s["k"], s["v"], *cache, s["lens"], cu_seqlens=s["cu"], max_seqlen=s["most"])
        return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return b200lab.kv8_read(*cache, s["cu"], s["longest"], s["total"], out_dtype=s["out_dtype"])


def _offsets(s, n):
    """Prefix sums of the tokens of a batch: given, or one token a sequence."""
    return torch.arange(n + 1, device="cuda") if s["cu"] is None else s["cu"].long()


def _places(cu, first, total):
    """The sequence and the position of every packed token; `first`: the position of each sequence's first one."""
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, first[b] + t - cu[b]


def _plain_read(s):
    P = s["block"]
    cu = s["cu"].long()
    b, pos = _places(cu, torch.zeros_like(cu[:-1]), s["total"])
    block, slot = s["table"].long()[b, pos // P], pos % P

    def values(cache, scale):
        x = cache.view(torch.uint8)[block, :, slot].view(E4M3).float()
        return (x * scale[block].unsqueeze(-1)).to(s["out_dtype"])

    return values(s["k_cache"], s["k_scale"]), values(s["v_cache"], s["v_scale"])


def _plain_append(s):
    P, total = s["block"], s["k"].shape[0]
    table, lens = s["table"].long(), s["lens"].long()
    cu = _offsets(s, lens.numel())
    start = lens - (cu[1:] - cu[:-1])
    b, pos = _places(cu, start, total)
    block, slot = table[b, pos // P], pos % P
    begun = table.gather(1, (start // P).unsqueeze(1)).squeeze(1)  # the block each sequence goes on in
    before = start % P                                             # and how many tokens it holds already
    kept = torch.arange(P, device="cuda") < before.unsqueeze(1)

    def write(x, cache, scale):
        x = x.float()
        a = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        a = torch.zeros_like(scale).index_reduce(0, block, a, "amax", include_self=True)
        m, e = torch.frexp(a)
        e = torch.where(m > 0.875, e - 8, e - 9)
        fits = _power(torch.where(a > 0, e, -MAX_E).clamp(-MAX_E, MAX_E))
        old = scale[begun]
        held = torch.where((before > 0).unsqueeze(1), torch.maximum(old, fits[begun]), fits[begun])
        scale[block] = fits[block]
        scale[begun] = held
        was = cache[begun]
        moved = (was.float() * (old / held)[:, :, None, None]).to(E4M3)
        codes = cache.view(torch.uint8)
        codes[begun] = torch.where(kept[:, None, :, None], moved.view(torch.uint8), was.view(torch.uint8))
        codes[block, :, slot] = (x / scale[block].unsqueeze(-1)).clamp(-448, 448).to(E4M3).view(torch.uint8)

    write(s["k"], s["k_cache"], s["k_scale"])
    write(s["v"], s["v_cache"], s["v_scale"])
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attend(s):
    P, D, Hq, Hkv, most = s["block"], s["D"], s["Hq"], s["Hkv"], s["most"]
    table, lens = s["table"].long(), s["lens"].long()
    B, S = table.shape[0], table.shape[1] * P
    total = s["q"].shape[0]
    cu = _offsets(s, B)
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    at = torch.where(i < new.unsqueeze(1), cu[:-1].unsqueeze(1) + i, 0)      # [B, most] packed token of each query
    limit = (lens - new).unsqueeze(1) + i + 1                                # [B, most] how many keys it sees
    j = torch.arange(S, device="cuda")

    def values(cache, scale):  # [B, Hkv, S, D], zeros behind each sequence's last token
        x = cache[table].float() * scale[table][..., None, None]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, S, D)
        return torch.where((j < lens.unsqueeze(1))[:, None, :, None], x, 0.0)

    q = s["q"][at].float().view(B, most, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = torch.matmul(q, values(s["k_cache"], s["k_scale"]).transpose(2, 3)) * (1.0 / math.sqrt(D))
    x = x.view(B, Hkv, Hq // Hkv, most, S)
    x = torch.where((j < limit.unsqueeze(2))[:, None, None], x, -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p.view(B, Hkv, -1, S), values(s["v_cache"], s["v_scale"]))
    o = o.view(B, Hkv, Hq // Hkv, most, D) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, Hq, D)
    b, pos = _places(cu, torch.zeros_like(lens), total)
    o = o[b, pos]
    if s["g"] is not None:
        o = o * torch.sigmoid(s["g"].float())
    return o.to(s["q"].dtype)


# ---- the definitions in 64 bits, one sequence after the other --------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    lens, new = _lengths(c)
    P, table = c["block"], s["table"].tolist()
    sides = (("k", s["k_cache"], s["k_scale"]), ("v", s["v_cache"], s["v_scale"]))

    def tokens(cache, scale, b, n):  # [n, Hkv, D]
        ids = torch.tensor(table[b][:-(-n // P)], device="cuda")
        x = cache[ids].double() * scale[ids].double()[:, :, None, None]
        return x.transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[:n]

    if c["op"] == "read":
        return tuple(torch.cat([tokens(cache, scale, b, n) for b, n in enumerate(lens)]) for _, cache, scale in sides)
    if c["op"] == "append":
        out = {}
        for name, cache, scale in sides:
            values, scales, t = cache.double(), scale.double(), 0
            for b, (n, m) in enumerate(zip(lens, new)):
                x = s[name][t:t + m].double()
                t += m
                for first in range((n - m) // P * P, n, P):
                    block = table[b][first // P]
                    lo, hi = max(first, n - m), min(first + P, n)
                    part = x[lo - (n - m):hi - (n - m)].transpose(0, 1)  # [Hkv, tokens, D]
                    big = part.abs().amax((1, 2))
                    e = torch.ceil(torch.log2(big.clamp_min(1e-300) / 448)).clamp(-MAX_E, MAX_E)
                    size = _power64(e)
                    size = torch.where(448 * size < big, 2 * size, size)  # log2 rounds
                    size = torch.where((448 * size / 2 >= big) & (e > -MAX_E), size / 2, size).clamp(2.0 ** -MAX_E, 2.0 ** MAX_E)
                    held = scales[block].clone()
                    if lo > first:
                        size = torch.maximum(size, held)
                        values[block, :, :lo - first] = _e4m3(values[block, :, :lo - first] * (held / size)[:, None, None])
                    values[block, :, lo - first:hi - first] = _e4m3(part / size[:, None, None])
                    scales[block] = size
            out[name], out[name + "_scale"] = values, scales
        return out
    rows, t = [], 0
    group = c["Hq"] // c["Hkv"]
    for b, (n, m) in enumerate(zip(lens, new)):
        K, V = (tokens(cache, scale, b, n) for _, cache, scale in sides)
        K, V = K.permute(1, 2, 0), V.transpose(0, 1)
        for i in range(m):
            seen = n - m + i + 1
            q = s["q"][t].double().view(c["Hkv"], group, c["D"])
            w = torch.softmax(q @ K[:, :, :seen] / math.sqrt(c["D"]), -1) @ V[:, :seen]
            w = w.reshape(c["Hq"], c["D"])
            if c["gate"]:
                w = w / (1 + torch.exp(-s["g"][t].double()))
            rows.append(w)
            t += 1
    return torch.stack(rows)


def _e4m3(x):
    """The nearest value of e4m3 (ties to the even code) of each of x, in 64 bits; what is larger than 448 becomes 448."""
    _, e = torch.frexp(x)
    step = _power64((e - 1).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)
