"""CPU tests of the 8-bit key/value cache: the entries refuse malformed calls before anything is
launched, the binding checks its tensors, and the 64-bit implementation that the GPU tests compare
with agrees with torch's own e4m3."""
import ctypes

import numpy as np
import pytest
import torch

import b200lab
import kv8_ref

P16 = 16  # stands for an aligned device pointer; never dereferenced


def _append(**kw):
    a = dict(k=P16, kt=256, kh=128, v=P16, vt=256, vh=128, kc=P16, vc=P16, ks=P16, vs=P16, table=P16, lens=P16, cu=P16,
             max_seqlen=4, total=8, B=2, max_blocks=4, n_blocks=8, block=64, Hkv=2, D=128, dtype=b200lab.BF16)
    a.update(kw)
    return b200lab.lib().kv8_append_sm100(*a.values(), None)


def _read(**kw):
    a = dict(kc=P16, vc=P16, ks=P16, vs=P16, table=P16, cu=P16, max_seqlen=4, total=8, k=P16, v=P16, B=2, max_blocks=4,
             n_blocks=8, block=64, Hkv=2, D=128, dtype=b200lab.BF16)
    a.update(kw)
    return b200lab.lib().kv8_read_sm100(*a.values(), None)


def _attend(**kw):
    a = dict(q=P16, qt=512, qh=128, g=None, gt=0, gh=0, kc=P16, vc=P16, ks=P16, vs=P16, table=P16, lens=P16, cu=P16,
             max_seqlen=4, total=8, o=P16, B=2, max_blocks=4, n_blocks=8, block=64, Hq=4, Hkv=2, D=128,
             scale=0.1, causal=1, dtype=b200lab.BF16, ws=P16, ws_bytes=1 << 30)
    a.update(kw)
    return b200lab.lib().attn_fwd_sm100_kv8(*a.values(), None)


COMMON = [(dict(kc=None), b200lab.ERR_INVALID), (dict(vs=None), b200lab.ERR_INVALID), (dict(table=None), b200lab.ERR_INVALID),
          (dict(kc=24), b200lab.ERR_INVALID), (dict(B=0), b200lab.ERR_INVALID), (dict(max_blocks=0), b200lab.ERR_INVALID),
          (dict(n_blocks=0), b200lab.ERR_INVALID), (dict(Hkv=0), b200lab.ERR_INVALID), (dict(total=0), b200lab.ERR_INVALID),
          (dict(max_seqlen=0), b200lab.ERR_INVALID), (dict(dtype=7), b200lab.ERR_INVALID),
          (dict(block=48), b200lab.ERR_UNSUPPORTED), (dict(block=256), b200lab.ERR_UNSUPPORTED),
          (dict(D=96), b200lab.ERR_UNSUPPORTED), (dict(max_blocks=1 << 26), b200lab.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(k=None), b200lab.ERR_INVALID), (dict(lens=None), b200lab.ERR_INVALID), (dict(k=24), b200lab.ERR_INVALID),
    (dict(kt=257), b200lab.ERR_INVALID), (dict(vh=-128), b200lab.ERR_INVALID),
    (dict(cu=None), b200lab.ERR_INVALID), (dict(cu=None, max_seqlen=1), b200lab.ERR_INVALID),
    (dict(B=1 << 28, max_blocks=8, max_seqlen=512, total=1 << 30), b200lab.ERR_UNSUPPORTED)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code


@pytest.mark.parametrize("kw,code", COMMON + [(dict(k=None), b200lab.ERR_INVALID), (dict(cu=None), b200lab.ERR_INVALID),
                                              (dict(v=24), b200lab.ERR_INVALID)])
def test_read_refusals(kw, code):
    assert _read(**kw) == code


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(q=None), b200lab.ERR_INVALID), (dict(o=None), b200lab.ERR_INVALID), (dict(lens=None), b200lab.ERR_INVALID),
    (dict(q=24), b200lab.ERR_INVALID), (dict(o=24), b200lab.ERR_INVALID), (dict(qt=516), b200lab.ERR_INVALID),
    (dict(Hq=3), b200lab.ERR_INVALID), (dict(Hq=0), b200lab.ERR_INVALID), (dict(scale=0.0), b200lab.ERR_INVALID),
    (dict(scale=float("nan")), b200lab.ERR_INVALID), (dict(scale=float("inf")), b200lab.ERR_INVALID),
    (dict(causal=2), b200lab.ERR_INVALID), (dict(dtype=b200lab.F32), b200lab.ERR_INVALID),
    (dict(g=P16, gt=-1), b200lab.ERR_INVALID),
    (dict(cu=None), b200lab.ERR_INVALID), (dict(ws=None), b200lab.ERR_WORKSPACE), (dict(ws_bytes=1000), b200lab.ERR_WORKSPACE)])
def test_attend_refusals(kw, code):
    assert _attend(**kw) == code


def test_workspace_size():
    f = b200lab.attn_fwd_kv8_workspace_bytes
    # parts of 8 or 16 rows, two a CTA, whatever the batch and the query counts
    assert 0 < f(32, 8, 1, 128) == f(8, 8, 8, 128) and 0 < f(32, 8, 4, 128) == f(32, 8, 8, 128) == f(32, 8, 1000, 128)
    assert 0 < f(24, 4, 1, 256) == f(24, 4, 2, 256) == f(24, 4, 100, 256)
    assert f(3, 2, 1, 128) == 0 and f(4, 2, 1, 96) == 0 and f(4, 2, 0, 128) == 0


def test_binding_checks():
    c = torch.zeros((4, 2, 16, 64), dtype=torch.float8_e4m3fn)
    s = torch.ones((4, 2))
    t = torch.zeros((1, 4), dtype=torch.int32)
    n = torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        b200lab.kv8_append(x, x, c, c, s, s, t, n)
    with pytest.raises(ValueError, match="CUDA"):
        b200lab.kv8_read(c, c, s, s, t, torch.zeros(2, dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        b200lab.attn_fwd_kv8(x, c, c, s, s, t, n)


def test_reference_codes_match_torch():
    codes = np.arange(256, dtype=np.uint8)
    mine = kv8_ref.TABLE[codes]
    theirs = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(mine, theirs, equal_nan=True)
    x = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[x.abs() <= 448]
    assert np.array_equal(kv8_ref.round_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    for a, s in [(0.0, 2.0 ** -40), (448.0, 1.0), (448.1, 2.0), (1.0, 2.0 ** -8), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7),
                 (1e30, 2.0 ** 40)]:
        assert kv8_ref.scale_for(a) == s
