"""GPU tests of calls at the edge of what the 8-bit key/value cache documents."""
import numpy as np
import pytest
import torch

import b200lab
import kv8_ref
from test_kv8_gpu import UNIT, Setup, Wide, _normal

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
