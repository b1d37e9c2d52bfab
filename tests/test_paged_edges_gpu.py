"""GPU: edges of the paged K/V cache operators: maxima that rise inside an item's
last block, captured loop bodies, empty steps, infinite scores, idle requests, long
prompts.  Tolerances as derived in test_paged_gpu."""
import math

import pytest
import torch

from test_paged_gpu import BF, FP, Paged, _i32, _no_device_error

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from std_b200 import ops as _ops

    assert torch.cuda.is_available()
    return _ops


def set_keys(x, b, keys):
    """Request b's keys of a Paged become `keys` [L, Hkv, D]."""
    x.keys[b] = (keys, x.keys[b][1])
    for i in range(-(-x.kv[b] // x.page)):
        rows = slice(i * x.page, min(x.kv[b], (i + 1) * x.page))
        x.k[x.table[b, i].item(), :, :rows.stop - rows.start] = keys[rows].permute(1, 0, 2)


# ------------------------------------------------------------------ running maxima
@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF)])
@pytest.mark.parametrize("tail", [0, 1, 15, 64, 65, 80, 127])
def test_maximum_rises_in_every_half_block(ops, D, dtype, tail):
    """Scores that jump by more than 2^8 from each 64 keys to the next, the last ones of
    an item included: O is rescaled in every half of every block, behind which no
    next score stands at an item's end.  Items of all forms follow one another in a CTA."""
    pairs = [(256 + tail, 1), (128 + tail, 19), (300 + tail, 3), (tail, 36), (512 + tail, 72), (700 + tail, 40)]
    pairs = pairs * 8 + [(2000 + tail, 25)] * 3
    x = Paged(pairs, 14, 2, D, 64, dtype, seed=tail)
    x.q = x.q.abs().clamp(0.5, 2)
    for b, (past, n) in enumerate(pairs):
        L = x.kv[b]
        half = torch.arange(L, device="cuda")[:, None, None] // 64
        set_keys(x, b, ((half + 1) * x.keys[b][0].float().abs().clamp(0.8, 1.2)).to(dtype))
    lse = torch.empty(x.q.shape[:2], device="cuda")
    for causal in (True, False):
        out = x.call(ops, causal, lse=lse)
        x.check(out, lse, causal)
        assert torch.equal(x.call(ops, causal), out)
    _no_device_error(ops)
