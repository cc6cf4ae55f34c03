"""Attention with weights where sequences are cut into parts that a second launch joins (tmac_attention_decode_weighted), with
the most query heads a kv head: every cache type, few and many parts a sequence, held to budget.attend64's bounds."""
import numpy as np
import pytest

from budget import TYPES
from test_gpu_budget import NAMES, no_fault, run_weighted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", TYPES, ids=[NAMES[t] for t in TYPES])
@pytest.mark.parametrize("n,nkv,group,longest", [(2, 1, 16, 12000), (1, 3, 11, 9001), (1, 1, 9, 20000),  # a head a workgroup joins
                                                 (40, 1, 16, 6000), (14, 3, 11, 5003), (30, 2, 8, 4500),  # a head a wave
                                                 (200, 1, 11, 6001), (120, 2, 16, 4999)])  # more than 2/3 of a CU each
def test_parts_with_many_heads(ctx, dt, n, nkv, group, longest):
    rng = np.random.default_rng(n + group)
    lens = rng.integers(0, 41, n)
    lens[n - 1] = longest
    if n > 2:
        lens[0], lens[n // 2] = longest - 17, longest // 2
    run_weighted(ctx, dt, nkv * group, nkv, lens, 2300 + n, max_len=longest)
    run_weighted(ctx, dt, nkv * group, nkv, lens, 2301 + n, max_len=longest, weights=False)
    run_weighted(ctx, dt, nkv * group, nkv, lens, 2302 + n, max_len=longest, in_place=True, stride=longest + 5)
    no_fault(ctx)
