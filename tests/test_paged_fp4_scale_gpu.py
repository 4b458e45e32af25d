"""paged_sdpa_fp4 where the scale is 0 or so small that its product with a row's power of two
is below every fp32 number, against the definition in 64 bits (bounds: test_paged_fp4_gpu.py)."""
import pytest
import torch

from test_paged_fp4_gpu import F16, F32, NAN, Fp4Batch
from test_paged_gpu import check

pytestmark = pytest.mark.gpu

ORDINARY = (0.0, 2.0 ** -60, 1e-30, 2.0 ** -140, 1.0)
CASES = [(F32, 0.0, ORDINARY + (1e30,)), (F32, 1e-12, ORDINARY), (F32, -1e-20, ORDINARY), (F32, 1e-30, ORDINARY),
         (F32, 2.0 ** -140, ORDINARY), (F16, 0.0, (0.0, 2.0 ** -20, 1.0)), (F16, 1e-12, (0.0, 1.0))]


@pytest.mark.parametrize("T,scale,sizes", CASES, ids=lambda x: str(x).replace("torch.", "")[:20])
@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("causal", [True, False])
def test_small_scales(pkg, T, scale, sizes, hint, causal):
    """Rows of zeros and of queries of very different size, in lengths that end inside a block of keys:
    all keys weigh alike, as the scores' differences are far below fp32's."""
    b = Fp4Batch(T, (3, 140, 1), (91, 300, 5), 4, 2, 64, 64, 16)
    for i, size in enumerate(sizes):
        b.q[i::len(sizes)] = (b.q[i::len(sizes)].double() * size).to(T)
    b.scale = scale
    check(pkg.paged_sdpa_fp4(*b.args(), scale=scale, causal_mask=causal, max_q_len=hint), b.reference(causal))


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
def test_a_scale_that_is_none(pkg, T, hint):
    b = Fp4Batch(T, (3, 140), (91, 300), 4, 2, 64, 64, 16)
    o, stats = pkg.paged_sdpa_fp4(*b.args(), scale=NAN, max_q_len=hint)
    assert bool(torch.isnan(o).all()) and bool(torch.isnan(stats).all())
