"""paged_sdpa, fp16: many weak keys beside a strong one.

Key 0 has the score 17.5 (in units of one product, which fp32 holds) and value -1, the n - 1
others the score 0 and value 1: each of them has e^-17.5 = 2^-25.25 of the strong one's weight,
below half of the smallest fp16 number, and together W = (n - 1) 2^-25.25, so
o = (W - 1) / (W + 1).

Bounds.  The weight of the others is off by a relative 8 u, u = 2^-24 (the exponent, of size 26,
is rounded twice, exp2 once: 2 x 26 u ln 2, below 40 u W in all).  The sums of weights and of
products run in fp32 in chains of at most n / 16 additions (in generation n / 64, as four waves
share the keys) to a number below 2, which is off by u each time: that for o and as much for the sum.  fp16 weights may be off by 2^-25 of a
number, the largest of which is at least 2^7: n 2^-32.  The result is rounded to fp16: 2^-11."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# 512 tiles, so that none is divided: all sequences have the same pages
@pytest.mark.parametrize("heads", [1, 32], ids=["generation", "chunks"])  # rows of a sequence: up to 16, more
@pytest.mark.parametrize("D", [64, 128])
def test_weak_keys(pkg, heads, D):
    N, n, page = 512, 400000, 64
    pages = n // page
    k = torch.zeros((pages, 1, page, D), device=DEV, dtype=torch.float16)
    v = torch.ones((pages, 1, page, D), device=DEV, dtype=torch.float16)
    k[0, 0, 0, 3], v[0, 0, 0] = 5, -1
    q = torch.zeros((N, heads, D), device=DEV, dtype=torch.float16)
    q[..., 3] = 3.5
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.arange(pages, device=DEV, dtype=torch.int32).expand(N, pages)
    o, stats = pkg.paged_sdpa(q, k, v, table, i32(range(N + 1)), i32([n] * N), scale=1.0, max_q_len=1)
    u = 2.0 ** -24
    W = (n - 1) * math.exp(-17.5)
    want, lse = (W - 1) / (W + 1), 17.5 + math.log1p(W)
    chains = n / (64 if heads == 1 else 16) * u
    assert float((o.double() - want).abs().max()) <= 2 * (40 * u * W + chains) + n * 2.0 ** -32 + 2.0 ** -11
    assert float((stats.double() - lse).abs().max()) <= 40 * u * W + chains + 2 * u * lse
