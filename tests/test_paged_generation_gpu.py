"""paged_sdpa by the kernels of few rows a sequence: pages that are none, masked
places and infinite values, which the tests of test_paged_gpu.py give to the
kernels of chunks, and a missing page in the middle of a divided tile."""
import functools

import pytest
import torch

import test_paged_gpu as full

pytestmark = pytest.mark.gpu
F16, F32 = full.F16, full.F32


class FewRows:
    """The package, its calls with max_q_len = 1 (which chooses kernels only)."""

    def __init__(self, pkg):
        self.pkg = pkg
        self.paged_sdpa = functools.partial(pkg.paged_sdpa, max_q_len=1)

    def __getattr__(self, name):
        return getattr(self.pkg, name)


@pytest.mark.parametrize("T", [F16, F32])
def test_pages_that_are_none(pkg, T):
    full.test_pages_that_are_none(FewRows(pkg), T)


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new,lens,page", [((60, 4), (100, 37), 16), ((300, 1), (700, 333), 64), ((9, 1), (3000, 33), 32)])
def test_masked_places_have_no_influence(pkg, T, new, lens, page):
    full.test_masked_places_have_no_influence(FewRows(pkg), T, new, lens, page)


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new,lens", [((3,), (300,)), ((150,), (400,)), ((5,), (9000,))])
def test_infinite_keys_and_queries(pkg, T, new, lens):
    full.test_infinite_keys_and_queries(FewRows(pkg), T, new, lens)


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("at", [0, 2500, 4999])  # the key on the missing page
@pytest.mark.parametrize("many", [False, True])  # few blocks: a share each; more: longer ones
def test_missing_page_in_one_share(pkg, T, page, at, many):
    new, lens = (1, 2, 1) + (1,) * (60 * many), (700, 5000, 90) + (1900,) * (60 * many)
    b = full.Batch(T, new, lens, 8, 2, 64, 64, page)
    ref = b.reference(True)
    q, kc, vc, table, starts, kv_lens = b.args()
    table[1, at // page] = b.pages
    o, stats = pkg.paged_sdpa(q, kc, vc, table, starts, kv_lens, scale=b.scale, max_q_len=2)
    # (tokens 1 and 2; the last key, 4999, is seen by token 2 alone, but lies in their tile)
    assert bool(torch.isnan(o[1:3]).all()) and bool(torch.isnan(stats[1:3]).all())
    keep = torch.ones(len(q), dtype=torch.bool)
    keep[1:3] = False
    full.check((o[keep.to(full.DEV)], stats[keep.to(full.DEV)]), [x[keep] for x in ref])
