"""Queries of very different size beside one another: every row of a call is
its own, whatever its neighbours hold.

The tolerance is ``formula``'s.  bf16 queries are held in fp16 times a power of
two that brings a row's largest value to [2^13, 2^14): what is 2^27 times
smaller than that leaves fp16's normal range and is off by half its smallest
step, 2^-25, which is 2^-38 of the row's largest value.  That adds up to
2^-38 D max|q| max|k| to a score, a small part of the (D + 4) 2^-24 of the sum
of |q||k| that the bound has already for these normal queries.
"""
import pytest
import torch

from gsq_b200.runtime.kernels import cached_attention
from test_gpu_cached_attention import DEV, check, filled, formula, i32, queries, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,group,cap", [(2, 6, 400), (12, 6, 400), (50, 6, 400), (9, 8, 8300)])  # tokens, units, row blocks
@pytest.mark.parametrize("big", [2.0 ** 30, 2.0 ** 40, 1e30])
def test_one_large_row_leaves_its_neighbours_alone(dim, n, group, cap, big):
    """Rows of ordinary size beside a few very large ones (which attend to one position each)."""
    start = [cap - n]
    cache = filled(1, 2, cap, dim, "int8", 51)
    q = queries(1, n, 2 * group, dim, torch.bfloat16, 52)
    rows = q.view(-1, dim)
    rows[3::29] *= big
    see = visible(1, n, cap, start, None, None)
    want, bound = formula(q, cache, see)
    bound = torch.where(torch.isfinite(bound), bound, torch.full_like(bound, 1e30))  # a large row's own scores
    check(cached_attention(q, cache, i32(*start)), want, bound)


@pytest.mark.parametrize("n,group", [(2, 6), (50, 6)])
def test_each_row_has_its_own_size(n, group):
    """Sizes from 2^-60 to 2^60, with a scale under which the middle ones' scores are of order 1."""
    cap, dim = 300, 128
    cache = filled(1, 1, cap, dim, "fp8", 53)
    q = queries(1, n, group, dim, torch.float32, 54)
    mixed = torch.randperm(n * group, generator=torch.Generator().manual_seed(57)).to(DEV)
    size = torch.exp2(torch.linspace(-60, 60, n * group, device=DEV)[mixed]).view(1, n, group, 1)
    q = (q * size).to(torch.bfloat16)
    see = visible(1, n, cap, [cap - n], None, None)
    want, bound = formula(q, cache, see)
    bound = torch.where(torch.isfinite(bound), bound, torch.full_like(bound, 1e30))
    check(cached_attention(q, cache, i32(cap - n)), want, bound)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_row_that_is_not_finite_is_lost_alone(value):
    cap, dim, n, group = 300, 128, 50, 6
    cache = filled(1, 1, cap, dim, "int8", 55)
    q = queries(1, n, group, dim, torch.bfloat16, 56)
    want = cached_attention(q, cache, i32(cap - n))
    q.view(-1, dim)[40, 7] = value
    got = cached_attention(q, cache, i32(cap - n)).view(-1, dim)
    others = torch.arange(n * group, device=DEV) != 40
    assert torch.equal(got[others], want.view(-1, dim)[others])
    assert torch.isnan(got[40]).all()
