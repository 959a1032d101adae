"""Attention over the 8-bit cache where pages, queries or scores lie many magnitudes apart, against the plain 64-bit form."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_gpu_kv_cache import TYPES, _cache, _np, dev  # noqa: F401

pytestmark = pytest.mark.gpu

# of sum p |v|: weights held in f16 and the result's rounding
SHARE = {torch.float32: 0.0, torch.bfloat16: 2.0**-7, torch.float16: 2.0**-10}


def _stored(dev, k, v):  # noqa: F811
    """One request's tokens [n, heads, width] in a cache of their own, and the rows it holds."""
    n, heads, width = k.shape
    pages = O.pages_of(n)
    cache = _cache(dev, requests=1, pages=pages, kv_heads=heads, head_width=width, max_blocks=pages)
    ref, ks, vs = O.Pages(1, pages, pages), O.Store(heads, width), O.Store(heads, width)
    cache.store(k, v, cache.resize([n], tokens=n))
    want = ref.resize([n])
    ks.put(_np(k), want[3])
    vs.put(_np(v), want[3])
    return cache, ks.rows(want[1]), vs.rows(want[1])


def assert_own_size(got, q, k, v, scale):
    """Each output within its own sums' float32 bound, and for the 16-bit types its share of sum p |v|."""
    want, bound = O.attend_with_bound(_np(q), [k], [v], scale)
    bound = bound + SHARE[got.dtype] * O.attend(_np(q), [k], [np.abs(v)], scale) + np.finfo(np.float32).tiny
    over = np.abs(_np(got) - want) / bound
    assert torch.isfinite(got).all() and (over <= 1).all(), float(over.max())


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("long", (False, True))
@pytest.mark.parametrize("sizes", [
    (2.0**60, 1.0, 2.0**-56), (1e30, 1e10, 1e-10), (1e-15, 1.0, 1e15, 1e30), (1e30, 0.0, 1e-10), (0.0, 1e-18, 1e30, 1.0),
])
def test_pages_whose_values_lie_far_apart(dev, dtype, long, sizes):  # noqa: F811
    """Falling and rising from page to page, all of like weight; and with the weight on ever later ones.  ``long``: tables too
    long for a block to each pair."""
    pages = len(sizes) * (17 if long else 1)
    gen = torch.Generator().manual_seed(11)
    v = torch.randn(64 * pages, 1, 32, generator=gen)
    v *= torch.tensor(sizes)[torch.arange(64 * pages) // 64 % len(sizes)][:, None, None]
    k = torch.randn(64 * pages, 1, 32, generator=gen) * 0.1
    q = torch.randn(1, 4, 32, generator=gen).to(dev, dtype) * 0.5
    q[..., 0] = 1.0
    for grow in (0.0, 32.0, -32.0):
        k[:, 0, 0] = grow * (torch.arange(64 * pages) // 64)
        cache, kr, vr = _stored(dev, k.to(dev, dtype), v.to(dev, dtype))
        assert_own_size(cache.attend(q, scale=1.0), q, kr, vr, 1.0)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("qsize", (1e34, 3e37, 1e-30))
def test_queries_near_the_ends_of_the_type(dev, dtype, qsize):  # noqa: F811
    gen = torch.Generator().manual_seed(12)
    k, v = (torch.randn(100, 1, 64, generator=gen).to(dev, dtype) for _ in range(2))
    cache, kr, vr = _stored(dev, k, v)
    q = (torch.randn(1, 4, 64, generator=gen).clamp(-2, 2) * qsize).to(dev, dtype)
    scale = 0.05 / qsize
    assert_own_size(cache.attend(q, scale=scale), q, kr, vr, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_values_of_the_type(dev, dtype):  # noqa: F811
    top = {torch.float16: 57344.0}.get(dtype, 448 * 2.0**119)  # exact in e4m3
    k = torch.zeros(150, 1, 32, device=dev, dtype=dtype)
    cache, kr, vr = _stored(dev, k, torch.full_like(k, -top))
    got = cache.attend(torch.ones(1, 2, 32, device=dev, dtype=dtype))
    torch.testing.assert_close(got.double(), torch.full_like(got, -top).double(), rtol=max(SHARE[dtype], 2.0**-19), atol=0.0)
