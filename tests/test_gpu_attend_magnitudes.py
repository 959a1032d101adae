"""Attention over the 8-bit cache where pages, queries or scores lie many magnitudes apart, against the plain 64-bit form."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_gpu_kv_cache import _cache, _np, dev  # noqa: F401

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
@pytest.mark.parametrize("qsize", (1e34, 3e37, 1e-30))
def test_queries_near_the_ends_of_the_type(dev, dtype, qsize):  # noqa: F811
    gen = torch.Generator().manual_seed(12)
    k, v = (torch.randn(100, 1, 64, generator=gen).to(dev, dtype) for _ in range(2))
    cache, kr, vr = _stored(dev, k, v)
    q = (torch.randn(1, 4, 64, generator=gen).clamp(-2, 2) * qsize).to(dev, dtype)
    scale = 0.05 / qsize
    assert_own_size(cache.attend(q, scale=scale), q, kr, vr, scale)
