"""Attention over the cache where its pages are cut into units of several for the warps, whose parts a second kernel joins,
against the plain form in 64 bits over what ``read`` gives, within float32's bound on each row's own sums and the
16-bit types' share of sum p |v|."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attend_magnitudes import SHARE
from tests.test_gpu_kv_cache import TYPES, _cache, dev  # noqa: F401

pytestmark = pytest.mark.gpu

WARPS = {32: 2368, 64: 2368, 96: 1776, 128: 1776}  # of the first kernel at most


def _long_cache(dev, lengths, heads, width, dtype, layers=1):  # noqa: F811
    pages = sum(-(-n // 64) for n in lengths)
    cache = _cache(dev, requests=len(lengths), pages=pages + 5, kv_heads=heads, head_width=width, max_blocks=-(-max(lengths) // 64),
                   layers=layers)
    cache.key_pages.view(torch.uint8).fill_(0x7f)  # NaN, what earlier requests left
    cache.value_pages.view(torch.uint8).fill_(0x7f)
    gen = torch.Generator(device=dev).manual_seed(width + heads)
    plan = cache.resize(lengths, tokens=sum(lengths))
    x = torch.randn(2, sum(lengths), heads, width, generator=gen, device=dev).to(dtype)
    cache.store(x[0], x[1], plan, layer=layers - 1)
    return cache, cache.read(plan.slots, layer=layers - 1, dtype=torch.float32)


def _plain(q, k, v, lengths, scale):
    q, group = q.double(), q.shape[1] // k.shape[1]
    out, bound, first = torch.zeros_like(q), torch.zeros_like(q), 0
    for b, n in enumerate(lengths):
        for h in range(q.shape[1]) if n else ():
            kk, vv = k[first:first + n, h // group].double(), v[first:first + n, h // group].double()
            p = torch.softmax(scale * (kk @ q[b, h]), 0)
            out[b, h] = p @ vv
            reach = abs(scale) * (kk.abs() @ q[b, h].abs()) + 1
            bound[b, h] = 2.0**-20 * ((p * reach) @ (vv - out[b, h]).abs() + p @ vv.abs())
        first += n
    return out, bound


def _share(q, k, v, lengths, scale, dtype):
    return SHARE[dtype] * _plain(q, k, v.abs(), lengths, scale)[0] if SHARE[dtype] else 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", (32, 64, 96, 128))
@pytest.mark.parametrize("heads,group", [(8, 4), (3, 9), (2, 17)])  # one, two and three turns of eight query heads
def test_units_of_several_pages(dev, dtype, width, heads, group):  # noqa: F811
    pairs = heads * -(-group // 8)
    pages = 5 * WARPS[width] // pairs  # some five pages to a warp: units of three, and small ones taken as warps get free
    few = [0, 1, 64, 65, 640, 0, 1300, 200]  # in one unit, in a few (joined by threads)
    long = [int(64 * pages * 0.55), int(64 * pages * 0.4)]  # in many (joined by warps)
    lengths = [long[0], *few[:4], long[1], *few[4:]]
    cache, (k, v) = _long_cache(dev, lengths, heads, width, dtype, layers=2)
    q = torch.randn(len(lengths), heads * group, width, generator=torch.Generator().manual_seed(3)).to(dev, dtype)
    scale = 2 * width**-0.5
    got = cache.attend(q, layer=1, scale=scale)
    want, bound = _plain(q, k, v, lengths, scale)
    over = (got.double() - want).abs() / (bound + _share(q, k, v, lengths, scale, dtype) + 1e-38)
    assert torch.isfinite(got).all() and float(over.max()) <= 1, float(over.max())
    for _ in range(3):  # which warp takes which unit does not show
        assert torch.equal(cache.attend(q, layer=1, scale=scale), got)
    cache.validate_invariants()


def test_a_join_replays_in_a_graph(dev):  # noqa: F811
    lengths = [64 * 1500, 64 * 700 + 3, 100]
    cache, _ = _long_cache(dev, lengths, 4, 128, torch.bfloat16)
    q = torch.randn(3, 16, 128, device=dev, dtype=torch.bfloat16)
    want = cache.attend(q).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
        q2 = torch.randn_like(q)
        want2 = cache.attend(q2)
        q.copy_(q2)
        graph.replay()
        assert torch.equal(out, want2)
        want = want2
