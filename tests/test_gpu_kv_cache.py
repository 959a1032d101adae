"""The paged 8-bit K/V cache (PagedKVCache) against its plain 64-bit form: block
tables, slot maps and the free stack exactly, codes and scales exactly, attention
within the rounding of its types.

Tolerance of an attention output o = sum p v / sum p, with |v| <= vmax and scores up to smax:
* 16-bit types, u the type's unit roundoff (2^-8 bfloat16, 2^-11 float16): the result is rounded once (u |o|) and a
  probability may be rounded once more, to the type or finer, which moves the mean by at most u vmax;
* float32: operands in two halves keep 22 bits, so a score is off by 2^-20 of
  sum |q k| <= width * qmax * kmax * scale, a probability by that and 2^-21, the mean by twice the same times vmax.
The float32 term is added to the 16-bit ones."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
TYPES = (torch.float32, torch.bfloat16, torch.float16)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _cache(dev, **kw):
    from copy_on_write_sdm_b200 import PagedKVCache

    return PagedKVCache.allocate(device=dev, **kw)


def _np(t):
    return t.detach().double().cpu().numpy()


def assert_attention(got, want, *, q, k, v, scale):
    u = ROUNDOFF[got.dtype]
    v = v[np.isfinite(v)]
    vmax = float(np.abs(v).max()) if v.size else 0.0
    reach = q.shape[-1] * float(np.abs(q).max()) * float(np.abs(k[np.isfinite(k)]).max(initial=0.0)) * abs(scale)
    atol = u * vmax + 2 * (2.0**-20 * reach + 2.0**-21) * vmax
    np.testing.assert_allclose(_np(got), want, atol=atol + 1e-30, rtol=u)


# ---- pages


def assert_pages(cache, ref, plan, want):
    starts, slots, positions, pieces = want
    np.testing.assert_array_equal(plan.starts.cpu().numpy(), starts)
    n = len(slots)
    np.testing.assert_array_equal(plan.slots.cpu().numpy()[:n], slots)
    np.testing.assert_array_equal(plan.positions.cpu().numpy()[:n], positions)
    assert bool((plan.slots[n:] == -1).all()) and bool((plan.positions[n:] == -1).all())
    assert plan.buffer[:2].tolist() == [len(pieces), n]
    np.testing.assert_array_equal(plan.pieces.cpu().numpy()[:len(pieces)], np.asarray(pieces, np.int64).reshape(-1, 4))
    np.testing.assert_array_equal(cache.block_tables.cpu().numpy(), ref.tables)
    np.testing.assert_array_equal(cache.lengths.cpu().numpy(), ref.lengths)
    count = int(cache.free_count)
    assert cache.free_pages[:count].tolist() == ref.free
    cache.validate_invariants()


@pytest.mark.parametrize("requests,max_blocks,pages,seed", [
    (1, 1, 1, 0), (1, 40, 40, 1), (5, 3, 9, 2), (33, 7, 120, 3), (700, 12, 3000, 4), (2049, 3, 4000, 5),
])
def test_resize_follows_the_plain_form(dev, requests, max_blocks, pages, seed):
    rng = np.random.default_rng(seed)
    cache = _cache(dev, requests=requests, pages=pages, kv_heads=1, head_width=32, max_blocks=max_blocks)
    ref = O.Pages(requests, pages, max_blocks)
    most = max_blocks * O.PAGE
    for step in range(12):
        cur = ref.lengths.copy()
        how = step % 4
        if how == 0:  # all kinds of moves in one call
            target = rng.integers(0, most + 1, requests)
        elif how == 1:  # the next token
            target = np.minimum(cur + 1, most)
        elif how == 2:  # some finish, some are cut
            target = np.where(rng.random(requests) < 0.5, 0, cur - rng.integers(0, 1 + cur))
        else:
            target = np.minimum(cur + rng.integers(0, 130, requests), most)
        while sum(O.pages_of(int(t)) for t in target) > pages:
            target = np.where(rng.random(requests) < 0.3, np.minimum(target, cur) // 2, target)
        new = int(np.maximum(target - cur, 0).sum())
        plan = cache.resize(torch.tensor(target, dtype=torch.int32, device=dev), tokens=new + (step % 3) * 5)
        assert_pages(cache, ref, plan, ref.resize(target))


def test_resize_takes_host_targets_and_no_tokens(dev):
    cache = _cache(dev, requests=3, pages=4, kv_heads=1, head_width=32, max_blocks=2)
    ref = O.Pages(3, 4, 2)
    for target in ([64, 0, 65], [64, 0, 65], [0, 0, 0]):
        new = sum(max(t - int(c), 0) for t, c in zip(target, ref.lengths))
        assert_pages(cache, ref, cache.resize(target, tokens=new), ref.resize(target))


@pytest.mark.parametrize("target,tokens,bit", [
    ([65, 65, 64], 300, "no free page"), ([-1, 0, 0], 300, "outside"), ([129, 0, 0], 300, "outside"),
    ([64, 64, 0], 124, "more tokens"),
])
def test_a_resize_that_does_not_fit_changes_nothing(dev, target, tokens, bit):
    cache = _cache(dev, requests=3, pages=4, kv_heads=1, head_width=32, max_blocks=2)
    cache.resize([3, 0, 70], tokens=73)
    before = [t.clone() for t in (cache.block_tables, cache.lengths, cache.free_pages, cache.free_count)]
    if bit == "no free page":
        target = [128, 65, 70]
    plan = cache.resize(target, tokens=tokens)
    for a, b in zip(before, (cache.block_tables, cache.lengths, cache.free_pages, cache.free_count)):
        assert torch.equal(a, b)
    assert plan.buffer[0] == 0 and bool((plan.slots == -1).all()) and bool((plan.starts == 0).all())
    with pytest.raises(RuntimeError, match=bit):
        cache.validate_invariants()
    cache.status_word.zero_()
    cache.resize([0, 0, 0], tokens=0)  # and the cache goes on
    cache.validate_invariants()


def test_pages_freed_and_taken_in_one_full_pool(dev):
    cache = _cache(dev, requests=2, pages=3, kv_heads=1, head_width=32, max_blocks=3)
    ref = O.Pages(2, 3, 3)
    for target in ([192, 0], [0, 192], [100, 60], [30, 128]):
        new = sum(max(t - int(c), 0) for t, c in zip(target, ref.lengths))
        assert_pages(cache, ref, cache.resize(target, tokens=new), ref.resize(target))


def test_largest_number_of_requests(dev):
    requests = 8192
    cache = _cache(dev, requests=requests, pages=requests, kv_heads=1, head_width=32, max_blocks=1)
    ref = O.Pages(requests, requests, 1)
    target = np.random.default_rng(0).integers(0, 3, requests)
    assert_pages(cache, ref, cache.resize(torch.tensor(target, dtype=torch.int32, device=dev), tokens=int(target.sum())),
                 ref.resize(target))


# ---- store and read


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,heads", [(32, 1), (64, 3), (96, 2), (128, 5)])
def test_store_is_exact(dev, dtype, width, heads):
    rng = np.random.default_rng(width + heads)
    requests, blocks = 5, 4
    cache = _cache(dev, requests=requests, pages=requests * blocks, kv_heads=heads, head_width=width, max_blocks=blocks, layers=2)
    ref = O.Pages(requests, requests * blocks, blocks)
    stores = [O.Store(heads, width), O.Store(heads, width)]
    length = np.zeros(requests, np.int64)
    for grow in ([1, 0, 64, 63, 130], [1, 65, 0, 1, 2], [62, 3, 1, 64, 100], [1, 1, 1, 1, 1]):
        length = length + grow
        want = ref.resize(length)
        plan = cache.resize(torch.tensor(length, dtype=torch.int32, device=dev), tokens=sum(grow))
        # magnitudes from far below to far above what the page holds
        size = 2.0 ** rng.integers(-12, 7, (sum(grow), heads, 1))
        k = torch.tensor(rng.standard_normal((sum(grow), heads, width)) * size, device=dev).to(dtype)
        v = torch.tensor(rng.standard_normal((sum(grow), heads, width)) * size[::-1].copy(), device=dev).to(dtype)
        for _ in range(2):  # storing a plan again writes the same
            cache.store(k, v, plan, layer=1)
        stores[0].put(_np(k), want[3])
        stores[1].put(_np(v), want[3])
        live = [s for b in range(requests) for p in range(length[b]) for s in [int(ref.tables[b, p // 64]) * 64 + p % 64]]
        got = cache.read(torch.tensor(live, dtype=torch.int32, device=dev), layer=1, dtype=torch.float32)
        for g, s in zip(got, stores):
            np.testing.assert_array_equal(_np(g), s.rows(live))
        for scales, s in zip((cache.key_scales, cache.value_scales), stores):
            for page, value in s.scales.items():
                np.testing.assert_array_equal(_np(scales[1, page]), value)
    assert not cache.key_pages[0].view(torch.uint8).any()  # the other layer


def test_scales_at_the_ends(dev):
    """Exactly 448 * 2^e, the next value above it, zeros, the smallest and largest magnitudes, infinities and NaN."""
    rows = [448.0, float(np.nextafter(np.float32(448), np.float32(1e9))), 0.0, 1e-38, 3e38, 2.0**-58, float("inf"), float("nan")]
    cache = _cache(dev, requests=len(rows), pages=len(rows), kv_heads=1, head_width=32, max_blocks=1)
    ref = O.Pages(len(rows), len(rows), 1)
    x = torch.zeros(len(rows), 1, 32, device=dev)
    x[:, 0, 3] = torch.tensor(rows)
    x[6:, 0, 4] = 5.0
    cache.store(x, -x, cache.resize([1] * len(rows), tokens=len(rows)))
    want = ref.resize([1] * len(rows))
    k, v = O.Store(1, 32), O.Store(1, 32)
    k.put(_np(x), want[3])
    v.put(_np(-x), want[3])
    got = cache.read(torch.tensor(want[1], dtype=torch.int32, device=dev), dtype=torch.float32)
    np.testing.assert_array_equal(_np(got[0]), k.rows(want[1]))
    np.testing.assert_array_equal(_np(got[1]), v.rows(want[1]))


def test_store_reads_strided_projections(dev):
    """Keys and values as views of one fused projection, as unaligned views and transposed."""
    cache = _cache(dev, requests=2, pages=8, kv_heads=2, head_width=64, max_blocks=4)
    plan = cache.resize([70, 5], tokens=75)
    fused = torch.randn(75, 3, 2, 64, device=dev, dtype=torch.bfloat16)
    off = torch.randn(75 * 128 + 1, device=dev, dtype=torch.bfloat16)[1:].view(75, 2, 64)
    turned = torch.randn(2, 75, 64, device=dev, dtype=torch.bfloat16).transpose(0, 1)
    for k, v in ((fused[:, 1], fused[:, 2]), (off, turned), (turned, off)):
        cache.store(k, v, plan)
        got = cache.read(plan.slots)
        cache.store(k.contiguous(), v.contiguous(), plan)
        want = cache.read(plan.slots)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_read_of_no_slot_is_zero(dev):
    cache = _cache(dev, requests=1, pages=2, kv_heads=1, head_width=32, max_blocks=2)
    plan = cache.resize([2], tokens=2)
    x = torch.ones(2, 1, 32, device=dev)
    cache.store(x, x, plan)
    k, v = cache.read(torch.tensor([-1, int(plan.slots[0]), 128], dtype=torch.int32, device=dev), dtype=torch.float32)
    for t in (k, v):
        assert t[0].eq(0).all() and t[1].eq(1).all() and t[2].eq(0).all()
    assert cache.read(plan.slots[:0])[0].shape == (0, 1, 32)


# ---- attend


def _filled(dev, lengths, heads, width, dtype, seed, extra_pages=0, layers=1, layer=0):
    rng = np.random.default_rng(seed)
    blocks = max(1, max(O.pages_of(n) for n in lengths))
    pages = sum(O.pages_of(n) for n in lengths) + extra_pages
    cache = _cache(dev, requests=len(lengths), pages=pages, kv_heads=heads, head_width=width, max_blocks=blocks, layers=layers)
    # what earlier requests left: NaN codes in every place
    cache.key_pages.view(torch.uint8).fill_(0x7f)
    cache.value_pages.view(torch.uint8).fill_(0x7f)
    half = [n // 2 for n in lengths]
    ref = O.Pages(len(lengths), pages, blocks)
    k, v = O.Store(heads, width), O.Store(heads, width)
    for target in (half, lengths):
        new = sum(target) - int(ref.lengths.sum())
        plan = cache.resize(target, tokens=new)
        want = ref.resize(target)
        x = torch.tensor(rng.standard_normal((2, new, heads, width)), device=dev).to(dtype)
        if new:
            cache.store(x[0], x[1], plan, layer=layer)
        k.put(_np(x[0]), want[3])
        v.put(_np(x[1]), want[3])
    rows = [[s for p in range(n) for s in [int(ref.tables[b, p // 64]) * 64 + p % 64]] for b, n in enumerate(lengths)]
    return cache, [k.rows(r) for r in rows], [v.rows(r) for r in rows]


CASES = [
    ([1], 1, 1, 32), ([0], 2, 2, 64), ([64], 1, 4, 128), ([65, 63, 0, 1, 64, 200], 2, 3, 96),
    ([300, 17], 1, 8, 128), ([5, 900], 3, 7, 64), ([128, 129], 2, 9, 32), ([2, 70], 1, 17, 128), ([513] * 40, 4, 1, 32),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group,width", CASES)
def test_attend_matches_the_plain_form(dev, dtype, lengths, heads, group, width):
    cache, k, v = _filled(dev, lengths, heads, width, dtype, len(lengths) + group)
    q = torch.randn(len(lengths), heads * group, width, generator=torch.Generator().manual_seed(1)).to(dev, dtype)
    for scale in (None, 0.7):
        s = width**-0.5 if scale is None else scale
        want = O.attend(_np(q), k, v, s)
        for _ in range(2):  # the workspace is left ready
            got = cache.attend(q, scale=scale)
            assert got.dtype == dtype and got.is_contiguous()
            assert_attention(got, want, q=_np(q), k=np.concatenate(k), v=np.concatenate(v), scale=s)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_with_a_scale_of_zero_weighs_all_tokens_alike(dev, dtype):
    cache, k, v = _filled(dev, [70, 1, 200], 2, 64, dtype, 3)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(4)).to(dev, dtype)
    assert_attention(cache.attend(q, scale=0.0), O.attend(_np(q), k, v, 0.0), q=_np(q), k=np.concatenate(k), v=np.concatenate(v), scale=0.0)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_attend_over_long_and_short_requests_together(dev, dtype):
    """Runs of many blocks, joined; and runs of many requests in one block."""
    lengths = [30000, 1, 7000] + [3] * 50 + [0, 9000, 64]
    cache, k, v = _filled(dev, lengths, 1, 32, dtype, 5)
    q = torch.randn(len(lengths), 2, 32, generator=torch.Generator().manual_seed(2)).to(dev, dtype) * 4
    want = O.attend(_np(q), k, v)
    got = cache.attend(q)
    assert_attention(got, want, q=_np(q), k=np.concatenate(k), v=np.concatenate(v), scale=32**-0.5)
    for _ in range(3):  # the order in which blocks finish does not show
        assert torch.equal(cache.attend(q), got)


def test_attend_large_and_small_scores_and_scales(dev):
    """Scores in the hundreds, queries far outside float16's range, pages whose scales lie 2^30 apart."""
    for qsize, vsize in ((30.0, 1.0), (1e30, 1e-30), (1e-30, 1e30), (0.0, 1.0)):
        cache = _cache(dev, requests=1, pages=4, kv_heads=1, head_width=64, max_blocks=4)
        ref, ks, vs = O.Pages(1, 4, 4), O.Store(1, 64), O.Store(1, 64)
        plan, want = cache.resize([250], tokens=250), ref.resize([250])
        gen = torch.Generator().manual_seed(7)
        k = (torch.randn(250, 1, 64, generator=gen) / max(qsize, 1.0) * (1.0 if qsize < 1e20 else 3.0)).to(dev)
        v = (torch.randn(250, 1, 64, generator=gen) * vsize).to(dev)
        v[64:128] *= 2.0**-30
        v[192:] *= 2.0**-25
        cache.store(k, v, plan)
        ks.put(_np(k), want[3])
        vs.put(_np(v), want[3])
        q = (torch.randn(1, 4, 64, generator=gen) * qsize).to(dev)
        got = cache.attend(q)
        kr, vr = ks.rows(want[1]), vs.rows(want[1])
        assert_attention(got, O.attend(_np(q), [kr], [vr]), q=_np(q), k=kr, v=vr, scale=0.125)


def test_attend_keeps_small_values_beside_large_ones(dev):
    """All weight on a page whose values are 2^40 below another's: the result has its own size."""
    cache = _cache(dev, requests=1, pages=2, kv_heads=1, head_width=32, max_blocks=2)
    plan = cache.resize([128], tokens=128)
    for big_first in (True, False):
        k = torch.zeros(128, 1, 32, device=dev)
        v = torch.ones(128, 1, 32, device=dev)
        small = slice(64, 128) if big_first else slice(0, 64)
        k[small] = 8.0
        v[small] *= 2.0**-40
        cache.store(k, v, plan)
        got = cache.attend(torch.full((1, 1, 32), 8.0, device=dev), scale=1.0)  # the other page's weight is e^-2048
        np.testing.assert_allclose(_np(got), 2.0**-40, rtol=1e-5)


def test_infinite_and_nan_queries_stay_in_their_rows(dev):
    cache, k, v = _filled(dev, [100, 100], 1, 32, torch.float32, 3)
    q = torch.randn(2, 4, 32, device=dev)
    clean = cache.attend(q)
    q[0, 1, 5], q[1, 2, 0] = float("nan"), float("inf")
    got = cache.attend(q)
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 2]).all()
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[0, 1] = keep[1, 2] = False
    assert torch.equal(got[keep], clean[keep])


def test_attend_layers_strides_and_streams(dev):
    cache, k, v = _filled(dev, [70, 130], 2, 64, torch.bfloat16, 9, layers=3, layer=2)
    fused = torch.randn(2, 3, 4, 64, device=dev, dtype=torch.bfloat16)
    want = cache.attend(fused[:, 1].contiguous(), layer=2)
    assert torch.equal(cache.attend(fused[:, 1], layer=2), want)
    off = torch.empty(2 * 256 + 1, device=dev, dtype=torch.bfloat16)[1:].view(2, 4, 64).copy_(fused[:, 1])
    assert torch.equal(cache.attend(off, layer=2), want)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = cache.attend(fused[:, 1], layer=2, workspace=cache.new_workspace(4))
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(other, want)


def test_offsets_past_32_bits(dev):
    """Pages whose codes begin beyond 2^31 bytes."""
    pages = 280_000  # 64 * 128 bytes each
    cache = _cache(dev, requests=2, pages=pages, kv_heads=1, head_width=128, max_blocks=4)
    plan = cache.resize([200, 3], tokens=203)  # from the top of the stack
    assert int(plan.slots.min()) * 128 > 2**31
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn(203, 1, 128, generator=gen).to(dev) for _ in range(2))
    cache.store(k, v, plan)
    got_k, got_v = cache.read(plan.slots, dtype=torch.float32)
    ref, ks, vs = O.Pages(2, pages, 4), O.Store(1, 128), O.Store(1, 128)
    want = ref.resize([200, 3])
    ks.put(_np(k), want[3])
    vs.put(_np(v), want[3])
    kr, vr = ks.rows(want[1]), vs.rows(want[1])
    np.testing.assert_array_equal(_np(got_k), kr)
    np.testing.assert_array_equal(_np(got_v), vr)
    q = torch.randn(2, 2, 128, generator=gen).to(dev)
    assert_attention(cache.attend(q), O.attend(_np(q), [kr[:200], kr[200:]], [vr[:200], vr[200:]]), q=_np(q), k=kr, v=vr,
                     scale=128**-0.5)


# ---- lifecycle, graphs, refusals


def test_requests_leave_and_join(dev):
    cache, k, v = _filled(dev, [70, 10, 200], 1, 32, torch.float32, 11, extra_pages=3)
    q = torch.randn(3, 2, 32, device=dev)
    before = cache.attend(q)
    cache.resize([70, 0, 200], tokens=0)
    cache = cache.with_requests([2, 0], new=1)
    cache.validate_invariants()
    plan = cache.resize([200, 70, 100], tokens=100)
    x = torch.randn(2, 100, 1, 32, device=dev)
    cache.store(x[0], x[1], plan)
    cache.validate_invariants()
    after = cache.attend(q[[2, 0, 1]])
    torch.testing.assert_close(after[:2], before[[2, 0]], rtol=1e-5, atol=1e-6)


def test_a_decode_step_replays_in_a_graph(dev):
    cache, _, _ = _filled(dev, [64, 100, 1], 2, 64, torch.bfloat16, 13, extra_pages=8)
    cache = cache.with_requests([0, 1, 2])
    x = torch.randn(2, 3, 2, 64, device=dev, dtype=torch.bfloat16)
    q = torch.randn(3, 4, 64, device=dev, dtype=torch.bfloat16)
    targets = cache.lengths.clone()
    cache.attend(q)  # the workspace exists before the capture
    targets += 1
    cache.store(x[0], x[1], cache.resize(targets, tokens=3))
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        targets += 1
        plan = cache.resize(targets, tokens=3)
        cache.store(x[0], x[1], plan)
        out = cache.attend(q)
    for step in range(3):
        graph.replay()
        assert cache.lengths.tolist() == [66 + step, 102 + step, 3 + step]
        assert torch.equal(out, cache.attend(q))
    cache.validate_invariants()


def test_refusals(dev):
    from copy_on_write_sdm_b200 import PagedKVCache

    for bad in (dict(head_width=48), dict(requests=8193), dict(kv_heads=0), dict(pages=-1), dict(layers=0), dict(device="cpu"),
                dict(max_blocks=1 << 24)):
        with pytest.raises(ValueError):
            PagedKVCache.allocate(**{**dict(requests=4, pages=4, kv_heads=2, head_width=32, max_blocks=2, device=dev), **bad})
    cache = _cache(dev, requests=2, pages=4, kv_heads=2, head_width=32, max_blocks=2)
    for targets in (torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int64, device=dev),
                    torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(ValueError):
            cache.resize(targets, tokens=0)
    with pytest.raises(ValueError):
        cache.resize([0, 0], tokens=-1)
    plan = cache.resize([3, 4], tokens=7)
    x = torch.zeros(7, 2, 32, device=dev)
    for k, v, kw in ((x[:6], x[:6], {}), (x, x.half(), {}), (x, x, dict(layer=1)), (x.cpu(), x.cpu(), {}), (x.double(), x.double(), {}),
                     (x.clone().requires_grad_(), x, {})):
        with pytest.raises(ValueError):
            cache.store(k, v, plan, **kw)
    cache.resize([3, 4], tokens=0)
    with pytest.raises(ValueError, match="last resize"):
        cache.store(x, x, plan)
    q = torch.zeros(2, 4, 32, device=dev)
    for bad, kw in ((q[:1], {}), (q[:, :3], {}), (q[..., :16], {}), (q.double(), {}), (q, dict(layer=-1)), (q.cpu(), {}),
                    (q, dict(workspace=torch.zeros(16, dtype=torch.uint8, device=dev)))):
        with pytest.raises(ValueError):
            cache.attend(bad, **kw)
    for slots in (torch.zeros(2, device=dev), torch.zeros(2, 2, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            cache.read(slots)
    cache.validate_invariants()


def test_caches_of_different_sizes_take_turns(dev):
    """Launches whose shared memory differs, large after small and back."""
    caches = []
    for requests in (4000, 3, 1500):
        cache, k, v = _filled(dev, [1 + i % 3 for i in range(requests)], 1, 128, torch.bfloat16, requests)
        q = torch.randn(requests, 1, 128, device=dev, dtype=torch.bfloat16)
        caches.append((cache, q, cache.attend(q)))
    for _ in range(2):
        for cache, q, want in caches:
            assert torch.equal(cache.attend(q), want)
