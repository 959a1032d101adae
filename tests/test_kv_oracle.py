"""CPU checks of the K/V cache's plain form and of its C entry points' refusals."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from copy_on_write_sdm_b200 import PagedKVCache, _lib, prompt_attention
from oracle import kv_oracle as O


def test_e4m3_rounding_equals_the_type():
    x = np.random.default_rng(0).standard_normal(4000) * np.exp2(np.random.default_rng(1).integers(-14, 9, 4000))
    x = np.clip(x, -448, 448).astype(np.float32)
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    middle = (every[:126] + every[1:127]) / 2  # ties
    for values in (x, every[np.isfinite(every)], middle):
        want = torch.tensor(values).to(torch.float8_e4m3fn).float().numpy()
        np.testing.assert_array_equal(O.e4m3(values), want)


def test_scale_is_the_least_power_that_holds():
    for most, want in ((448.0, 1.0), (448.001, 2.0), (224.0, 0.5), (1.0, 2.0**-8), (0.0, 2.0**-64), (1e-30, 2.0**-64)):
        assert O.scale_of(np.array([most, -most / 2, np.inf, np.nan])) == want


def test_pages_are_given_back_in_the_order_they_were_taken():
    pages = O.Pages(3, 10, 4)
    pages.resize([100, 64, 200])
    before = pages.tables.copy(), list(pages.free)
    starts, slots, positions, pieces = pages.resize([130, 64, 256])
    assert starts == [0, 30, 30, 86] and pieces[0][1:2] + pieces[0][3:] == [28, 36]
    pages.resize([100, 64, 200])
    assert (pages.tables == before[0]).all() and pages.free == before[1]
    pages.resize([0, 0, 0])
    assert sorted(pages.free) == list(range(10))


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        prompt_attention(torch.zeros(2, 2, 32), torch.zeros(2, 1, 32), torch.zeros(2, 1, 32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache.allocate(requests=1, pages=1, kv_heads=1, head_width=32, max_blocks=1, device="cpu")


def test_entry_points_reject_bad_arguments_without_a_gpu():
    lib = _lib.load()
    ws = ctypes.create_string_buffer(4096)
    base = (ctypes.addressof(ws) + 15) & ~15
    good = dict(requests=4, max_blocks=2, pages=8, layers=1, kv_heads=2, width=32)

    def cache(**kw):
        c = _lib.CowKVPages(*([base] * 10))
        for name, value in {**good, **kw}.items():
            setattr(c, name, value)
        return ctypes.addressof(c), c

    # plan: header, pieces of at most min(tokens, tokens / 64 + 2 requests), starts, slots, positions
    assert lib.cow_pages_plan_words(4, 10) == 4 + 4 * 8 + 5 + 20
    assert lib.cow_pages_plan_words(4, 3) == 4 + 4 * 3 + 5 + 6
    assert lib.cow_pages_plan_words(-1, 3) == -1 and lib.cow_pages_plan_words(8193, 3) == -1
    assert lib.cow_pages_plan_words(1, -1) == -1 and lib.cow_pages_plan_words(1, 1 << 31) == -1
    at, keep = cache()
    assert lib.cow_pages_resize(None, base, 3, base, 100, None) == _lib.ERR_INVALID
    assert lib.cow_pages_resize(at, base, 3, base, 26, None) == _lib.ERR_INVALID  # plan too small
    assert lib.cow_pages_resize(at, None, 3, base, 100, None) == _lib.ERR_INVALID
    assert lib.cow_pages_resize(at, base, 3, base + 4, 100, None) == _lib.ERR_INVALID  # unaligned plan
    at, keep = cache(max_blocks=1 << 24)
    assert lib.cow_pages_resize(at, base, 3, base, 100, None) == _lib.ERR_UNSUPPORTED
    at, keep = cache()
    store = lib.cow_kv8_store
    assert store(at, 1, base, 64, 32, base, 64, 32, 0, base, 3, None) == _lib.ERR_INVALID  # no such layer
    assert store(at, 0, base, 63, 32, base, 64, 32, 0, base, 3, None) == _lib.ERR_INVALID  # rows off 16 bytes
    assert store(at, 0, None, 64, 32, base, 64, 32, 0, base, 3, None) == _lib.ERR_INVALID
    assert store(at, 0, base, 64, 32, base, 64, 32, 7, base, 3, None) == _lib.ERR_INVALID
    assert lib.cow_kv8_read(at, 0, None, 3, base, base, 0, None) == _lib.ERR_INVALID
    assert lib.cow_kv8_read(at, 0, base, -1, base, base, 0, None) == _lib.ERR_INVALID
    need = lib.cow_kv8_attend_workspace_bytes(at, 4)
    assert need > 0 and lib.cow_kv8_attend_workspace_bytes(at, 3) == -1
    assert lib.cow_kv8_attend(at, 0, base, 128, 32, 0, 4, 1.0, base, base, need - 1, None) == _lib.ERR_INVALID
    assert lib.cow_kv8_attend(at, 0, base, 127, 32, 0, 4, 1.0, base, base, need, None) == _lib.ERR_INVALID
    at, keep = cache(width=48)
    assert store(at, 0, base, 64, 32, base, 64, 32, 0, base, 3, None) == _lib.ERR_UNSUPPORTED
    assert lib.cow_kv8_attend_workspace_bytes(at, 4) == -1
    del keep

    def prompt(width=32, heads=4, kv_heads=2, dtype=0, q=base, stride=128, out=base):
        return lib.cow_prompt_attention(q, stride, 32, base, 64, 32, base, 64, 32, base, 1, 8, heads, kv_heads, width, dtype,
                                        1.0, out, None, None)
    assert prompt(q=None) == _lib.ERR_INVALID
    assert prompt(out=None) == _lib.ERR_INVALID
    assert prompt(stride=126) == _lib.ERR_INVALID
    assert prompt(heads=3) == _lib.ERR_INVALID
    assert prompt(dtype=5) == _lib.ERR_INVALID
    assert prompt(width=136) == _lib.ERR_UNSUPPORTED
    assert prompt(width=36) == _lib.ERR_UNSUPPORTED
    assert prompt(heads=130) == _lib.ERR_UNSUPPORTED


def test_the_float32_bound_tells_half_the_bits():
    """Outputs whose queries and keys, values or weights were rounded to 11 bits lie outside it, float32 ones inside."""
    rng = np.random.default_rng(0)
    for length, width in ((60, 32), (120, 64), (90, 128)):
        q, k, v = (rng.standard_normal((length, 1, width)).astype(np.float32) for _ in range(3))
        want, bound = O.prompt_with_bound(q, k, v, [0, length])
        np.testing.assert_allclose(want, O.prompt(q, k, v, [0, length]), rtol=1e-9, atol=1e-12)

        def outside(q, k, v, weight=lambda p: p, t=np.float64):
            got = np.zeros(want.shape)
            for i in range(length):
                s = (k[:i + 1, 0].astype(t) @ q[i, 0].astype(t)) * t(width**-0.5)
                p = np.exp(s - s.max())
                got[i, 0] = (weight(p).astype(t) @ v[:i + 1, 0].astype(t)) / p.sum()
            return float((np.abs(got - want) > bound).mean())

        def half(x):
            return x.astype(np.float16).astype(np.float32)

        assert outside(q, k, v, t=np.float32) == 0
        assert outside(half(q), half(k), v) > 0.1
        assert outside(q, k, half(v)) > 0.1
        assert outside(q, k, v, weight=half) > 0.1
