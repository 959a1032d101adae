"""Prompt attention where blocks take tile after tile, and with more sequences than a warp keeps in its registers,
against the plain form in 64 bits on the same GPU; and 16-bit inputs near the ends of their types.

Tolerance of an output, from its row's own sums: float32's bound (``oracle.kv_oracle.prompt_with_bound``), and for a type of
unit roundoff u (2^-8 bfloat16, 2^-11 float16) 2 u of sum p |v|: the weight's rounding to the type (with float16's
last place, 2^-25, of sum |v|) and the result's."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv_cache import TYPES, dev  # noqa: F401
from tests.test_gpu_prompt_attention import _inputs

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def plain(q, k, v, starts, scale=None):
    """The formula in 64 bits, and each output's bound."""
    u = ROUNDOFF[q.dtype]
    last_place = 2.0**-25 if q.dtype == torch.float16 else 0.0
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for a, z in zip(starts[:-1], starts[1:]):
        if a == z:
            continue
        seen = torch.ones(z - a, z - a, dtype=torch.bool, device=q.device).tril()
        for h in range(q.shape[1]):
            qq, kk, vv = q[a:z, h], k[a:z, h // group], v[a:z, h // group]
            p = torch.softmax((scale * (qq @ kk.T)).masked_fill(~seen, -float("inf")), 1)
            o = p @ vv
            p_reach = p * (abs(scale) * (qq.abs() @ kk.abs().T) + 1)
            # sum_j w_j |v_j - o| <= sum_j w_j |v_j| + |o| sum_j w_j
            moved = p_reach @ vv.abs() + o.abs() * p_reach.sum(1, keepdim=True)
            out[a:z, h] = o
            bound[a:z, h] = 2.0**-20 * (moved + p @ vv.abs()) + 2 * u * (p @ vv.abs()) + last_place * vv.abs().cumsum(0)
    return out, bound


def assert_within(got, want, bound):
    over = (got.double() - want).abs() / (bound + torch.finfo(torch.float32).tiny)
    assert torch.isfinite(got).all() and float(over.max()) <= 1, float(over.max())


def _lengths(count, seed):
    """Mostly short, some of several key tiles, some of none."""
    gen = torch.Generator().manual_seed(seed)
    short = torch.randint(0, 40, (count,), generator=gen)
    long = torch.randint(100, 420, (count,), generator=gen)
    return torch.where(torch.rand(count, generator=gen) < 0.12, long, short).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", (32, 64, 96, 128))
@pytest.mark.parametrize("count,heads,group", [(100, 6, 1), (300, 2, 3)])  # 600 and more tiles; and over 128 sequences
def test_blocks_that_take_several_tiles(dev, dtype, width, count, heads, group):  # noqa: F811
    """Every phase of the barriers, with values that are not finite where no row of the others sees them."""
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, _lengths(count, width + count), heads, group, width, dtype, width)
    got = prompt_attention(q, k, v, device_starts)
    assert_within(got, *plain(q, k, v, starts))
    assert torch.equal(prompt_attention(q, k, v, device_starts), got)
    bad = v.clone()
    seen = torch.zeros(q.shape[:2], dtype=torch.bool, device=dev)
    for i in range(0, count, 5):
        a, z = int(starts[i]), int(starts[i + 1])
        if z - a > 2:
            at, head = a + (z - a) // 2, i % heads
            bad[at, head, i % width] = (float("nan"), float("inf"), -float("inf"))[i % 3]
            seen[at:z, head * group:(head + 1) * group] = True
    dirty = prompt_attention(q, k, bad, device_starts)
    assert torch.equal(dirty[~seen], got[~seen])
    assert not torch.isfinite(dirty[seen]).all(1).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_as_many_sequences_as_tokens(dev, dtype):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, _, device_starts = _inputs(dev, [1] * 1500, 2, 2, 32, dtype, 1)
    got = prompt_attention(q, k, v, device_starts)
    assert_within(got, v.double().repeat_interleave(2, 1), 2 * ROUNDOFF[dtype] * v.double().abs().repeat_interleave(2, 1) + 2.0**-20)


@pytest.mark.parametrize("dtype,sizes", [(torch.bfloat16, (1e4, 1e10, 1e30)), (torch.float16, (3e2, 1e4))])
@pytest.mark.parametrize("width", (64, 128))
def test_much_larger_keys(dev, dtype, sizes, width):  # noqa: F811
    """Scores far above 2^31: one token takes all the weight of the rows that see it, or none; the rows before it see the others."""
    from copy_on_write_sdm_b200 import prompt_attention

    for size in sizes:
        q, k, v, starts, device_starts = _inputs(dev, [200, 150], 1, 2, width, dtype, 21)
        k[[9, 130, 220]] = (k[[9, 130, 220]].float() * size).to(dtype).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)
        q[150:] = (q[150:].float() * 1e4).clamp(-6e4, 6e4).to(dtype)
        assert_within(prompt_attention(q, k, v, device_starts), *plain(q, k, v, starts))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_the_largest_values_of_the_type(dev, dtype):  # noqa: F811
    """Means of numbers whose sums lie beyond float32."""
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, [300], 1, 2, 64, dtype, 22)
    v[:] = 0.98 * torch.finfo(dtype).min
    assert_within(prompt_attention(q, k, v, device_starts), *plain(q, k, v, starts))
