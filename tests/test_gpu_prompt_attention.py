"""Packed causal prompt attention (prompt_attention) against its plain 64-bit form.

Tolerance of o = sum p v / sum p, |v| <= vmax: with u the type's unit roundoff (2^-8
bfloat16, 2^-11 float16) the result is rounded once (u |o|) and each probability at most
once to the type, which moves the mean by u vmax; in float32 arithmetic a score is off by 2^-20 of
sum |q k| <= width * qmax * kmax * scale, a probability by that and 2^-21, the mean by twice the same times vmax."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_gpu_kv_cache import TYPES, _np, assert_attention, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _inputs(dev, lengths, heads, group, width, dtype, seed=0):  # noqa: F811
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)
    q = torch.randn(total, heads * group, width, generator=gen).to(dev, dtype)
    k, v = (torch.randn(total, heads, width, generator=gen).to(dev, dtype) for _ in range(2))
    starts = np.concatenate(([0], np.cumsum(lengths)))
    return q, k, v, starts, torch.tensor(starts, dtype=torch.int32, device=dev)


def _check(got, q, k, v, starts, scale=None):
    s = q.shape[2] ** -0.5 if scale is None else scale
    assert_attention(got, O.prompt(_np(q), _np(k), _np(v), starts, s), q=_np(q), k=_np(k), v=_np(v), scale=s)


CASES = [
    ([1], 1, 1, 32), ([2, 1, 3], 2, 2, 64), ([0, 5, 0, 64, 65, 0], 1, 4, 128), ([127, 128, 129], 2, 1, 128),
    ([300, 17, 256], 1, 3, 96), ([511], 1, 8, 64), ([33, 1, 40], 2, 7, 40), ([70], 1, 64, 8), ([130, 2], 1, 33, 128),
    ([1] * 70, 1, 2, 32), ([260, 4], 1, 16, 120), ([700], 2, 1, 64), ([1030, 5], 1, 2, 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group,width", CASES)
def test_prompt_attention_matches_the_plain_form(dev, dtype, lengths, heads, group, width):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, lengths, heads, group, width, dtype, len(lengths) + width)
    got = prompt_attention(q, k, v, device_starts)
    assert got.dtype == dtype and got.shape == q.shape and got.is_contiguous()
    _check(got, q, k, v, starts)
    assert torch.equal(prompt_attention(q, k, v, device_starts), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dev, dtype):  # noqa: F811
    """Scores in the hundreds, of both signs: the running maximum moves far, up and not at all."""
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, [400, 90], 1, 2, 64, dtype, 3)
    q = (q.float() * 12).to(dtype)
    k = (k.float() * torch.linspace(0.2, 12, k.shape[0], device=dev)[:, None, None]).to(dtype)
    _check(prompt_attention(q, k, v, device_starts, scale=0.3), q, k, v, starts, 0.3)
    flipped = k.flip(0).contiguous()
    _check(prompt_attention(q, flipped, v, device_starts, scale=-0.3), q, flipped, v, starts, -0.3)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_views(dev, dtype):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    heads, group, width, lengths = 2, 3, 64, [90, 150]
    total = sum(lengths)
    fused = torch.randn(total, (heads * group + 2 * heads) * width, device=dev).to(dtype)
    q, k, v = fused.split([heads * group * width, heads * width, heads * width], dim=1)
    q, k, v = q.view(total, -1, width), k.view(total, -1, width), v.view(total, -1, width)
    starts = torch.tensor([0, 90, 240], dtype=torch.int32, device=dev)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts)
    assert torch.equal(prompt_attention(q, k, v, starts), want)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*turned, starts), want)
    off = [torch.empty(t.numel() + 1, device=dev, dtype=dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*off, starts), want)
    one = k[:, :1].expand(total, heads, width)  # a broadcast head: stride 0
    assert torch.equal(prompt_attention(q, one, v, starts), prompt_attention(q, one.contiguous(), v, starts))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
def test_what_a_query_does_not_see_does_not_touch_it(dev, dtype, bad):  # noqa: F811
    """NaN and infinities in later tokens and in other sequences leave a row as it was; rows that see them have them."""
    from copy_on_write_sdm_b200 import prompt_attention

    lengths = [200, 37, 150]
    q, k, v, starts, device_starts = _inputs(dev, lengths, 2, 2, 64, dtype, 17)
    clean = prompt_attention(q, k, v, device_starts)
    for which in ("k", "v"):
        k2, v2 = k.clone(), v.clone()
        at = 200 + 20  # in the second sequence
        (k2 if which == "k" else v2)[at, 0] = bad
        got = prompt_attention(q, k2, v2, device_starts)
        seen = torch.zeros(sum(lengths), 4, dtype=torch.bool, device=dev)
        seen[at:237, :2] = True
        assert torch.isfinite(got[~seen]).all()
        u = {torch.float32: 2.0**-18, torch.bfloat16: 2.0**-7, torch.float16: 2.0**-10}[dtype]
        torch.testing.assert_close(got[~seen], clean[~seen], rtol=u, atol=u)
        if which == "v":
            assert not torch.isfinite(got[at:237, :2]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_scale_of_zero_weighs_all_tokens_alike(dev, dtype):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, [300, 17], 2, 2, 64, dtype, 5)
    _check(prompt_attention(q, k, v, device_starts, scale=0.0), q, k, v, starts, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_key_of_score_minus_infinity_has_no_weight(dev, dtype):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, [200, 150], 2, 2, 64, dtype, 6)
    q[..., 3] = -q[..., 3].abs() - 0.5
    k[[20, 220], :, 3] = float("inf")
    _check(prompt_attention(q, k, v, device_starts), q, k, v, starts)


def test_tokens_outside_every_sequence(dev):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, _, _ = _inputs(dev, [100], 1, 2, 32, torch.bfloat16, 1)
    starts = torch.tensor([10, 40, 75], dtype=torch.int32, device=dev)
    k[:10], v[:10], k[75:], v[75:] = (float("nan"),) * 4
    got = prompt_attention(q, k, v, starts)
    want = O.prompt(_np(q[10:75]), _np(k[10:75]), _np(v[10:75]), [0, 30, 65])
    assert_attention(got[10:75], want, q=_np(q), k=_np(k[10:75]), v=_np(v[10:75]), scale=32**-0.5)


def test_nothing_to_do(dev):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q = torch.empty(0, 4, 32, device=dev)
    for starts in ([0], [0, 0, 0]):
        assert prompt_attention(q, q[:, :2], q[:, :2], torch.tensor(starts, dtype=torch.int32, device=dev)).shape == (0, 4, 32)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_offsets_past_32_bits(dev, dtype):  # noqa: F811
    """Rows that lie beyond 2^31 elements of the key and value storage."""
    from copy_on_write_sdm_b200 import prompt_attention

    stride = 1 << 24  # elements between tokens
    big = torch.empty((150 * stride,), dtype=dtype, device=dev)
    view = big.view(150, stride)
    gen = torch.Generator().manual_seed(5)
    k, v = view[:, :64].unsqueeze(1), view[:, 64:128].unsqueeze(1)
    k.copy_(torch.randn(150, 1, 64, generator=gen))
    v.copy_(torch.randn(150, 1, 64, generator=gen))
    q = torch.randn(150, 2, 64, generator=gen).to(dev, dtype)
    starts = torch.tensor([0, 10, 150], dtype=torch.int32, device=dev)
    assert torch.equal(prompt_attention(q, k, v, starts), prompt_attention(q, k.contiguous(), v.contiguous(), starts))


def test_refusals(dev):  # noqa: F811
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, _, starts = _inputs(dev, [6], 2, 2, 32, torch.float32)
    for a, b, c, s in (
        (q[:5], k, v, starts), (q, k[:, :1].expand(6, 3, 32), v[:, :1].expand(6, 3, 32), starts), (q, k, v[..., :16], starts),
        (q[..., :12], k[..., :12], v[..., :12], starts), (q, k.half(), v, starts), (q.double(), k.double(), v.double(), starts),
        (q, k, v, starts.long()), (q, k, v, starts.cpu()), (q.cpu(), k.cpu(), v.cpu(), starts), (q[0], k[0], v[0], starts),
        (q.repeat(1, 1, 5), k.repeat(1, 1, 5), v.repeat(1, 1, 5), starts), (q.repeat(1, 33, 1), k, v, starts),
        (q, k, v, starts[:0]), (q.clone().requires_grad_(), k, v, starts),
    ):
        with pytest.raises(ValueError):
            prompt_attention(a, b, c, s)
