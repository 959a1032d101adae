"""Prompt attention in float32 held to each output's own sums (``oracle.kv_oracle.prompt_with_bound``): the
accuracy of float32 on ordinary inputs, and the same whatever the magnitudes of other tokens, seen or not,
of other widths and of other tiles of the same call."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_gpu_kv_cache import _np, dev  # noqa: F401
from tests.test_gpu_prompt_attention import _inputs

pytestmark = pytest.mark.gpu


def assert_within_own_sums(q, k, v, starts, device_starts, scale=None):
    from copy_on_write_sdm_b200 import prompt_attention

    got = _np(prompt_attention(q, k, v, device_starts, scale=scale))
    want, bound = O.prompt_with_bound(_np(q), _np(k), _np(v), starts, scale)
    bound = bound + np.finfo(np.float32).tiny  # below it the type has no bits left to hold
    over = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (over <= 0).all(), float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)))


@pytest.mark.parametrize("lengths,heads,group,width", [
    ([200], 1, 1, 32), ([300, 17, 90], 1, 3, 96), ([311], 1, 8, 64), ([33, 1, 40], 2, 7, 40), ([130, 2], 1, 33, 128),
    ([400], 2, 1, 64), ([330, 5], 1, 2, 128), ([70], 1, 64, 8), ([65, 64, 63], 2, 2, 120),
])
def test_float32_accuracy(dev, lengths, heads, group, width):  # noqa: F811
    assert_within_own_sums(*_inputs(dev, lengths, heads, group, width, torch.float32, width + len(lengths)))


@pytest.mark.parametrize("width", (32, 64, 128))
@pytest.mark.parametrize("times", (1e6, 1e12, 1e30))
def test_a_much_larger_key_changes_only_the_rows_that_see_it(dev, width, times):  # noqa: F811
    """One key of each of two tiles, among the others' keys: rows before it do not see it, rows after it see a score far
    above or far below the others'."""
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 3)
    k[[9, 100, 160]] *= times
    assert_within_own_sums(q, k, v, starts, device_starts)


@pytest.mark.parametrize("width", (32, 64, 128))
def test_much_larger_queries_of_other_tokens(dev, width):  # noqa: F811
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 4)
    q[::7] *= 1e-25
    q[3::7] *= 1e25
    assert_within_own_sums(q, k, v, starts, device_starts)


@pytest.mark.parametrize("width", (32, 64, 128))
def test_keys_of_unlike_widths(dev, width):  # noqa: F811
    """Widths far apart in keys and queries, whose products are alike; and a width that only the keys have."""
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 5)
    apart = torch.logspace(-12, 12, width, device=dev)
    q, k = q / apart, k * apart
    q[..., 5], k[..., 5] = 0.0, 1e20
    assert_within_own_sums(q, k, v, starts, device_starts)


@pytest.mark.parametrize("width", (32, 64, 128))
@pytest.mark.parametrize("times", (1e6, 1e12, 1e30))
def test_a_much_larger_value_changes_only_the_rows_that_see_it(dev, width, times):  # noqa: F811
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 6)
    v[[9, 100, 160]] *= times
    assert_within_own_sums(q, k, v, starts, device_starts)


@pytest.mark.parametrize("width", (32, 128))
def test_a_much_larger_value_of_no_weight(dev, width):  # noqa: F811
    """Every row sees it, with a weight of e^-300."""
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 7)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[[0, 70, 150], :, 0] = -300 * width**0.5
    v[[0, 70, 150]] *= 1e30
    assert_within_own_sums(q, k, v, starts, device_starts)


@pytest.mark.parametrize("width", (32, 64, 128))
def test_values_of_unlike_widths(dev, width):  # noqa: F811
    q, k, v, starts, device_starts = _inputs(dev, [150, 40], 1, 2, width, torch.float32, 8)
    assert_within_own_sums(q, k, v * torch.logspace(-25, 25, width, device=dev), starts, device_starts)


@pytest.mark.parametrize("sizes", [
    (2.0**60, 1.0, 2.0**-60), (2.0**33, 2.0**-17, 2.0**-66), (1e4, 1e-12, 1e-26), (1e30, 1e10, 1e-10, 1e-30), (0.0, 1e-20, 1e-25),
    (0.0, 0.0, 1e20, 1e-20), (1e-30, 1.0, 1e30), (1e30, 0.0, 1e-30),
])
@pytest.mark.parametrize("width", (32, 128))
def test_values_that_fall_or_rise_from_tile_to_tile(dev, sizes, width):  # noqa: F811
    """Also where the weight moves along with them: the second sequence's scores grow by hundreds from tile to tile, so
    that the last tile's values alone are left."""
    n = 64 * len(sizes)
    q, k, v, starts, device_starts = _inputs(dev, [n, n], 1, 2, width, torch.float32, 9)
    v *= torch.tensor(sizes * 2, device=dev).repeat_interleave(64)[:, None, None]
    q[..., 0] = 1.0
    k[n:, :, 0] = 400.0 * torch.arange(n, device=dev)[:, None].div(64, rounding_mode="floor") * width**0.5
    assert_within_own_sums(q, k, v, starts, device_starts)


def test_the_largest_values_of_the_type(dev):  # noqa: F811
    """Means of numbers that would overflow if they were added up first (a little below the largest: a result rounded up
    from that one is infinite)."""
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, starts, device_starts = _inputs(dev, [200], 1, 2, 32, torch.float32, 10)
    v[:] = 0.99 * torch.finfo(torch.float32).min
    got = prompt_attention(q, k, v, device_starts)
    torch.testing.assert_close(got, torch.full_like(got, 0.99 * torch.finfo(torch.float32).min), rtol=2.0**-19, atol=0.0)


def test_values_that_are_not_finite_in_a_long_prompt(dev):  # noqa: F811
    """Few of them, in spans of more than one key tile; each row has the sum of those that it sees."""
    from copy_on_write_sdm_b200 import prompt_attention

    q, k, v, _, device_starts = _inputs(dev, [17000, 100], 1, 1, 32, torch.float32, 11)
    clean = prompt_attention(q, k, v, device_starts)
    inf, nan = float("inf"), float("nan")
    bad = {(700, 3): inf, (9001, 3): inf, (12000, 3): -inf, (16990, 4): -inf, (5, 5): nan, (17050, 6): inf}
    for (token, d), x in bad.items():
        v[token, 0, d] = x
    got = prompt_attention(q, k, v, device_starts)
    want = clean.clone()
    for (token, d), x in bad.items():
        want[token:17000 if token < 17000 else None, 0, d] += x
    same = want.isfinite()
    torch.testing.assert_close(got[~same], want[~same], rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(got[same], clean[same], rtol=0, atol=0)
