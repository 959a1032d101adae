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
