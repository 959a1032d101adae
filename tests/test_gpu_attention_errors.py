"""What the attention layers' operators report of errors on the device, and what they refuse on the host.  The words are
set by hand: no test makes a kernel's wait run out."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv_cache import _cache, dev  # noqa: F401
from tests.test_gpu_paged_serving import _model, _prompts

pytestmark = pytest.mark.gpu


def test_a_wait_that_gave_up_is_raised_by_name(dev):  # noqa: F811
    from copy_on_write_sdm_b200 import _lib

    cache = _cache(dev, requests=1, pages=1, kv_heads=1, head_width=32, max_blocks=1)
    cache.status_word.fill_(_lib.ST_WAIT_TIMEOUT)
    with pytest.raises(RuntimeError, match="wait .* gave up"):
        cache.validate_invariants()


def test_prompts_report_to_the_word_they_are_given(dev, monkeypatch):  # noqa: F811
    from copy_on_write_sdm_b200 import kv_cache, prompt_attention, prompt_attention_status

    words, call = [], kv_cache._call

    def watched(device, what, *args):
        if what == "cow_prompt_attention":
            words.append(args[-1])
        call(device, what, *args)

    monkeypatch.setattr(kv_cache, "_call", watched)
    x = torch.randn(5, 2, 32, device=dev)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    prompt_attention(x, x, x, starts)
    prompt_attention(x, x, x, starts, status=word)
    assert words == [prompt_attention_status(dev).data_ptr(), word.data_ptr()] and not word.item()
    for bad in (word.long(), word.cpu(), torch.zeros(2, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            prompt_attention(x, x, x, starts, status=bad)


def test_serving_reports_attention_errors(dev, monkeypatch):  # noqa: F811
    from copy_on_write_sdm_b200 import _lib, kv_cache
    from copy_on_write_sdm_b200.paged import PagedServing

    words, call = [], kv_cache._call

    def watched(device, what, *args):
        if what == "cow_prompt_attention":
            words.append(args[-1])
        call(device, what, *args)

    monkeypatch.setattr(kv_cache, "_call", watched)
    serving = PagedServing(_model(dev, "BA"), pages=6, sdm_growth_quantum_rows=64)
    serving.admit(_prompts([5, 70], 0), ["a", "b"])
    assert words == [serving.cache.status_word.data_ptr()]
    serving.validate_invariants()
    serving.cache.status_word.fill_(_lib.ST_WAIT_TIMEOUT)
    with pytest.raises(RuntimeError, match="gave up"):
        serving.validate_invariants()


def test_buffers_that_are_kept_are_not_made_in_a_capture(dev, monkeypatch):  # noqa: F811
    """Their zeroing would wait for the first replay."""
    from copy_on_write_sdm_b200 import kv_cache, prompt_attention

    cache = _cache(dev, requests=1, pages=2, kv_heads=1, head_width=32, max_blocks=2)
    x = torch.randn(2, 5, 1, 32, device=dev)
    cache.store(x[0], x[1], cache.resize([5], tokens=5))
    q = torch.randn(1, 2, 32, device=dev)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    monkeypatch.setattr(kv_cache, "_PROMPT_STATUS", {})
    for early in (lambda: cache.attend(q), lambda: cache.new_workspace(2), lambda: prompt_attention(x[0], x[0], x[1], starts)):
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                early()
    want = cache.attend(q), prompt_attention(x[0], x[0], x[1], starts)  # made here, ready at once
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attend(q), prompt_attention(x[0], x[0], x[1], starts)
    graph.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_workspaces_that_attend_cannot_use(dev):  # noqa: F811
    cache = _cache(dev, requests=1, pages=1, kv_heads=1, head_width=32, max_blocks=1)
    q = torch.zeros(1, 2, 32, device=dev)
    good = cache.new_workspace(2)
    for bad in (good.cpu(), good.view(torch.float32), torch.zeros(2 * good.numel(), dtype=torch.uint8, device=dev)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            cache.attend(q, workspace=bad)
    assert cache.attend(q, workspace=good).eq(0).all()


def test_a_bound_on_new_tokens_near_2_to_the_31(dev):  # noqa: F811
    """The maps' last steps, of a resize that fits and of one that does not."""
    tokens = 2**31 - 1
    cache = _cache(dev, requests=2, pages=3, kv_heads=1, head_width=32, max_blocks=2)
    for target in ([65, 3], [0, 129]):
        plan = cache.resize(target, tokens=tokens)
        new = 68 if target[0] else 0
        assert plan.starts.tolist() == ([0, 65, 68] if new else [0, 0, 0])
        for words in (plan.slots, plan.positions):
            assert bool((words[:new] >= 0).all()) and bool((words[-(1 << 20):] == -1).all()) and int(words[new:].max()) == -1
        del plan, words
        torch.cuda.empty_cache()
    assert int(cache.status_word) and cache.lengths.tolist() == [65, 3]
    with pytest.raises(ValueError):
        cache.resize([65, 3], tokens=tokens + 1)


def test_store_for_no_request(dev):  # noqa: F811
    """Room for tokens in the plan of a cache without requests: nothing is stored, nothing raised."""
    cache = _cache(dev, requests=0, pages=1, kv_heads=1, head_width=32, max_blocks=1)
    for tokens in (0, 5, 200):
        x = torch.ones(tokens, 1, 32, device=dev)
        cache.store(x, x, cache.resize([], tokens=tokens))
    assert not cache.key_pages.view(torch.uint8).any()
    cache.validate_invariants()


def test_forward_mode_tangents_are_refused(dev):  # noqa: F811
    """As inputs that ask for a gradient are: they would be dropped."""
    from torch.autograd import forward_ad

    from copy_on_write_sdm_b200 import prompt_attention

    cache = _cache(dev, requests=1, pages=1, kv_heads=1, head_width=32, max_blocks=1)
    x = torch.randn(3, 1, 32, device=dev)
    starts = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    plan = cache.resize([3], tokens=3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: prompt_attention(x, dual, x, starts), lambda: cache.store(x, dual, plan), lambda: cache.attend(dual[:1])):
            with pytest.raises(ValueError, match="gradient"):
                call()
        prompt_attention(x, x, x, starts)  # inputs without one pass


def test_requests_that_cannot_be_kept(dev):  # noqa: F811
    """A slot that is not there would be an index out of range on the device, one kept twice two owners of its pages."""
    cache = _cache(dev, requests=3, pages=3, kv_heads=1, head_width=32, max_blocks=1)
    cache.resize([1, 2, 3], tokens=6)
    for keep in ([3], [-1], [0, 0], [0.5], torch.tensor([0, 7]), torch.tensor([1, 1], device=dev), torch.tensor([[0]])):
        with pytest.raises(ValueError):
            cache.with_requests(keep)
    plan = cache.resize([1, 2, 0], tokens=0)
    assert plan.starts.tolist() == [0, 0, 0, 0]
    kept = cache.with_requests(torch.tensor([1, 0], device=dev), new=1)
    assert kept.lengths.tolist() == [2, 1, 0]
    kept.validate_invariants()
