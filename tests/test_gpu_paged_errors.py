"""PagedServing where a call raises part way, on the host: an admission leaves the batch as it was, a decode step or release says
that the batch is unusable."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_serving import _model, _prompts, dev  # noqa: F401

pytestmark = pytest.mark.gpu


class Stop(Exception):
    pass


def _raise_after(monkeypatch, owner, name, calls):
    """``owner.name`` raises from its call number ``calls`` on."""
    real, count = getattr(owner, name), [0]

    def wrapped(*args, **kw):
        count[0] += 1
        if count[0] > calls:
            raise Stop
        return real(*args, **kw)

    monkeypatch.setattr(owner, name, wrapped)


def _serving(dev, layout):  # noqa: F811
    from copy_on_write_sdm_b200.paged import PagedServing

    return PagedServing(_model(dev, layout), pages=12, sdm_growth_quantum_rows=64)


PLACES = {
    "embedding": lambda m: (m, "_embed", 0),
    "attention": lambda m: (m.stack.attention_layers["1"].attention, "prefill_packed", 0),
    "after attention": lambda m: (m.stack.attention_layers["1"].mlp, "forward", 0),
    "second group of an SDM layer": lambda m: (m.stack.sdm_layers["2"], "prefill", 1),
    "logits": lambda m: (m.final_norm, "forward", 0),
}


@pytest.mark.parametrize("first", (False, True))
@pytest.mark.parametrize("place", [*PLACES, "second cohort"])
def test_an_admission_that_raises_leaves_the_batch_as_it_was(dev, monkeypatch, place, first):  # noqa: F811
    from copy_on_write_sdm_b200.inference import FaithfulSDMDecodeState

    serving, other = _serving(dev, "BAB"), _serving(dev, "BAB")
    if not first:
        for s in (serving, other):
            s.admit(_prompts([70, 3, 64], 1), ["a", "b", "c"])
            s.decode(torch.tensor([1, 2, 3]))
    with monkeypatch.context() as patch:
        # the first group of the batch's first admission makes its state without `admit`
        _raise_after(patch, *(PLACES[place](serving.model) if place in PLACES else (FaithfulSDMDecodeState, "admit", 0 if first else 1)))
        with pytest.raises(Stop):
            serving.admit(_prompts([5, 66, 5, 130], 2), ["d", "e", "f", "g"])
    assert serving.requests == other.requests and serving.lengths == other.lengths and serving.free_pages == other.free_pages
    serving.validate_invariants()
    assert serving.free_pages == int(serving.cache.free_count)
    for s in (serving, other):  # and both go on alike
        s.logits = [s.admit(_prompts([9, 80], 3), ["x", "y"])]
        for step in range(2):
            s.logits.append(s.decode(torch.arange(len(s.requests)) + step))
    serving.validate_invariants()
    assert serving.requests == other.requests and torch.equal(serving.cache.block_tables, other.cache.block_tables)
    for a, b in zip(serving.logits, other.logits):
        torch.testing.assert_close(a, b, atol=1e-5, rtol=1e-5)


def test_an_admission_that_no_kernel_takes(dev):  # noqa: F811
    serving = _serving(dev, "BA")
    serving.admit(_prompts([3], 0), ["a"])
    for bad in (torch.tensor([1.0, 2.0]), torch.tensor([1, 97]), torch.tensor([-1])):
        with pytest.raises(ValueError):
            serving.admit([torch.tensor([1]), bad], ["b", "c"])
        with pytest.raises(ValueError):
            serving.decode(bad[-1:])
    assert serving.requests == ["a"] and serving.free_pages == 11
    serving.admit([torch.tensor([4, 5]), torch.tensor([6], device=dev)], ["b", "c"])  # some here, some there
    serving.decode(torch.tensor([1, 2, 3], device=dev, dtype=torch.int32))
    serving.validate_invariants()


@pytest.mark.parametrize("call", ("decode", "release"))
def test_a_batch_left_part_way_says_so(dev, monkeypatch, call):  # noqa: F811
    serving = _serving(dev, "BAB")
    serving.admit(_prompts([3, 70], 0), ["a", "b"])
    with monkeypatch.context() as patch:
        if call == "decode":
            _raise_after(patch, serving.model.stack.attention_layers["1"].mlp, "forward", 0)
        else:
            _raise_after(patch, serving.sdm, "release_and_compact", 0)
        with pytest.raises(Stop):
            serving.decode(torch.tensor([1, 2])) if call == "decode" else serving.release(["a"])
    for again in (lambda: serving.decode(torch.tensor([1, 2])), lambda: serving.admit(_prompts([1], 0), ["c"]),
                  lambda: serving.release(["b"])):
        with pytest.raises(RuntimeError, match="unusable"):
            again()
