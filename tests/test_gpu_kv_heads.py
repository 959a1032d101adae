"""Models whose query heads share key and value heads, and models in bfloat16, through every path that serves them.

A model with ``kv_heads`` equals the one with all heads whose key and value projections are repeated: 1e-4 in float32, the
whole-model tolerance of the other tests.  A bfloat16 model is held to the float32 one with the same (bfloat16) weights:
its activations are rounded a few times a layer, relative 2^-9 each, and its decode sees keys and values in e4m3, so
that the logits' relative error stays below 2^-4."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_serving import _prompts, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _model(dev, layout, heads, kv_heads, dtype=torch.float32, width=128):  # noqa: F811
    from copy_on_write_sdm_b200.model import LanguageModel

    model = LanguageModel(vocab_size=97, maximum_sequence_length=256, layout=layout, width=width, heads=heads, kv_heads=kv_heads, slots=64,
                          reads=8, writes=2, memory_heads=2, activation_dtype=dtype)
    model.initialize_role_keyed(1)
    return model.to(dev, dtype).eval()


def _with_all_heads(dev, model, layout, heads, kv_heads):  # noqa: F811
    other = _model(dev, layout, heads, None)
    state = model.state_dict()
    for name, weight in state.items():
        if name.endswith("attention.qkv.weight"):
            width = weight.shape[1]
            q, k, v = weight.split([width, (weight.shape[0] - width) // 2, (weight.shape[0] - width) // 2])
            k, v = (t.view(kv_heads, width // heads, width).repeat_interleave(heads // kv_heads, 0).reshape(width, width) for t in (k, v))
            state[name] = torch.cat((q, k, v))
    other.load_state_dict(state)
    return other


@pytest.mark.parametrize("layout,heads,kv_heads", [("BA", 4, 1), ("BAB", 4, 2)])
def test_shared_heads_on_the_fixed_capacity_paths(dev, layout, heads, kv_heads, tmp_path):  # noqa: F811
    from copy_on_write_sdm_b200 import checkpoint
    from copy_on_write_sdm_b200.graph import GraphedDecode

    model = _model(dev, layout, heads, kv_heads)
    other = _with_all_heads(dev, model, layout, heads, kv_heads)
    ids = torch.stack(_prompts([20, 20, 20], 1)).to(dev)
    torch.testing.assert_close(model(ids), other(ids), atol=1e-4, rtol=1e-4)
    states = []
    for m in (model, other):
        logits, state = m.prefill(ids, capacity=64, sdm_growth_quantum_rows=64)
        states.append((logits, state))
    torch.testing.assert_close(states[0][0], states[1][0], atol=1e-4, rtol=1e-4)
    assert states[0][1].dense_keys[0].shape[1] == kv_heads
    for step in range(2):
        token = torch.full((3, 1), 5 + step, device=dev)
        torch.testing.assert_close(model.decode(token, states[0][1]), other.decode(token, states[1][1]), atol=1e-4, rtol=1e-4)
    for m, (_, state) in zip((model, other), states):  # positions of their own
        m.admit(torch.stack(_prompts([7], 2)).to(dev), state)
    token = torch.arange(4, device=dev)[:, None]
    torch.testing.assert_close(model.decode(token, states[0][1]), other.decode(token, states[1][1]), atol=1e-4, rtol=1e-4)
    # a graph's tokens are those of the eager path, and a checkpoint's requests go on as the ones they were taken from
    graphed = GraphedDecode(model, states[0][1])
    for step in range(3):
        got = graphed.step(token + step)
        torch.testing.assert_close(got, other.decode(token + step, states[1][1]), atol=1e-4, rtol=1e-4)
    saved = checkpoint.export_requests(states[0][1], [1, 3])
    saved.save(tmp_path / "two")
    memories = [model.stack.sdm_layers[str(i)].initial_memory for i in states[0][1].sdm_layer_positions]
    restored = checkpoint.restore_requests(checkpoint.ServingCheckpoint.load(tmp_path / "two"), memories)
    got, want = model.decode(token[[1, 3]], restored), other.decode(token, states[1][1])[[1, 3]]
    torch.testing.assert_close(got, want, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, 2.0**-4), (torch.float16, 2.0**-4)])
@pytest.mark.parametrize("layout,heads,kv_heads", [("A", 4, 2), ("AA", 2, 2), ("AA", 1, 1)])  # heads of 32, 64, 128
def test_models_in_16_bits_are_served(dev, layout, heads, kv_heads, dtype, bound):  # noqa: F811
    """Prompts of one to four key tiles through the tensor-core kernel, pages and attend, in the type of the model."""
    from copy_on_write_sdm_b200.paged import PagedServing

    model = _model(dev, layout, heads, kv_heads, dtype)
    exact = _model(dev, layout, heads, kv_heads)
    exact.load_state_dict({name: weight.float() for name, weight in model.state_dict().items()})
    serving = PagedServing(model, pages=24)
    ids = {}

    def check(logits):
        assert logits.dtype == dtype and torch.isfinite(logits).all()
        for row, name in zip(logits.float(), serving.requests):
            want = exact(torch.tensor(ids[name], device=dev)[None])[0, -1]
            assert float((row - want).norm()) <= bound * float(want.norm()), (name, len(ids[name]))

    for names, lengths in ((list("abcde"), [200, 1, 64, 129, 65]), (list("fg"), [100, 17])):
        prompts = _prompts(lengths, len(names))
        ids.update({name: p.tolist() for name, p in zip(names, prompts)})
        live = len(serving.requests)
        logits = serving.admit(prompts, names)
        for row, name in zip(logits.float(), serving.requests[live:]):
            want = exact(torch.tensor(ids[name], device=dev)[None])[0, -1]
            assert float((row - want).norm()) <= bound * float(want.norm()), (name, len(ids[name]))
        for step in range(3):
            new = torch.arange(len(serving.requests)) * 7 + step
            logits = serving.decode(new)
            for name, i in zip(serving.requests, new.tolist()):
                ids[name].append(i)
            check(logits)
        serving.release([serving.requests[0]])
    serving.validate_invariants()
