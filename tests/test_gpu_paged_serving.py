"""Paged serving of ragged requests (PagedServing, the packed attention methods) against the
model's own full forward and against a plain attention over the rows that the cache holds.

Prompt logits go through float32 attention only: 1e-4, the whole-model tolerance of the other
tests.  Decode logits of layouts that end in attention see keys and values rounded to e4m3, a
relative 2^-4 each at most: the logits' relative error stays below 2^-4.  An SDM layer after attention turns
that rounding into other routes now and then, which no bound holds; there the keys and values are
made zero (exact in 8 bits), and decode logits are held to 1e-4 too."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.backends.cudnn.allow_tf32 = False
    return torch.device("cuda:0")


def _model(dev, layout, kv_heads=None, seed=0):
    from copy_on_write_sdm_b200.model import LanguageModel

    model = LanguageModel(vocab_size=97, maximum_sequence_length=200, layout=layout, width=64, heads=2, kv_heads=kv_heads, slots=64,
                          reads=8, writes=2, memory_heads=2, activation_dtype=torch.float32)
    model.initialize_role_keyed(seed)
    return model.to(dev).eval()


def _prompts(lengths, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 97, (n,), generator=gen) for n in lengths]


@pytest.mark.parametrize("layout,kv_heads", [("A", None), ("BBA", 2), ("BA", 1), ("BAB", 1), ("ABBA", 2)])
def test_ragged_requests_follow_the_full_forward(dev, layout, kv_heads):
    from copy_on_write_sdm_b200.paged import PagedServing

    model = _model(dev, layout, kv_heads)
    ends_in_attention = layout.rstrip("A").find("A") < 0
    if not ends_in_attention:
        for block in model.stack.attention_layers.values():
            with torch.no_grad():
                block.attention.qkv.weight[block.attention.width:] = 0
    serving = PagedServing(model, pages=24, sdm_growth_quantum_rows=64)
    ids = {}

    def check(logits, tolerance):
        for row, name in zip(logits, serving.requests):
            want = model(torch.tensor(ids[name], device=dev)[None])[0, -1]
            assert float((row - want).norm()) <= tolerance * float(want.norm()), (name, len(ids[name]))

    def admit(lengths, names, seed):
        before = list(serving.requests)
        prompts = _prompts(lengths, seed)
        logits = serving.admit(prompts, names)
        ids.update({name: p.tolist() for name, p in zip(names, prompts)})
        assert serving.requests[:len(before)] == before and logits.shape == (len(names), 97)
        for row, name in zip(logits, serving.requests[len(before):]):
            want = model(torch.tensor(ids[name], device=dev)[None])[0, -1]
            torch.testing.assert_close(row, want, atol=1e-4, rtol=1e-4)

    def step(seed):
        new = torch.randint(0, 97, (len(serving.requests),), generator=torch.Generator().manual_seed(seed))
        logits = serving.decode(new)
        for name, i in zip(serving.requests, new.tolist()):
            ids[name].append(i)
        check(logits, 2.0**-4 if ends_in_attention else 1e-4)

    admit([70, 1, 64, 64, 130], list("abcde"), 1)
    for s in range(3):
        step(10 + s)
    serving.release(["a", "d"])
    admit([5, 63], ["f", "g"], 2)
    for s in range(2):
        step(20 + s)
    serving.cache.validate_invariants()
    for state in serving.sdm.sdm_states:
        state.validate_invariants()
    assert serving.free_pages == int(serving.cache.free_count)
    assert serving.cache.lengths.tolist() == serving.lengths == [len(ids[n]) for n in serving.requests]
    serving.release(list(serving.requests))
    assert serving.free_pages == 24 and not serving.requests
    admit([9], ["h"], 3)
    step(30)


def test_decode_attends_over_what_the_cache_holds(dev):
    from copy_on_write_sdm_b200 import PagedKVCache
    from copy_on_write_sdm_b200.model import CausalSelfAttention

    torch.manual_seed(3)
    att = CausalSelfAttention(128, 4, kv_heads=2).to(dev).eval()
    lengths = [66, 3, 130]
    cache = PagedKVCache.allocate(requests=3, pages=8, kv_heads=2, head_width=32, max_blocks=3, layers=2, device=dev)
    plan = cache.resize(lengths, tokens=199)
    with torch.no_grad():
        att.prefill_packed(torch.randn(199, 128, device=dev), plan, cache, layer=1)
        tokens = torch.randn(3, 128, device=dev)
        plan = cache.resize([n + 1 for n in lengths], tokens=3)
        got = att.decode_packed(tokens, plan, cache, layer=1)
        q = att._project_packed(tokens)[0]
        for b, n in enumerate(lengths):
            p = torch.arange(n + 1, device=dev)
            slots = cache.block_tables[b, (p // 64).long()] * 64 + (p % 64).int()
            k, v = cache.read(slots, layer=1, dtype=torch.float32)
            k, v = (t.repeat_interleave(2, dim=1).transpose(0, 1).double() for t in (k, v))
            s = torch.softmax((k @ q[b].double()[:, :, None])[..., 0] / 32**0.5, -1)
            want = att.output((s[:, None] @ v)[:, 0].reshape(1, 128).float())
            torch.testing.assert_close(got[b:b + 1], want, atol=1e-5, rtol=1e-5)


def test_refusals(dev):
    from copy_on_write_sdm_b200.model import CausalSelfAttention
    from copy_on_write_sdm_b200.paged import PagedServing

    with pytest.raises(ValueError):
        CausalSelfAttention(64, 4, kv_heads=3)
    with pytest.raises(ValueError, match="attention layers"):
        PagedServing(_model(dev, "B"), pages=4)
    with pytest.raises(ValueError, match="eval"):
        PagedServing(_model(dev, "A").train(), pages=4)
    serving = PagedServing(_model(dev, "A"), pages=3, sdm_growth_quantum_rows=16)
    with pytest.raises(ValueError):
        serving.decode(torch.zeros(0, dtype=torch.int64))
    for prompts, names in ((_prompts([200], 0), ["a"]), (_prompts([3], 0), ["a", "b"]), (_prompts([3, 3], 0), ["a", "a"]),
                           (_prompts([201], 0), ["a"]), ([torch.zeros(0, dtype=torch.int64)], ["a"])):
        with pytest.raises(ValueError):
            serving.admit(prompts, names)
    serving.admit(_prompts([64, 128], 0), ["a", "b"])
    with pytest.raises(ValueError, match="name"):
        serving.admit(_prompts([1], 0), ["a"])
    with pytest.raises(ValueError, match="free pages"):
        serving.decode(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        serving.release(["c"])
    serving.release(["a"])
    assert serving.decode(torch.zeros(1, dtype=torch.int64)).shape == (1, 97)
