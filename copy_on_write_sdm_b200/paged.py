"""Continuous batching of requests of different lengths over a whole model: packed SDM
pools for its "B" layers (``FaithfulSDMDecodeState``) and one paged 8-bit K/V cache for
its "A" layers (``PagedKVCache``).

``FaithfulSDMDecodeState`` alone keeps, as the reference does
(copy_on_write_sdm/inference.py:293-306), a cache of the batch's full capacity per
request and attention layer in the activation type, and admits cohorts of one length.  Here
prompts of any lengths are admitted together: attention layers run them packed, SDM
layers by groups of equal length, and a request's K/V holds pages only for its own tokens.
"""

from __future__ import annotations

from typing import Sequence

import torch

from .inference import FaithfulSDMDecodeState, _decode_faithful_sdm_layer
from .kv_cache import PAGE_TOKENS, PagedKVCache
from .model import LanguageModel


class PagedServing:
    """A live batch over one ``LanguageModel`` in eval mode.

    ``requests`` lists the live requests' names in batch order; ids go in and logits
    come out in that order.  ``pages`` is the K/V pool's size in pages of 64 tokens, shared by
    all requests; one page holds 64 tokens of every attention layer.

    An ``admit`` that raises leaves the batch as it was.  A ``decode`` or ``release`` that raises on its way through the
    layers does not, as the pools have taken some of its writes: every later call then raises ``RuntimeError``.
    """

    def __init__(self, model: LanguageModel, *, pages: int, sdm_growth_quantum_rows: int = 1024) -> None:
        if model.training:
            raise ValueError("paged serving requires model.eval()")
        if sdm_growth_quantum_rows <= 0:
            raise ValueError("paged serving requires a growth quantum for the SDM pools")
        stack = model.stack
        self.model, self.sdm_growth_quantum_rows = model, sdm_growth_quantum_rows
        self.requests: list[object] = []
        self.lengths: list[int] = []
        self.sdm: FaithfulSDMDecodeState | None = None
        self._unusable: str | None = None
        attention = [stack.attention_layers[str(i)].attention for i, kind in enumerate(stack.layout) if kind == "A"]
        if not attention:
            raise ValueError("paged serving is for models with attention layers")
        device = model.token_embedding.weight.device
        self.cache = PagedKVCache.allocate(
            requests=0, pages=pages, kv_heads=attention[0].kv_heads, head_width=attention[0].head_width,
            max_blocks=-(-model.maximum_sequence_length // PAGE_TOKENS), layers=len(attention), device=device)

    @property
    def free_pages(self) -> int:
        """Free K/V pages, from the host's record of the lengths."""
        return self.cache.pages - sum(-(-n // PAGE_TOKENS) for n in self.lengths)

    def _check_usable(self) -> None:
        if self._unusable is not None:
            raise RuntimeError(f"paged serving is unusable: {self._unusable} failed part way")

    def _ids(self, ids: torch.Tensor) -> torch.Tensor:
        """Token ids on the model's device; those on the host are checked, as one outside the vocabulary faults there."""
        if ids.dtype not in (torch.int32, torch.int64):
            raise ValueError("token ids must be int32 or int64")
        if not ids.is_cuda and ids.numel() and not 0 <= int(ids.min()) <= int(ids.max()) < self.model.token_embedding.num_embeddings:
            raise ValueError("token ids lie outside the vocabulary")
        return ids.to(self.cache.device)

    @torch.no_grad()
    def admit(self, prompts: Sequence[torch.Tensor], names: Sequence[object]) -> torch.Tensor:
        """Prefill prompts (vectors of ids, any lengths) and add them to the batch, ordered by
        length after the live requests; the logits after each prompt's last token, in batch order."""
        self._check_usable()
        if len(prompts) != len(names) or len(set(names)) != len(names) or set(names) & set(self.requests):
            raise ValueError("admitted requests need one new name each")
        if not prompts:
            return self.model.output.weight.new_zeros(0, self.model.output.out_features)
        if any(p.ndim != 1 or not 1 <= p.shape[0] <= self.model.maximum_sequence_length for p in prompts):
            raise ValueError("prompts must be vectors of 1 to maximum_sequence_length ids")
        order = sorted(range(len(prompts)), key=lambda i: prompts[i].shape[0])
        counts = [prompts[i].shape[0] for i in order]
        if sum(-(-n // PAGE_TOKENS) for n in counts) > self.free_pages:
            raise ValueError("the K/V cache has too few free pages for the admitted prompts")
        ids = torch.cat([self._ids(prompts[i]) for i in order])
        live, cache, sdm = len(self.requests), self.cache, self.sdm
        try:
            logits = self._admit(ids, counts, live)
        except BaseException:
            self._unusable = "an admission and its undoing"
            if self.cache is not cache:  # pages and rows taken so far go back
                self.cache.resize(self.lengths + [0] * len(counts), tokens=0)
                self.cache = self.cache.with_requests(range(live))
            self.sdm = sdm
            if sdm is not None:
                if sdm.batch > live:
                    sdm.release_and_compact(list(range(live, sdm.batch)))
                heads = [self.model.stack.sdm_layers[str(i)].memory_heads for i in sdm.sdm_layer_positions]
                if [state.banks for state in sdm.sdm_states] != [live * h for h in heads]:
                    raise
            self._unusable = None
            raise
        self.requests += [names[i] for i in order]
        self.lengths += counts
        return logits

    def _admit(self, ids: torch.Tensor, counts: list[int], live: int) -> torch.Tensor:
        model, stack = self.model, self.model.stack
        self.cache = self.cache.with_requests(range(live), new=len(counts))
        plan = self.cache.resize(self.lengths + counts, tokens=sum(counts))
        tokens = model._embed(ids, plan.positions.long())

        groups: list[tuple[int, int, int]] = []  # first token, requests, length
        at = 0
        for n in counts:
            if groups and groups[-1][2] == n:
                groups[-1] = (groups[-1][0], groups[-1][1] + 1, n)
            else:
                groups.append((at, 1, n))
            at += n
        pools: list[list] = [[] for _ in groups]
        layer = 0
        for i, kind in enumerate(stack.layout):
            if kind == "A":
                block = stack.attention_layers[str(i)]
                tokens = tokens + block.attention.prefill_packed(tokens, plan, self.cache, layer=layer)
                tokens = tokens + block.mlp(tokens)
                layer += 1
                continue
            mixed = torch.empty_like(tokens)
            for (first, many, n), kept in zip(groups, pools):
                out, pool = stack.sdm_layers[str(i)].prefill(tokens[first:first + many * n].view(many, n, -1),
                                                             growth_quantum_rows=self.sdm_growth_quantum_rows)
                mixed[first:first + many * n] = out.reshape(many * n, -1)
                kept.append(pool)
            tokens = tokens + mixed
            tokens = tokens + stack.sdm_mlps[str(i)](tokens)
        b_layers = tuple(i for i, kind in enumerate(stack.layout) if kind == "B")
        for (_, many, n), kept in zip(groups, pools):
            cohort = FaithfulSDMDecodeState(
                layout=stack.layout, position=n, capacity=model.maximum_sequence_length, activation_dtype=tokens.dtype,
                active_sequences=torch.ones(many, device=ids.device, dtype=torch.bool), sdm_layer_positions=b_layers,
                sdm_states=tuple(kept), dense_keys=(), dense_values=())
            if self.sdm is None:
                self.sdm = cohort
            else:
                self.sdm.admit(cohort)
        ends = plan.starts[live + 1:].long() - 1
        return model.output(model.final_norm(tokens[ends]))

    @torch.no_grad()
    def decode(self, ids: torch.Tensor) -> torch.Tensor:
        """One more token of every live request, ``[requests]`` ids to ``[requests, vocabulary]`` logits."""
        self._check_usable()
        count = len(self.requests)
        if ids.shape != (count,) or count == 0:
            raise ValueError(f"decode ids must be [{count}], one for each live request")
        model = self.model
        if max(self.lengths) >= model.maximum_sequence_length:
            raise ValueError("sequence exceeds maximum_sequence_length")
        if sum(n % PAGE_TOKENS == 0 for n in self.lengths) > self.free_pages:
            raise ValueError("the K/V cache has too few free pages for the next token")
        ids = self._ids(ids)
        self._unusable = "a decode step"
        tokens = self._decode(ids, count)
        self._unusable = None
        self.lengths = [n + 1 for n in self.lengths]
        return model.output(model.final_norm(tokens))

    def _decode(self, ids: torch.Tensor, count: int) -> torch.Tensor:
        model, stack = self.model, self.model.stack
        plan = self.cache.resize(self.cache.lengths + 1, tokens=count)
        tokens = model._embed(ids, plan.positions.long())
        a = b = 0
        for i, kind in enumerate(stack.layout):
            if kind == "A":
                block = stack.attention_layers[str(i)]
                tokens = tokens + block.attention.decode_packed(tokens, plan, self.cache, layer=a)
                tokens = tokens + block.mlp(tokens)
                a += 1
            else:
                tokens = _decode_faithful_sdm_layer(stack.sdm_layers[str(i)], tokens[:, None], self.sdm.sdm_states[b],
                                                    mlp=stack.sdm_mlps[str(i)])[:, 0]
                b += 1
        if self.sdm.positions is None:
            self.sdm.position += 1
        else:
            self.sdm.positions.add_(1)
            self.sdm.position += 1
        return tokens

    @torch.no_grad()
    def release(self, names: Sequence[object]) -> None:
        """Finish requests: their pool rows and K/V pages return, the others keep their order."""
        self._check_usable()
        gone = [self.requests.index(name) for name in names]
        if len(set(gone)) != len(gone):
            raise ValueError("released requests are named twice")
        if not gone:
            return
        keep = [i for i in range(len(self.requests)) if i not in set(gone)]
        self._unusable = "a release"
        self.cache.resize([0 if i in set(gone) else n for i, n in enumerate(self.lengths)], tokens=0)
        self.cache = self.cache.with_requests(keep)
        self.sdm.release_and_compact(gone)
        self.requests = [self.requests[i] for i in keep]
        self.lengths = [self.lengths[i] for i in keep]
        if not keep:
            self.sdm = None
        self._unusable = None

    def validate_invariants(self) -> None:
        """Raise on any device error so far, of attention or of the pools, and where pages or rows are lost (synchronises)."""
        self.cache.validate_invariants()
        for state in () if self.sdm is None else self.sdm.sdm_states:
            state.validate_invariants()
        if self.cache.lengths.tolist() != self.lengths:
            raise AssertionError("the K/V cache's lengths are not the requests'")

    def storage_bytes(self) -> dict[str, int]:
        """The SDM state's bytes (``FaithfulSDMDecodeState``'s keys) and the K/V cache's."""
        sdm = {} if self.sdm is None else self.sdm.storage_bytes()
        return {**sdm, **self.cache.storage_bytes()}
