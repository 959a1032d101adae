"""What is measured of the attention layers' serving operators, and their plain forms.

Four operators of one path: a prompt's attention (``prompt_attention``), the pages its
tokens go to (``PagedKVCache.resize``), the 8-bit cache that keeps its keys and values
(``store`` / ``read``) and the attention of single tokens over that cache (``attend``).

Formulas, for pages of 64 tokens:

* pages: a request of length n holds ceil(n / 64) pages.  Moving every request from its
  length to a target frees the pages past a shorter target and then takes pages for the
  longer ones, from one stack: the r-th page taken (request by request, block by block) is
  ``free_pages[free_count - 1 - r]``, and freed pages go back so that the first freed is
  the next taken.  A new token's slot is ``64 * page + position % 64``.
* store: per page and head, the scale is the smallest power of two 2^e, e >= -64, with
  max|x| <= 448 * 2^e over the page's tokens (a page that held tokens keeps its scale where that is
  larger, and its codes are rounded again to a larger one); codes are x / scale rounded to
  e4m3, to nearest even.  Read back: code * scale.
* attend: o = softmax(scale * q . K) V over the request's cached tokens, per query head,
  ``heads / kv_heads`` query heads sharing one key and value head; scale = 1 / sqrt(width).
* prompt: the same over the tokens up to the query's own, in its own sequence.
"""

import math

import torch

own = False

PAGE = 64
LARGEST = 448.0  # largest finite e4m3 value
LEAST = -64  # least exponent of a scale
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of a serving batch: every request grows by its next token
        dict(name="pages_step", op="pages", requests=64, shortest=64, longest=4096, kept="step"),
        # admission: every second request is new and brings its whole prompt, the others their next token
        dict(name="pages_admit", op="pages", requests=1024, shortest=64, longest=4096, kept="half"),
        # the K/V of one decode token of a serving batch into pages that hold tokens already
        dict(name="store_step", op="store", requests=64, shortest=1, longest=512, kept="step", kv_heads=8, width=128, type="bf16"),
        # the attention layer of the fp32 model: four heads of 32, sixteen prompts of 256
        dict(name="store_model", op="store", requests=16, shortest=256, longest=256, kept="none", kv_heads=4, width=32, type="f32"),
        # whole prompts of a continuous batch
        dict(name="store_prompts", op="store", requests=32, shortest=64, longest=4096, kept="none", kv_heads=8, width=128, type="bf16"),
        # the fp32 model's prefill: sixteen prompts of 256
        dict(name="prompt_model", op="prompt", requests=16, shortest=256, longest=256, heads=4, kv_heads=4, width=32, type="f32"),
        # a continuous batch's prompts, short and long ones packed
        dict(name="prompt_batch", op="prompt", requests=32, shortest=64, longest=2048, heads=16, kv_heads=4, width=64, type="bf16"),
        # odd lengths from one token on, seven query heads to a key head
        dict(name="prompt_odd", op="prompt", requests=21, shortest=1, longest=777, heads=14, kv_heads=2, width=96, type="f16"),
        # long prompts
        dict(name="prompt_long", op="prompt", requests=2, shortest=8192, longest=8192, heads=32, kv_heads=8, width=128, type="bf16"),
        # the fp32 model's decode token: sixteen requests between prefix and end
        dict(name="attend_model", op="attend", requests=16, shortest=256, longest=512, heads=4, kv_heads=4, width=32, type="f32"),
        # a serving batch of requests of all lengths
        dict(name="attend_batch", op="attend", requests=64, shortest=64, longest=4096, heads=32, kv_heads=8, width=128, type="bf16"),
        # few requests, each with a long cache
        dict(name="attend_long", op="attend", requests=4, shortest=65536, longest=65536, heads=32, kv_heads=8, width=128, type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("pages", "store", "prompt", "attend"))
    case = dict(op=op)
    if op == "pages":
        longest = _log(rng, 64, 4096)
        case.update(requests=_log(rng, 4, 1024), shortest=_log(rng, 1, longest), longest=longest, kept=rng.choice(("step", "half", "none")))
        return case
    case.update(width=rng.choice((32, 64, 96, 128)), type=rng.choice(("bf16", "bf16", "f16", "f32")))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    if op == "store":
        longest = _log(rng, 16, 4096)
        case.update(requests=_log(rng, 4, 32), shortest=_log(rng, 1, longest), longest=longest,
                    kept=rng.choice(("step", "half", "none")), kv_heads=kv_heads)
        return case
    case.update(heads=kv_heads * rng.choice((1, 2, 3, 4, 7, 8)), kv_heads=kv_heads)
    if op == "prompt":
        longest = _log(rng, 16, 2048)
        most = max(1, min(32, int(2.0**32 / (case["heads"] * longest * longest))))
    else:
        longest = _log(rng, 64, 65536)
        most = max(1, min(256, int(2.0**28 / (kv_heads * 128 * longest))))
    case.update(requests=_log(rng, 1, most), shortest=_log(rng, 1, longest), longest=longest)
    return case


def _lengths(case):
    """The requests' lengths: spread over [shortest, longest] without order, the longest among them."""
    low, high, count = case["shortest"], case["longest"], case["requests"]
    got = [low + int((high - low + 1) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(count)]
    got[count // 2] = high
    return got


def _kept(case, lengths):
    """What of each request is there before the call: all but the last token, nothing, or one after the other."""
    how = case["kept"]
    return [n - 1 if how == "step" or (how == "half" and i % 2) else 0 for i, n in enumerate(lengths)]


def _blocks(n):
    return -(-n // PAGE)


def work(case):
    lengths = _lengths(case)
    total = sum(lengths)
    if case["op"] == "pages":
        kept = _kept(case, lengths)
        moved = sum(_blocks(n) - _blocks(k) for n, k in zip(lengths, kept))
        new = total - sum(kept)
        # both moves read targets and lengths and write lengths; pages leave the tables for the stack and come back;
        # starts, slots and positions are written
        return {"bytes": 4.0 * (2 * 3 * len(lengths) + 4 * moved + len(lengths) + 1 + 2 * new), "flops": 0}
    size = TYPES[case["type"]].itemsize
    row = case["kv_heads"] * case["width"]
    if case["op"] == "store":
        kept = _kept(case, lengths)
        back = sum(n - k // PAGE * PAGE for n, k in zip(lengths, kept))
        new = total - sum(kept)
        # new tokens read and their codes written; the touched pages' tokens read and given back
        return {"bytes": 2.0 * row * (new * (size + 1) + back * (1 + size)) + 4 * back, "flops": 0}
    wide = case["heads"] * case["width"]
    if case["op"] == "prompt":
        return {"bytes": 2.0 * size * total * (wide + row), "flops": 4.0 * wide * sum(n * (n + 1) // 2 for n in lengths)}
    pages = sum(_blocks(n) for n in lengths)
    return {"bytes": 2.0 * total * row + pages * (8.0 * case["kv_heads"] + 4) + 2.0 * size * len(lengths) * wide, "flops": 4.0 * wide * total}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)


def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = _lengths(case)
    dtype = TYPES[case["type"]]
    total, width = sum(lengths), case["width"]
    x = {"lengths": lengths}
    # keys of some heads are larger than those of others, as trained projections' are
    loud = torch.rand(case["kv_heads"], 1, generator=gen, device="cuda") + 0.5
    x["k"] = (_normal(gen, (total, case["kv_heads"], width), dtype) * loud).to(dtype)
    x["v"] = _normal(gen, (total, case["kv_heads"], width), dtype)
    if case["op"] == "prompt":
        x["q"] = _normal(gen, (total, case["heads"], width), dtype)
    elif case["op"] == "attend":
        x["q"] = _normal(gen, (len(lengths), case["heads"], width), dtype)
    return x


def _starts(counts):
    got = [0]
    for n in counts:
        got.append(got[-1] + n)
    return got


def prepare(case, seed):
    op = case["op"]
    state = {"op": op}
    if op == "pages":
        return _prepare_pages(case, seed, state)
    x = _inputs(case, seed)
    lengths = x["lengths"]
    starts = _starts(lengths)
    if op == "prompt":
        state.update(q=x["q"], k=x["k"], v=x["v"], starts=_ints(starts), longest=max(lengths))
        return state
    kept = _kept(case, lengths) if op == "store" else [0] * len(lengths)
    tokens = torch.arange(starts[-1], device="cuda")
    request = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), torch.tensor(lengths, device="cuda"))
    position = tokens - torch.tensor(starts[:-1], device="cuda")[request]
    old = position < torch.tensor(kept, device="cuda")[request]
    new = ~old
    count = sum(_blocks(n) for n in lengths)
    if own:
        from copy_on_write_sdm_b200 import PagedKVCache

        cache = PagedKVCache.allocate(requests=len(lengths), pages=count, kv_heads=case["kv_heads"], head_width=case["width"],
                                      max_blocks=_blocks(max(lengths)), device="cuda")
        if any(kept):
            cache.store(x["k"][old], x["v"][old], cache.resize(_ints(kept), tokens=sum(kept)))
        plan = cache.resize(_ints(lengths), tokens=starts[-1] - sum(kept))
        if op == "attend":
            cache.store(x["k"], x["v"], plan)
            state.update(q=x["q"], cache=cache)
            return state
        # the slots of all tokens of the pages that the call writes to
        back = position >= (torch.tensor(kept, device="cuda") // PAGE * PAGE)[request]
        pages = cache.block_tables.long()[request[back], position[back] // PAGE]
        slots = (pages * PAGE + position[back] % PAGE).int()
        state.update(k=x["k"][new].contiguous(), v=x["v"][new].contiguous(), cache=cache, plan=plan, slots=slots, dtype=TYPES[case["type"]])
        return state
    # plain: pages in the order of requests and blocks
    first = torch.tensor(_starts([_blocks(n) for n in lengths]), device="cuda")
    slot = (first[:-1][request] + position // PAGE) * PAGE + position % PAGE
    for name in ("k", "v"):
        codes = torch.zeros(count * PAGE, case["kv_heads"], case["width"], dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.zeros(count, case["kv_heads"], device="cuda")
        stored = old if op == "store" else torch.ones_like(old)
        state[name + "_codes"], state[name + "_scales"] = _plain_store(codes, scales, x[name][stored], slot[stored])
    if op == "attend":
        tables = torch.arange(max(_blocks(n) for n in lengths), device="cuda") + first[:-1, None]
        state.update(q=x["q"], tables=tables.clamp_(max=count - 1), lengths=torch.tensor(lengths, device="cuda"))
        return state
    back = position >= (torch.tensor(kept, device="cuda") // PAGE * PAGE)[request]
    state.update(k=x["k"][new].contiguous(), v=x["v"][new].contiguous(), slot=slot[new], back=slot[back], dtype=TYPES[case["type"]])
    return state


def _prepare_pages(case, seed, state):
    lengths = _lengths(case)
    kept = _kept(case, lengths)
    gen = torch.Generator().manual_seed(seed)
    # the seed says in which order the requests of these lengths stand
    order = torch.randperm(len(lengths), generator=gen).tolist()
    lengths, kept = [lengths[i] for i in order], [kept[i] for i in order]
    count = sum(_blocks(n) for n in lengths) + 7
    blocks = _blocks(max(lengths))
    state.update(low=_ints(kept), high=_ints(lengths), tokens=sum(lengths) - sum(kept))
    if own:
        from copy_on_write_sdm_b200 import PagedKVCache

        cache = PagedKVCache.allocate(requests=len(lengths), pages=count, kv_heads=1, head_width=32, max_blocks=blocks, device="cuda")
        cache.resize(state["low"], tokens=sum(kept))
        cache.resize(state["high"], tokens=state["tokens"])
        state.update(cache=cache)
        return state
    state.update(tables=torch.full((len(lengths), blocks), -1, dtype=torch.int32, device="cuda"),
                 lengths=_ints([0] * len(lengths)), free_pages=torch.arange(count, dtype=torch.int32, device="cuda"),
                 free_count=torch.tensor(count, dtype=torch.int32, device="cuda"))
    _plain_resize(state, state["low"], sum(kept))
    _plain_resize(state, state["high"], state["tokens"])
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------


def run(state):
    op = state["op"]
    if own:
        return _run_own(op, state)
    if op == "pages":
        _plain_resize(state, state["low"], 0)
        starts, slots, positions = _plain_resize(state, state["high"], state["tokens"])
        return {"starts": starts, "slots": slots, "positions": positions, "tables": state["tables"], "lengths": state["lengths"],
                "free_pages": state["free_pages"], "free_count": state["free_count"]}
    if op == "store":
        return [_plain_read(*_plain_store(state[n + "_codes"], state[n + "_scales"], state[n], state["slot"]), state["back"], state["dtype"])
                for n in ("k", "v")]
    if op == "attend":
        return _plain_attend(state)
    return _plain_prompt(state)


def _run_own(op, state):
    from copy_on_write_sdm_b200 import prompt_attention

    if op == "pages":
        cache = state["cache"]
        cache.resize(state["low"], tokens=0)
        plan = cache.resize(state["high"], tokens=state["tokens"])
        return {"starts": plan.starts, "slots": plan.slots, "positions": plan.positions, "tables": cache.block_tables,
                "lengths": cache.lengths, "free_pages": cache.free_pages, "free_count": cache.free_count}
    if op == "store":
        state["cache"].store(state["k"], state["v"], state["plan"])
        return list(state["cache"].read(state["slots"], dtype=state["dtype"]))
    if op == "attend":
        return state["cache"].attend(state["q"])
    return prompt_attention(state["q"], state["k"], state["v"], state["starts"])


def _plain_resize(state, target, tokens):
    """Every request to its target length: (starts, slots, positions) of its new tokens; tables, lengths and stack change in place."""
    tables, lengths, stack, count = state["tables"], state["lengths"], state["free_pages"], state["free_count"]
    block = torch.arange(tables.shape[1], device="cuda")
    had, wants = (lengths[:, None] + PAGE - 1) // PAGE, (target[:, None] + PAGE - 1) // PAGE
    freed = (block >= wants) & (block < had)
    pages = tables[freed]
    at = count.long() + pages.numel() - 1 - torch.arange(pages.numel(), device="cuda")
    stack[at] = pages
    tables[freed] = -1
    count += pages.numel()
    taken = (block >= had) & (block < wants)
    rank = torch.arange(int(taken.sum()), device="cuda")
    tables[taken] = stack[count.long() - 1 - rank]
    count -= rank.numel()
    new = (target - lengths).clamp(min=0)
    starts = torch.cat((new.new_zeros(1), new.cumsum(0, dtype=torch.int32)))
    request = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=tokens)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) - starts[request] + lengths[request]
    slots = tables[request, positions.long() // PAGE] * PAGE + positions % PAGE
    lengths.copy_(target)
    return starts, slots, positions


def _plain_store(codes, scales, x, slot):
    """Codes [slots, heads, width] and scales [pages, heads] after x [tokens, heads, width] went to its slots."""
    x = x.float()
    heads = x.shape[1]
    page = slot // PAGE
    most = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(most > 0, exponent - 9 + (mantissa > 0.875), LEAST).clamp(min=LEAST)
    need = torch.ldexp(torch.ones_like(most), exponent)
    touched = torch.zeros(scales.shape[0], 1, dtype=torch.bool, device="cuda").index_fill_(0, page, True)
    grown = torch.where(touched, torch.maximum(scales, need), scales)
    values = codes.float().view(-1, PAGE, heads, x.shape[2])
    again = torch.where(grown > 0, scales / grown, 0.0)[:, None, :, None]
    after = (values * again).view_as(codes)
    after[slot] = x / grown[page][:, :, None]
    return after.to(torch.float8_e4m3fn), grown


def _plain_read(codes, scales, slot, dtype):
    values = codes.view(torch.uint8)[slot].view(torch.float8_e4m3fn).float()
    return (values * scales[slot // PAGE][:, :, None]).to(dtype)


def _plain_attend(state):
    q, tables, lengths = state["q"], state["tables"], state["lengths"]
    requests, heads, width = q.shape
    slots = (tables[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")).view(requests, -1)
    k = _plain_read(state["k_codes"], state["k_scales"], slots.view(-1), torch.float32).view(requests, slots.shape[1], -1, width)
    v = _plain_read(state["v_codes"], state["v_scales"], slots.view(-1), torch.float32).view(requests, slots.shape[1], -1, width)
    grouped = q.float().view(requests, k.shape[2], -1, width)
    scores = torch.matmul(grouped, k.permute(0, 2, 3, 1)) * width**-0.5  # [requests, kv heads, group, tokens]
    hidden = torch.arange(slots.shape[1], device="cuda") >= lengths[:, None]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    out = torch.matmul(scores, v.permute(0, 2, 1, 3)) / scores.sum(-1, keepdim=True)
    return out.reshape(requests, heads, width).to(q.dtype)


def _plain_prompt(state):
    q, k, v, starts, longest = (state[n] for n in ("q", "k", "v", "starts", "longest"))
    total, heads, width = q.shape
    kv_heads = k.shape[1]
    starts = starts.long()
    place = torch.arange(longest, device="cuda")
    there = place < (starts[1:] - starts[:-1])[:, None]  # [requests, longest]
    token = torch.where(there, starts[:-1, None] + place, 0)
    grouped = q.float()[token].view(*token.shape, kv_heads, heads // kv_heads, width).permute(0, 2, 3, 1, 4)
    keys = k.float()[token].permute(0, 2, 3, 1)[:, :, None]
    values = v.float()[token].permute(0, 2, 1, 3)[:, :, None]
    scores = torch.matmul(grouped * width**-0.5, keys)  # [requests, kv heads, group, queries, keys]
    scores.masked_fill_(place > place[:, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    out = torch.matmul(scores, values)
    out /= scores.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4)[there].reshape(total, heads, width).to(q.dtype)


# ---------------------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------------------


def _e4m3(x):
    """The e4m3 value nearest to x, ties to the even one; |x| <= 448."""
    _, exponent = torch.frexp(x)
    # x = m 2^exponent, m in [0.5, 1): four significant bits, the least normal value is 2^-6
    step = torch.ldexp(torch.ones_like(x), exponent.clamp(min=-5) - 4)
    return torch.round(x / step) * step


def _exact_pages(x, kept, n):
    """One request's x [n, heads, width] as a cache holds it: stored up to `kept`, then the rest; 64 bits."""

    def put(part, scale, held):
        most = part.abs().amax((0, 2))
        exponent = torch.where(most > 0, torch.ceil(torch.log2(most.clamp(min=1e-300) / LARGEST)), float(LEAST)).clamp(min=LEAST)
        for off in (-1.0, 0.0):  # the least power that holds, whatever log2 rounded
            less = exponent + off
            exponent = torch.where((less >= LEAST) & (most <= LARGEST * torch.exp2(less)), torch.minimum(less, exponent), exponent)
        exponent = torch.where(most > LARGEST * torch.exp2(exponent), exponent + 1, exponent)
        need = torch.exp2(exponent)
        now = need if scale is None else torch.maximum(scale, need)
        got = _e4m3(part / now[:, None])
        return (got if held is None else torch.cat((_e4m3(held * (scale / now)[:, None]), got))), now

    got = []
    for begin in range(0, n, PAGE):
        page = x[begin:min(n, begin + PAGE)].double()
        there = min(max(kept - begin, 0), page.shape[0])
        held, scale = put(page[:there], None, None) if there else (None, None)
        if there < page.shape[0]:
            held, scale = put(page[there:], scale, held)
        got.append(held * scale[:, None])
    return torch.cat(got) if got else x.double()


def _exact_full(x):
    """x [n, heads, width], stored in one go, as a cache holds it; 64 bits."""
    n, heads, width = x.shape
    padded = torch.zeros(_blocks(n) * PAGE, heads, width, dtype=torch.float64, device=x.device)
    padded[:n] = x
    padded = padded.view(-1, PAGE, heads, width)
    most = padded.abs().amax((1, 3))
    mantissa, exponent = torch.frexp(most / LARGEST)  # exact enough: 448 = 7 * 64, in 53 bits
    exponent = torch.where(most > 0, exponent - (mantissa == 0.5).int(), LEAST).clamp(min=LEAST)
    scale = torch.exp2(exponent.double())[:, None, :, None]
    return (_e4m3(padded / scale) * scale).view(-1, heads, width)[:n]


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None  # whole numbers
    x = _inputs(case, seed)
    lengths = x["lengths"]
    starts = _starts(lengths)
    if op == "store":
        kept = _kept(case, lengths)
        if sum(_blocks(n) for n in lengths) > 4000:
            return None
        got = []
        for name in ("k", "v"):
            parts = []
            for b, n in enumerate(lengths):
                rows = x[name][starts[b]:starts[b + 1]]
                begin = kept[b] // PAGE * PAGE
                parts.append(_exact_pages(rows[begin:], kept[b] - begin, n - begin) if kept[b] else _exact_full(rows))
            got.append(torch.cat(parts))
        return got
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        k, v = x["k"][starts[b]:starts[b + 1]], x["v"][starts[b]:starts[b + 1]]
        k, v = (_exact_full(k), _exact_full(v)) if op == "attend" else (k.double(), v.double())
        for h in range(kv_heads):
            group = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            if op == "attend":
                p = torch.softmax(x["q"][b, group].double() @ kt / math.sqrt(width), -1)
                out[b, group] = p @ vh
                continue
            for begin in range(0, n, 2048):
                end = min(n, begin + 2048)
                s = x["q"][starts[b] + begin:starts[b] + end, group].double().transpose(0, 1) @ kt[:, :end] / math.sqrt(width)
                later = torch.arange(end, device="cuda") > torch.arange(begin, end, device="cuda")[:, None]
                p = torch.softmax(s.masked_fill_(later, float("-inf")), -1)
                out[starts[b] + begin:starts[b] + end, group] = (p @ vh[:end]).transpose(0, 1)
    return out
