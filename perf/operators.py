"""Cases of the decoding operators: attention of one new token over a paged key-value cache, writing prompts into its pages, forking and
compacting the pages, and one step of a beam search.  `own` selects between the plain torch form and the framework's kernels
(multimodal_amd.ops); both compute the same outputs from the same inputs.

The plain forms use elementary torch operations in 32 bits (64 for the beam search, where two candidates may lie next to each other)."""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one image being captioned greedily by the CoCa L/14 text decoder (12 heads of 64, at most 77 tokens): a launch-bound step
        {"name": "attend caption", "op": "attend", "rows": 1, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "length": 40, "spread": "same", "new": True, "dtype": "bf16"},
        # a serving batch whose sequences are of very different ages, the same heads
        {"name": "attend ragged", "op": "attend", "rows": 61, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "length": 8192, "spread": "log", "new": True, "dtype": "bf16"},
        # few long sequences, four query heads to a key head
        {"name": "attend long", "op": "attend", "rows": 4, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "length": 65536, "spread": "same", "new": True, "dtype": "bf16"},
        # cross-attention over states that are kept in float32 (nothing is stored by the step), odd counts, a page that is no power of two
        {"name": "attend fp32", "op": "attend", "rows": 13, "heads": 6, "kv_heads": 2, "dim": 96, "page": 24, "length": 2999, "spread": "log", "new": False, "dtype": "fp32"},
        # 32 captions of full length written behind nothing
        {"name": "append captions", "op": "append", "rows": 32, "kv_heads": 12, "dim": 64, "page": 16, "tokens": 77, "spread": "same", "dtype": "bf16"},
        # long prompts of different lengths, padded to the longest
        {"name": "append prompts", "op": "append", "rows": 23, "kv_heads": 8, "dim": 128, "page": 32, "tokens": 4001, "spread": "log", "dtype": "bf16"},
        # a beam search over captions between two tokens: 32 images, 5 beams, all 12 layers of a CoCa L/14 decoder in a page
        {"name": "fork captions", "op": "fork", "groups": 32, "beams": 5, "kept": 2, "length": 33, "blocks": 288, "dim": 64, "page": 16, "dtype": "bf16"},
        # the same over long texts with large pages
        {"name": "fork long", "op": "fork", "groups": 48, "beams": 8, "kept": 3, "length": 1500, "blocks": 64, "dim": 128, "page": 64, "dtype": "bf16"},
        # a small pool after a few sequences ended
        {"name": "compact small", "op": "compact", "pages": 250, "live": 97, "moves": 31, "rows": 16, "slots": 12, "blocks": 288, "dim": 64, "page": 16, "dtype": "bf16"},
        # a large pool before it is cut down
        {"name": "compact large", "op": "compact", "pages": 12000, "live": 5000, "moves": 2900, "rows": 200, "slots": 40, "blocks": 96, "dim": 64, "page": 16, "dtype": "bf16"},
        # one image, five beams over the CLIP vocabulary
        {"name": "beam one image", "op": "beam", "groups": 1, "beams": 5, "vocab": 49408, "tokens": 77, "step": 20, "penalty": 1.0, "dtype": "fp32"},
        # a captioning batch
        {"name": "beam batch", "op": "beam", "groups": 128, "beams": 4, "vocab": 49408, "tokens": 77, "step": 31, "penalty": 0.0, "dtype": "fp32"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    case = _drawn(rng)
    while work(case)["bytes"] > 1.0e9:
        case = _drawn(rng)
    return case


def _drawn(rng):
    op = rng.choice(["attend", "attend", "append", "fork", "compact", "beam"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    dim = rng.choice([64, 96, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "attend":
        kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        length = _log_int(rng, 1, 32768)
        size = {"bf16": 2, "fp32": 4}[dtype]
        rows = _log_int(rng, 1, 256)
        while rows > 1 and rows * length * kv * dim * size * 2 > 9e8:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page, "length": length,
                "spread": rng.choice(["same", "log"]), "new": rng.random() < 0.7, "dtype": dtype}
    if op == "append":
        tokens = _log_int(rng, 1, 4001)
        kv = rng.choice([1, 2, 4, 6, 8, 12])
        rows = max(1, min(_log_int(rng, 1, 128), 90000 // tokens))
        return {"op": op, "rows": rows, "kv_heads": kv, "dim": dim, "page": page, "tokens": tokens, "spread": rng.choice(["same", "log"]), "dtype": dtype}
    if op == "fork":
        beams = rng.randint(1, 10)
        groups = _log_int(rng, 1, 40)
        length = _log_int(rng, 1, 1500)
        blocks = rng.choice([2, 8, 48, 64])
        return {"op": op, "groups": groups, "beams": beams, "kept": rng.randint(1, beams), "length": length, "blocks": blocks, "dim": dim, "page": rng.choice([8, 16, 24, 32, 64]), "dtype": dtype}
    if op == "compact":
        pages = _log_int(rng, 20, 12000)
        live = rng.randint(1, pages - 1)
        return {"op": op, "pages": pages, "live": live, "moves": rng.randint(0, min(live, pages - live)), "rows": rng.randint(1, 200), "slots": rng.randint(1, 60),
                "blocks": rng.choice([2, 8, 24, 48]), "dim": 64, "page": rng.choice([8, 16]), "dtype": dtype}
    beams = rng.randint(1, 12)
    vocab = rng.choice([49408, 30522, 8192, 50021, 997, 101])
    step = rng.randint(0, 60)
    return {"op": op, "groups": _log_int(rng, 1, 96 if beams < 5 else 40), "beams": beams, "vocab": vocab, "tokens": rng.choice([64, 77, 128]), "step": step,
            "penalty": rng.choice([0.0, 0.6, 1.0]), "dtype": dtype}


def _lengths(case, most):
    """The lengths of a case's rows, the longest among them: all the same, or spread evenly over their logarithm from nothing on."""
    rows = case["rows"]
    if case["spread"] == "same" or rows == 1:
        return [most] * rows
    rng = random.Random(rows * 1000003 + most)
    return [most] + [int(math.exp(rng.uniform(0.0, math.log(most + 1)))) - 1 for _ in range(rows - 1)]


def _shuffled(values, gen, device):
    v = torch.tensor(values, dtype=torch.int32, device=device)
    return v[torch.randperm(len(values), generator=gen, device=device)]


def _table(used, slots, pages, gen, device):
    """A page table [rows, slots] whose first used[r] entries are pages in random order, each once; the others are -1."""
    order = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
    used = used.to(torch.int64)
    before = torch.cumsum(used, 0) - used
    at = before[:, None] + torch.arange(slots, device=device)
    return torch.where(torch.arange(slots, device=device) < used[:, None], order[at.clamp(max=pages - 1)], torch.full_like(order[:1], -1))


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed * 9973 + 17)
    dt, op = TYPES[case["dtype"]], case["op"]
    state = {"case": case}

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=dtype or dt) * scale).to(dtype or dt)

    if op == "attend":
        rows, page, dim = case["rows"], case["page"], case["dim"]
        lengths = _shuffled(_lengths(case, case["length"]), gen, dev)
        slots = case["length"] // page + 1
        used = lengths // page + 1
        pages = int(used.sum()) + 3
        pool = normal(pages, 2, case["kv_heads"], page, dim)
        state.update(table=_table(used, slots, pages, gen, dev), lengths=lengths, pool=pool,
                     qkv=normal(rows, (case["heads"] + 2 * case["kv_heads"]) * dim))
    elif op == "append":
        rows, page = case["rows"], case["page"]
        counts = _shuffled(_lengths(case, case["tokens"]), gen, dev)
        start = torch.randint(0, 2 * page, (rows,), generator=gen, device=dev, dtype=torch.int32)
        slots = (case["tokens"] + 2 * page) // page + 1
        used = (start + counts) // page + 1
        pages = int((counts // page).sum()) + 3 * rows + 2  # whatever the starts are
        state.update(table=_table(used, slots, pages, gen, dev), counts=counts, start=start, pool=normal(pages, 2, case["kv_heads"], page, case["dim"]),
                     kv=normal(rows, case["tokens"], 2 * case["kv_heads"] * case["dim"]))
    elif op == "fork":
        groups, beams, page = case["groups"], case["beams"], case["page"]
        rows = groups * beams
        lengths = torch.tensor(_fork_lengths(case), dtype=torch.int32, device=dev).repeat_interleave(beams)
        slots = (case["length"] + page) // page + 2
        used = (lengths + page - 1) // page
        shared = torch.clamp(used - 2, min=0)  # the pages of a prompt are shared by the beams of a group, the last two are each beam's own
        pages = int(used.sum()) + 3 * rows + 5
        table = _table(used, slots, pages, gen, dev)
        first = table.view(groups, beams, slots)[:, :1].expand(groups, beams, slots).reshape(rows, slots)
        table = torch.where(torch.arange(slots, device=dev) < shared[:, None], first, table).contiguous()
        refcounts = torch.bincount(table[table >= 0].to(torch.int64), minlength=pages).to(torch.int32)
        # `kept` beams of each group go on, the lowest ones twice or more often
        pick = torch.rand(groups, beams, generator=gen, device=dev).argsort(1)[:, :case["kept"]]
        child = torch.arange(beams, device=dev) % case["kept"]
        parents = (torch.gather(pick, 1, child.expand(groups, beams)) + beams * torch.arange(groups, device=dev)[:, None]).reshape(-1).to(torch.int32)
        state.update(table=table, lengths=lengths, refcounts=refcounts, parents=parents, pool=normal(pages, case["blocks"], page, case["dim"]))
    elif op == "compact":
        pages, live, moves = case["pages"], case["live"], case["moves"]
        low = torch.randperm(live, generator=gen, device=dev)[: live - moves]
        high = live + torch.randperm(pages - live, generator=gen, device=dev)[:moves]
        ids = torch.cat([low, high])
        ids = ids[torch.randperm(live, generator=gen, device=dev)].to(torch.int32)
        table = torch.full((case["rows"] * case["slots"],), -1, dtype=torch.int32, device=dev)
        n = min(live, table.numel())
        table[torch.randperm(table.numel(), generator=gen, device=dev)[:n]] = ids[:n]
        refcounts = torch.zeros(pages, dtype=torch.int32, device=dev)
        refcounts[ids.to(torch.int64)] = torch.randint(1, 4, (live,), generator=gen, device=dev, dtype=torch.int32)
        state.update(table=table.view(case["rows"], case["slots"]), refcounts=refcounts, pool=normal(pages, case["blocks"], case["page"], case["dim"]))
    else:
        groups, beams, vocab, step = case["groups"], case["beams"], case["vocab"], case["step"]
        scores = -torch.rand(groups, beams, generator=gen, device=dev).cumsum(1) * (1 + step)
        if step == 0:  # a search begins with one beam
            scores = torch.where(torch.arange(beams, device=dev) > 0, torch.full_like(scores, -math.inf), torch.zeros_like(scores))
        finished = torch.rand(groups, beams, generator=gen, device=dev) < (0.15 if step else 0.0)
        lengths = torch.full((groups, beams), step, dtype=torch.int32, device=dev)
        lengths = torch.where(finished, torch.randint(1, max(2, step), (groups, beams), generator=gen, device=dev, dtype=torch.int32), lengths)
        sequences = torch.randint(0, vocab, (groups, beams, case["tokens"]), generator=gen, device=dev)
        state.update(logits=normal(groups * beams, vocab, scale=2.5), scores=scores.contiguous(), lengths=lengths, finished=finished, sequences=sequences, eos=vocab - 1)
    return state


def _fork_lengths(case):
    return [max(1, case["length"] - (5 * g) % case["page"]) for g in range(case["groups"])]


def _split(state):
    """q, k, v as views of the rows that a projection of all three gives."""
    case, qkv = state["case"], state["qkv"]
    h, g, d = case["heads"] * case["dim"], case["kv_heads"] * case["dim"], case["dim"]
    return qkv[:, :h].unflatten(1, (-1, d)), qkv[:, h:h + g].unflatten(1, (-1, d)), qkv[:, h + g:].unflatten(1, (-1, d))


def run(state):
    op = state["case"]["op"]
    return {"attend": _attend, "append": _append, "fork": _fork, "compact": _compact, "beam": _beam}[op](state)


def _attend(state):
    case, pool = state["case"], state["pool"]
    q, k, v = _split(state)
    keys, values = pool[:, 0], pool[:, 1]
    table, lengths = state["table"], state["lengths"]
    if own:
        from multimodal_amd import ops
        out = ops.paged_attention(q, keys, values, table, lengths, k if case["new"] else None, v if case["new"] else None)
        return (out, pool) if case["new"] else out
    rows, heads, dim = q.shape
    page, kv = keys.shape[2], keys.shape[1]
    n = lengths.to(torch.int64)
    if case["new"]:
        at = torch.gather(table, 1, (n // page)[:, None])[:, 0].to(torch.int64)
        keys[at, :, n % page] = k
        values[at, :, n % page] = v
        n = n + 1
    ids = table.clamp(min=0).to(torch.int64)
    gathered = pool[ids].float()  # [rows, slots, 2, kv, page, dim]
    both = gathered.permute(2, 0, 3, 1, 4, 5).reshape(2, rows, kv, -1, dim)
    s = torch.matmul(q.float().reshape(rows, kv, heads // kv, dim), both[0].transpose(-1, -2)) / math.sqrt(dim)
    s = torch.where(torch.arange(s.shape[-1], device=s.device) < n[:, None, None, None], s, torch.full_like(s[..., :1], -math.inf))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, both[1]) / torch.where(total > 0, total, torch.ones_like(total))
    out = o.reshape(rows, heads, dim).to(q.dtype)
    return (out, pool) if case["new"] else out


def _append(state):
    case, pool, table = state["case"], state["pool"], state["table"]
    keys, values = pool[:, 0], pool[:, 1]
    k, v = state["kv"].unflatten(2, (2, case["kv_heads"], case["dim"])).unbind(2)
    if own:
        from multimodal_amd import ops
        ops.paged_append(k, v, keys, values, table, state["start"], state["counts"])
        return pool
    page = keys.shape[2]
    j = torch.arange(case["tokens"], device=pool.device)
    row, col = (j < state["counts"][:, None]).nonzero(as_tuple=True)
    pos = state["start"].to(torch.int64)[row] + col
    at = table[row, pos // page].to(torch.int64)
    keys[at, :, pos % page] = k[row, col]
    values[at, :, pos % page] = v[row, col]
    return pool


def _fork(state):
    pool, table, lengths, refs, parents = (state[n] for n in ("pool", "table", "lengths", "refcounts", "parents"))
    if own:
        from multimodal_amd import ops
        return (*ops.paged_fork(pool, table, lengths, refs, parents, reserve=1), pool)
    page, pages, slots = pool.shape[2], pool.shape[0], table.shape[1]
    p = parents.to(torch.int64)
    n = lengths[p].to(torch.int64)
    j = torch.arange(slots, device=pool.device)
    old = table[p].to(torch.int64)
    full, rest = n // page, n % page
    partial = (j == full[:, None]) & (rest > 0)[:, None]
    r = torch.arange(p.numel(), device=pool.device)
    first = torch.full_like(lengths, p.numel(), dtype=torch.int64).scatter_reduce(0, p, r, "amin")
    keeps = (first[p] == r)[:, None] & (refs[old.clamp(min=0)] == 1)
    copied = partial & ~keeps
    fresh = copied | ((j >= ((n + page - 1) // page)[:, None]) & (j < ((n + 1 + page - 1) // page)[:, None]))
    free = torch.sort((refs > 0).to(torch.int8), stable=True).indices
    rank = torch.cumsum(fresh.reshape(-1).to(torch.int64), 0).view_as(fresh) - 1
    given = torch.where(rank < (refs <= 0).sum(), free[rank.clamp(0, pages - 1)], torch.full_like(rank, -1))
    kept = (j < full[:, None]) | (partial & keeps)
    new = torch.where(fresh, given, torch.where(kept, old, torch.full_like(old, -1)))
    row, slot = copied.nonzero(as_tuple=True)
    src, dst = old[row, slot], new[row, slot]
    inside = (torch.arange(page, device=pool.device) < rest[row][:, None])[:, None, :, None]
    pool[dst] = torch.where(inside, pool[src], pool[dst])
    ones = torch.ones(table.numel(), dtype=torch.int32, device=pool.device)
    counts = torch.cat([refs, refs.new_zeros(1)])
    counts = counts.index_add(0, torch.where(table >= 0, table, pages).reshape(-1).to(torch.int64), -ones)
    counts = counts.index_add(0, torch.where(new >= 0, new, pages).reshape(-1), ones[:1].expand(new.numel()))
    short = (fresh & (new < 0)).sum(dtype=torch.int32).reshape(1)
    return new.to(torch.int32), n.to(torch.int32), counts[:pages], short, pool


def _compact(state):
    pool, table, refs = (state[n] for n in ("pool", "table", "refcounts"))
    if own:
        from multimodal_amd import ops
        return (*ops.paged_compact(pool, table, refs), pool)
    ids = torch.arange(pool.shape[0], device=pool.device)
    live = refs > 0
    count = live.sum()
    src, dst = (live & (ids >= count)).nonzero()[:, 0], (~live & (ids < count)).nonzero()[:, 0]
    pool[dst] = pool[src]
    to = ids.clone()
    to[src] = dst
    new = torch.where(table >= 0, to[table.clamp(min=0).to(torch.int64)], torch.full_like(ids[:1], -1)).to(torch.int32)
    counts = torch.where(live, refs, torch.zeros_like(refs))
    moved = counts[src]
    counts[src] = 0
    counts[dst] = moved
    return new, counts, count.to(torch.int32).reshape(1), pool


def _beam(state):
    case, logits, scores, lengths = state["case"], state["logits"], state["scores"], state["lengths"]
    finished, sequences, eos = state["finished"], state["sequences"], state["eos"]
    if own:
        from multimodal_amd import ops
        return tuple(ops.beam_search_step(logits, scores, lengths, finished, sequences, eos, length_penalty=case["penalty"]))
    groups, beams = scores.shape
    vocab = logits.shape[1]
    x = logits.double().view(groups, beams, vocab)
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    total = scores.double()[..., None] + x
    ended = torch.where(torch.arange(vocab, device=x.device) == eos, scores.double()[..., None], torch.full_like(total[..., :1], -math.inf))
    total = torch.where(finished[..., None], ended, total)
    after = lengths + (~finished).to(torch.int32)
    rank = total / after.double().clamp(min=1)[..., None] ** case["penalty"]
    best = torch.sort(rank.view(groups, -1), dim=1, descending=True, stable=True).indices[:, :beams]
    beam, token = best // vocab, best % vocab
    done = torch.gather(finished, 1, beam)
    was = torch.gather(lengths, 1, beam)
    rows = torch.gather(sequences, 1, beam[..., None].expand(groups, beams, sequences.shape[2]))
    put = (torch.arange(sequences.shape[2], device=x.device) == was[..., None]) & ~done[..., None]
    return (torch.gather(total.view(groups, -1), 1, best).float(), torch.gather(after, 1, beam), done | (token == eos), token,
            (beam + beams * torch.arange(groups, device=x.device)[:, None]).to(torch.int32), torch.where(put, token[..., None], rows))


def work(case):
    size, op = {"bf16": 2, "fp32": 4}[case["dtype"]], case["op"]
    if op == "attend":
        n = [length + (1 if case["new"] else 0) for length in _lengths(case, case["length"])]
        token = case["kv_heads"] * case["dim"] * size * 2
        per_row = 2 * case["heads"] * case["dim"] * size + (token if case["new"] else 0) + 4
        return {"bytes": sum(n) * token + case["rows"] * per_row + 4 * sum(-(-x // case["page"]) for x in n), "flops": 4 * case["heads"] * case["dim"] * sum(n)}
    if op == "append":
        tokens = sum(_lengths(case, case["tokens"]))
        return {"bytes": 2 * tokens * case["kv_heads"] * case["dim"] * 2 * size + 8 * case["rows"] + 4 * (tokens // case["page"]), "flops": 0}
    if op == "fork":
        lens, page = _fork_lengths(case), case["page"]
        rest = sum(n % page for n in lens) * (case["beams"] - case["kept"])
        rows, slots = case["groups"] * case["beams"], (case["length"] + page) // page + 2
        pages = case["beams"] * sum(-(-n // page) for n in lens) + 3 * rows + 5
        return {"bytes": 2 * rest * case["blocks"] * case["dim"] * size + 8 * rows * slots + 8 * pages + 12 * rows, "flops": 0}
    if op == "compact":
        return {"bytes": 2 * case["moves"] * case["blocks"] * case["page"] * case["dim"] * size + 8 * case["rows"] * case["slots"] + 8 * case["pages"], "flops": 0}
    rows = case["groups"] * case["beams"]
    return {"bytes": rows * case["vocab"] * size + rows * (16 * case["tokens"] + 40), "flops": 4 * rows * case["vocab"]}


def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "fork": _exact_fork, "compact": _exact_compact, "beam": _exact_beam}[case["op"]](case, state)


def _exact_attend(case, s):
    pool, page, dim = s["pool"].clone(), case["page"], case["dim"]
    rows, kv = case["rows"], case["kv_heads"]
    group = case["heads"] // kv
    q = s["qkv"][:, :case["heads"] * dim].double().view(rows, kv, group, dim)
    rest = s["qkv"][:, case["heads"] * dim:].view(rows, 2, kv, dim)
    out = torch.zeros(rows, kv, group, dim, dtype=torch.float64, device=pool.device)
    lengths, table = s["lengths"].tolist(), s["table"].tolist()
    for r in range(rows):
        n = lengths[r]
        if case["new"]:
            pool[table[r][n // page], :, :, n % page] = rest[r]
            n += 1
        if n == 0:
            continue
        held = pool[table[r][: -(-n // page)]].double().transpose(0, 1)  # [2, pages, kv, page, dim]
        for h in range(kv):
            key, value = held[0, :, h].reshape(-1, dim)[:n], held[1, :, h].reshape(-1, dim)[:n]
            w = torch.softmax(key @ q[r, h].T / math.sqrt(dim), 0)
            out[r, h] = w.T @ value
    out = out.view(rows, -1, dim)
    return (out, pool) if case["new"] else out


def _exact_append(case, s):
    pool, page = s["pool"].clone(), case["page"]
    rows = s["kv"].view(case["rows"], case["tokens"], 2, case["kv_heads"], case["dim"])
    start, counts, table = s["start"].tolist(), s["counts"].tolist(), s["table"].tolist()
    for r in range(case["rows"]):
        done = 0
        while done < counts[r]:
            at = start[r] + done
            n = min(page - at % page, counts[r] - done)
            pool[table[r][at // page], :, :, at % page: at % page + n] = rows[r, done: done + n].permute(1, 2, 0, 3)
            done += n
    return pool


def _exact_fork(case, s):
    pool, page = s["pool"].clone(), case["page"]
    table, lengths, refs, parents = (s[n].tolist() for n in ("table", "lengths", "refcounts", "parents"))
    free = [x for x, c in enumerate(refs) if c == 0]
    new, lens, heirs, short = [], [], set(), 0
    for p in parents:
        n = lengths[p]
        row = table[p][: n // page]
        wanted = []
        if n % page:
            src = table[p][n // page]
            if refs[src] == 1 and p not in heirs:
                row.append(src)
            else:
                wanted.append(src)
        else:
            wanted.append(None)
        heirs.add(p)
        for src in wanted:
            row.append(free.pop(0) if free else -1)
            short += row[-1] < 0
            if src is not None and row[-1] >= 0:
                pool[row[-1], :, : n % page] = s["pool"][src, :, : n % page]
        new.append(row + [-1] * (len(table[p]) - len(row)))
        lens.append(n)
    counts = list(refs)
    for t, by in ((table, -1), (new, 1)):
        for row in t:
            for x in row:
                if x >= 0:
                    counts[x] += by
    dev = pool.device
    return (torch.tensor(new, dtype=torch.int32, device=dev), torch.tensor(lens, dtype=torch.int32, device=dev), torch.tensor(counts, dtype=torch.int32, device=dev),
            torch.tensor([short], dtype=torch.int32, device=dev), pool)


def _exact_compact(case, s):
    pool, refs = s["pool"].clone(), s["refcounts"].tolist()
    count = sum(c > 0 for c in refs)
    holes = [x for x in range(count) if refs[x] <= 0]
    to, counts = {x: x for x in range(count)}, [max(c, 0) for c in refs]
    for x in range(count, len(refs)):
        if refs[x] > 0:
            to[x] = holes.pop(0)
            pool[to[x]] = s["pool"][x]
            counts[to[x]], counts[x] = refs[x], 0
    new = [[to[x] if x >= 0 else -1 for x in row] for row in s["table"].tolist()]
    dev = pool.device
    return torch.tensor(new, dtype=torch.int32, device=dev), torch.tensor(counts, dtype=torch.int32, device=dev), torch.tensor([count], dtype=torch.int32, device=dev), pool


def _exact_beam(case, s):
    groups, beams, vocab, eos = case["groups"], case["beams"], case["vocab"], s["eos"]
    scores, lengths, finished = s["scores"].tolist(), s["lengths"].tolist(), s["finished"].tolist()
    found = [[], [], [], [], [], []]
    for g in range(groups):
        pool = []
        logp = torch.log_softmax(s["logits"][g * beams: (g + 1) * beams].double(), -1)
        for b in range(beams):
            if finished[g][b]:
                pool.append((scores[g][b] / max(1, lengths[g][b]) ** case["penalty"], b * vocab + eos, scores[g][b]))
                continue
            dead = scores[g][b] == -math.inf
            val, idx = torch.sort(logp[b], descending=True, stable=True)
            idx = list(range(min(vocab, beams))) if dead else idx[:beams].tolist()
            for i, lp in zip(idx, val[:beams].tolist()):
                total = scores[g][b] + lp
                pool.append((total / (lengths[g][b] + 1) ** case["penalty"], b * vocab + i, total))
        pool += [(-math.inf, b * vocab + i, -math.inf) for b in range(beams) if finished[g][b] for i in range(min(vocab, beams)) if i != eos]
        pool.sort(key=lambda c: (-c[0], c[1]))
        for _, flat, total in pool[:beams]:
            b, token = divmod(flat, vocab)
            row = s["sequences"][g, b].clone()
            if not finished[g][b] and lengths[g][b] < row.numel():
                row[lengths[g][b]] = token
            for to, x in zip(found, (total, lengths[g][b] + (not finished[g][b]), finished[g][b] or token == eos, token, g * beams + b, row)):
                to.append(x)
    dev = s["logits"].device
    kinds = (torch.float64, torch.int32, torch.bool, torch.int64, torch.int32)
    outs = [torch.tensor(x, dtype=t, device=dev).view(groups, beams) for x, t in zip(found, kinds)]
    return (*outs, torch.stack(found[5]).view(groups, beams, -1))
