"""The paged key-value cache's operators (csrc/paged_attention.hip, csrc/paged_pages.hip) against 64-bit restatements (oracle/decoding_oracle.py)."""
import math

import numpy as np
import pytest
import torch

from multimodal_amd import ops
from oracle import decoding_oracle as od

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _built():
    from multimodal_amd import build

    build.build()


def host(t):
    t = t.detach().cpu()
    return t.float().numpy() if t.is_floating_point() else t.numpy()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(seed, rows, heads, kv, dim, page, lengths, dtype, slots=None, spare=2, layout="heads"):
    """A cache whose rows have `lengths` tokens and room for one more, its pages in random order, with unused places full of NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [n // page + 1 for n in lengths]
    slots = slots or max(need)
    pages = sum(min(x, slots) for x in need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = np.full((rows, slots), -1, np.int32)
    for r in range(rows):
        for j in range(min(need[r], slots)):
            table[r, j] = order.pop()
    pool = torch.full((2, pages, kv, page, dim), float("nan"))
    for r in range(rows):
        for t in range(min(max(lengths[r], 0), slots * page)):
            pool[:, table[r, t // page], :, t % page] = torch.randn(2, kv, dim, generator=g)
    if layout == "heads":
        pool = pool.to(dtype).cuda()
    else:  # the tokens' heads side by side
        pool = pool.to(dtype).permute(0, 1, 3, 2, 4).contiguous().cuda().permute(0, 1, 3, 2, 4)
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).to(dtype).cuda()
    q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], 1)
    return pool[0], pool[1], i32(table), q.unflatten(1, (heads, dim)), k.unflatten(1, (kv, dim)), v.unflatten(1, (kv, dim))


# bf16 weights are used as two bf16 parts: each part is off by at most 2^-9 of itself, so 2^-18 of a weight is lost
WEIGHT_LOSS = {BF16: 2.0 ** -18, F32: 0.0}


def step_error(out, want, err, dtype):
    """How far the output lies beyond half a step of its type and what the oracle says that 32-bit sums may lose (and the division at the end: 2^-23)."""
    half = torch.finfo(dtype).eps / 2
    return np.abs(host(out) - want) - (half * np.abs(want) + (err + np.abs(want) * 2.0 ** -23) * (1 + half))


def check_attention(case, new, dtype, scale=None):
    kp, vp, table, q, k, v = case[:6]
    lengths = case[6]
    before = host(kp), host(vp)
    want, kp2, vp2, err = od.paged_attention(host(q), *before, host(table), np.array(lengths), host(k) if new else None, host(v) if new else None, scale,
                                           WEIGHT_LOSS[dtype])
    out = ops.paged_attention(q, kp, vp, table, i32(lengths), k if new else None, v if new else None, scale=scale)
    assert out.dtype == dtype and out.shape == q.shape and out.is_contiguous()
    bad = step_error(out, want, err, dtype)
    assert np.isfinite(host(out)).all() and bad.max(initial=0.0) <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))
    np.testing.assert_array_equal(host(kp), kp2)  # the new tokens, bit for bit, and nothing else (NaN where nothing was)
    np.testing.assert_array_equal(host(vp), vp2)


SHAPES = [
    # rows, heads, kv_heads, dim, page, lengths
    (1, 1, 1, 64, 16, [0]),
    (1, 12, 12, 64, 16, [40]),
    (3, 12, 12, 64, 16, [0, 15, 16]),
    (4, 4, 2, 96, 24, [1, 23, 47, 200]),
    (5, 6, 2, 128, 7, [0, 6, 7, 129, 300]),
    (2, 8, 1, 64, 1, [63, 64]),
    (2, 16, 2, 128, 64, [127, 1000]),
    (3, 15, 3, 64, 32, [511, 512, 513]),
    (2, 5, 1, 96, 5, [255, 256]),
    (7, 3, 3, 128, 16, [1, 2, 3, 4, 5, 6, 2100]),
    (2, 32, 2, 64, 128, [3000, 17]),
    (1, 33, 1, 64, 16, [130]),
    (40, 2, 2, 64, 16, list(range(0, 80, 2))),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new", [False, True], ids=["read", "new"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "r%d-h%d-%d-d%d-p%d" % s[:5])
def test_attention(shape, new, dtype):
    rows, heads, kv, dim, page, lengths = shape
    for layout in ("heads", "tokens"):
        check_attention((*make(rows * 7 + heads, rows, heads, kv, dim, page, lengths, dtype, layout=layout), lengths), new, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 1), (6, 2)])
def test_attention_long(heads, kv, dtype):
    """Split over the length and joined; a short row beside a long one; an explicit scale."""
    lengths = [20000, 0, 1, 4095]
    check_attention((*make(3, 4, heads, kv, 64, 32, lengths, dtype), lengths), True, dtype, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("group", [1, 2, 8])
def test_attention_holes_and_bad_lengths(group, dtype):
    """Pages that are not mapped (-1, and numbers beyond the pool), lengths that are negative or beyond the table: those positions take no part."""
    lengths = [100, 100, 100, -5, 1000, 63, 64, -1]
    kp, vp, table, q, k, v = make(5, 8, 2 * group, 2, 64, 16, [100, 100, 100, 0, 112, 63, 64, 0], dtype, slots=7)
    table[0, 1] = -1
    table[0, 3] = 2 ** 31 - 1
    table[1, :] = -7
    table[2, 6] = kp.shape[0]  # where its new token would go
    table[6, 4] = -1
    for new in (False, True):
        check_attention((kp, vp, table, q, k, v, lengths), new, dtype)


@pytest.mark.parametrize("group", [1, 4, 8])
def test_attention_large_scores(group):
    """Scores far apart and far from nothing: the running maximum carries them."""
    lengths = [700, 5]
    kp, vp, table, q, k, v = make(11, 2, 2 * group, 2, 64, 16, lengths, F32)
    want, _, _, err = od.paged_attention(host(q) * 300, host(kp), host(vp), host(table), np.array(lengths))
    out = ops.paged_attention((q * 300).contiguous(), kp, vp, table, i32(lengths))
    assert (np.abs(host(out) - want) <= err + 2.0 ** -23 * np.abs(want)).all()
    # keys of one value: the mean of the values, whatever the scores are
    kp.fill_(1.0)
    out = ops.paged_attention(q * 1e4, kp, vp, table, i32(lengths))
    for r in range(2):
        vals = np.stack([host(vp)[host(table)[r, t // 16], :, t % 16] for t in range(lengths[r])]).astype(np.float64)
        mean, mag = np.repeat(vals.mean(0), group, 0), np.repeat(np.abs(vals).mean(0), group, 0)
        assert (np.abs(host(out)[r] - mean) <= (2 * (lengths[r] / 16 + 64) * 2.0 ** -24 + 2.0 ** -20) * mag + 2.0 ** -23 * np.abs(mean)).all()


def test_attention_lowest_values_and_ties():
    """Keys at the type's lowest value push every weight to one token, equal ones share."""
    lengths = [33]
    for dtype in (BF16, F32):
        kp, vp, table, q, k, v = make(13, 1, 2, 2, 64, 16, lengths, dtype)
        q = torch.ones_like(q)
        kp.fill_(torch.finfo(dtype).min / 128)
        kp[table[0, 1].long(), :, 4] = 0.0
        out = ops.paged_attention(q, kp, vp, table, i32(lengths))
        assert torch.equal(out[0], vp[table[0, 1].long(), :, 4])


def test_attention_strides_offsets_and_out():
    """q, k, v as slices of wider rows, tables as slices, pages as one layer of a pool of several; a given output."""
    g = torch.Generator().manual_seed(2)
    pool = torch.randn(9, 3, 2, 4, 16, 64, generator=g).to(BF16).cuda()
    kp, vp = pool[:, 1, 0], pool[:, 1, 1]
    wide = torch.randn(3, 5000, generator=g).to(BF16).cuda()
    q, k, v = wide[:, 64:64 + 1024].unflatten(1, (16, 64))[:, ::2], wide[:, 2048:2048 + 256].unflatten(1, (4, 64)), wide[:, 4000:4256].unflatten(1, (4, 64))
    table = torch.tensor([[9, 0, 1, 2, 9], [9, 3, 4, 5, 9], [9, 6, 7, 8, 9]], dtype=torch.int32, device="cuda")[:, 1:4]
    lengths = [47, 20, 33]
    rest = pool[:, [0, 2]].clone()
    want, kp2, vp2, err = od.paged_attention(host(q), host(kp), host(vp), host(table), np.array(lengths), host(k), host(v), weight_loss=WEIGHT_LOSS[BF16])
    out = torch.empty(3, 8, 64, dtype=BF16, device="cuda")
    assert ops.paged_attention(q, kp, vp, table, i32(lengths), k, v, out=out) is out
    assert step_error(out, want, err, BF16).max() <= 0
    np.testing.assert_array_equal(host(kp), kp2)
    np.testing.assert_array_equal(host(vp), vp2)
    assert torch.equal(pool[:, [0, 2]], rest)
    assert ops.paged_attention(q[:0], kp, vp, table[:0], i32([]), k[:0], v[:0]).shape == (0, 8, 64)


def test_attention_offsets_beyond_32_bits():
    """A pool of more than 2^32 elements: the last pages are reached."""
    pages, page = 4200, 128
    pool = torch.empty(pages, 2, 64, page, 64, dtype=BF16, device="cuda")  # 2^32 elements and some
    assert pool.numel() > 2 ** 32
    ids = [pages - 1, 1, pages - 2]
    pool[ids] = torch.randn(3, 2, 64, page, 64, device="cuda", dtype=BF16)
    q = torch.randn(1, 64, 64, device="cuda", dtype=BF16)
    k, v = (torch.randn(1, 64, 64, device="cuda", dtype=BF16) for _ in range(2))
    n = 2 * page + 100
    out = ops.paged_attention(q, pool[:, 0], pool[:, 1], i32([ids]), i32([n]), k, v)
    few = host(pool[ids])
    assert torch.equal(pool[pages - 2, 0, :, 100], k[0]) and torch.equal(pool[pages - 2, 1, :, 100], v[0])
    want, _, _, err = od.paged_attention(host(q), few[:, 0], few[:, 1], np.array([[0, 1, 2]]), np.array([n + 1]), weight_loss=WEIGHT_LOSS[BF16])
    assert step_error(out, want, err, BF16).max() <= 0
    # and the writes of a prompt
    ops.paged_append(k[:, None], v[:, None], pool[:, 0], pool[:, 1], i32([ids]), i32([n + 1]))
    assert torch.equal(pool[pages - 2, 0, :, 101], k[0])
    state = ops.paged_fork(pool, i32([ids, [-1] * 3]), i32([n, 0]), i32([0, 1] + [0] * 2 + [1] * (pages - 4)), i32([0, 0]), reserve=0)
    assert host(state.page_table).tolist() == [ids, ids[:2] + [0]] and int(state.shortage) == 0
    assert torch.equal(pool[0, :, :, :100], pool[pages - 2, :, :, :100])
    del pool


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_attention_streams_and_graphs(dtype):
    """Two calls at once on two streams, and a captured one that is replayed with other inputs between eager work."""
    lengths = [900, 33, 0]
    cases = [make(s, 3, 4, 2, 64, 16, lengths, dtype) for s in (21, 22)]
    wants = [od.paged_attention(*map(host, (c[3], c[0], c[1], c[2])), np.array(lengths), host(c[4]), host(c[5]), weight_loss=WEIGHT_LOSS[dtype]) for c in cases]
    n = i32(lengths)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                outs.append(ops.paged_attention(c[3], c[0], c[1], c[2], n, c[4], c[5]))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert step_error(o, wants[i % 2][0], wants[i % 2][3], dtype).max() <= 0
        assert torch.equal(o, outs[i % 2])  # no atomics: the same bits every time
    kp, vp, table, q, k, v = cases[0]
    q2, n2 = q.clone(), n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.paged_attention(q2, kp, vp, table, n2)
    for seed in range(4):
        q2.copy_(torch.randn(q2.shape, generator=torch.Generator().manual_seed(seed)))
        n2.copy_(i32([[900, 33, 0], [1, 0, 1], [17, 34, 1], [0, 0, 0]][seed]))
        graph.replay()
        eager = ops.paged_attention(q2, kp, vp, table, n2)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,tokens,kv,dim,page", [(1, 1, 1, 64, 16), (3, 77, 12, 64, 16), (4, 33, 2, 96, 5), (2, 300, 3, 128, 64), (5, 0, 2, 64, 16), (0, 4, 2, 64, 16)])
def test_append(rows, tokens, kv, dim, page, dtype):
    g = torch.Generator().manual_seed(rows + tokens)
    start = [(3 * r * r) % (2 * page) for r in range(rows)]
    slots = (tokens + 2 * page) // page + 1
    pages = rows * slots + 2
    table = torch.randperm(pages, generator=g)[: rows * slots].view(rows, slots).to(torch.int32)
    if rows > 2:
        table[1, 1] = -1
        table[2, 0] = pages
        start[0] = -2                      # the first two have no place
        start[2] = slots * page - 3        # only three fit
    counts = [max(0, tokens - 5 * r) for r in range(rows)]
    if rows > 3:
        counts[3] = -4
    pool = torch.randn(2, pages, page, kv, dim, generator=g).to(dtype).cuda().permute(0, 1, 3, 2, 4)
    src = torch.randn(rows, tokens, 3 * kv * dim, generator=g).to(dtype).cuda()
    k, v = src[..., :kv * dim].unflatten(2, (kv, dim)), src[..., 2 * kv * dim:].unflatten(2, (kv, dim))
    for c in (counts, None):
        want = od.paged_append(host(k), host(v), host(pool[0]), host(pool[1]), host(table), start, c)
        ops.paged_append(k, v, pool[0], pool[1], table.cuda(), i32(start), None if c is None else i32(c))
        np.testing.assert_array_equal(host(pool[0]), want[0])
        np.testing.assert_array_equal(host(pool[1]), want[1])


def random_tables(g, rows, slots, page, pages, shared):
    """Rows whose first pages are shared in pairs, with counts; some entries bad."""
    rng = np.random.default_rng(g)
    table = np.full((rows, slots), -1, np.int32)
    lengths = rng.integers(0, slots * page + 1, rows).astype(np.int32)
    free = rng.permutation(pages).tolist()
    for r in range(rows):
        for j in range(-(-int(lengths[r]) // page)):
            if shared and r % 2 and j < int(lengths[r]) // page - 1 and table[r - 1, j] >= 0 and j < int(lengths[r - 1]) // page - 1:
                table[r, j] = table[r - 1, j]
            elif free:
                table[r, j] = free.pop()
    refs = np.bincount(table[table >= 0].ravel(), minlength=pages).astype(np.int32)
    return table, lengths, refs


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("seed,rows,slots,page,pages", [(0, 1, 1, 1, 4), (1, 4, 5, 16, 40), (2, 9, 7, 5, 200), (3, 33, 4, 8, 150), (4, 6, 3, 16, 5000), (5, 5, 6, 4, 31), (6, 1200, 3, 4, 9000), (7, 4500, 2, 2, 12000)])
def test_fork(seed, rows, slots, page, pages, dtype):
    rng = np.random.default_rng(seed)
    table, lengths, refs = random_tables(seed, rows, slots, page, pages, True)
    dim = 64
    blocks = (2, 2, 3) if rows < 100 else (1,)
    pool = torch.randn(pages, *blocks, page, dim, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    new_rows = int(rows * 1.5) + 1
    for parents, reserve in [
        (rng.integers(0, rows, new_rows), 1),
        (np.arange(rows), 0),
        (rng.integers(-2, rows + 2, new_rows), rng.integers(-3, 3 * page, new_rows).astype(np.int32)),
        (np.full(3, 0), page),
        (np.full(2, -1), 0),
        (np.zeros(0, np.int64), 0),
    ]:
        before = pool.clone()
        want = od.paged_fork(host(pool), table, lengths, refs, parents, reserve)
        state = ops.paged_fork(pool, i32(table), i32(lengths), i32(refs), i32(parents), reserve=reserve if np.isscalar(reserve) else i32(reserve))
        np.testing.assert_array_equal(host(state.page_table), want[1])
        np.testing.assert_array_equal(host(state.lengths), want[2])
        np.testing.assert_array_equal(host(state.refcounts), want[3])
        assert int(state.shortage) == want[4]
        np.testing.assert_array_equal(host(pool), want[0])
        pool.copy_(before)


def test_fork_bad_state_and_externally_held_pages():
    """Lengths out of range, entries that are no pages, a partial page that somebody else holds too, counts below zero."""
    page, pages = 4, 12
    table = np.array([[0, 1, 2], [3, -1, 4], [5, 99, -3], [6, 7, 8]], np.int32)
    lengths = np.array([9, 6, 100, -4], np.int32)
    refs = np.array([1, 1, 2, 1, 1, 1, 1, 1, 1, -2, 0, 0], np.int32)
    pool = torch.randn(pages, 3, page, 64).cuda()
    parents = np.array([0, 1, 2, 3, 0, 1])
    want = od.paged_fork(host(pool), table, lengths, refs, parents, 3)
    state = ops.paged_fork(pool, i32(table), i32(lengths), i32(refs), i32(parents), reserve=3)
    np.testing.assert_array_equal(host(state.page_table), want[1])
    np.testing.assert_array_equal(host(state.lengths), want[2])
    np.testing.assert_array_equal(host(state.refcounts), want[3])
    assert int(state.shortage) == want[4] > 0
    np.testing.assert_array_equal(host(pool), want[0])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("seed,pages,live", [(0, 1, 0), (1, 1, 1), (2, 7, 3), (3, 1024, 400), (4, 1025, 1024), (5, 5000, 4000), (6, 3100, 1024), (7, 64, 0), (8, 64, 64), (9, 70000, 33000)])
def test_compact(seed, pages, live, dtype):
    rng = np.random.default_rng(seed)
    refs = np.zeros(pages, np.int32)
    refs[rng.permutation(pages)[:live]] = rng.integers(1, 5, live)
    if pages > 10:
        refs[np.nonzero(refs == 0)[0][:2]] = -1
    table = rng.integers(-3, pages + 3, (11, 13)).astype(np.int32)
    wide = 2 if pages < 10000 else 1
    pool = torch.randn(pages, wide, 3, 64, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    want = od.paged_compact(host(pool), table, refs)
    got = ops.paged_compact(pool, i32(table), i32(refs))
    np.testing.assert_array_equal(host(got.page_table), want[1])
    np.testing.assert_array_equal(host(got.refcounts), want[2])
    assert int(got.live) == want[3]
    np.testing.assert_array_equal(host(pool), want[0])


def test_fork_and_compact_in_a_graph():
    """Captured and replayed with other states, eager calls in between."""
    page, pages, rows = 4, 1300, 6
    pool = torch.randn(pages, 2, page, 64).cuda()
    table, lengths, refs, parents = i32(np.zeros((rows, 5), np.int32)), i32([0] * rows), i32([0] * pages), i32([0] * rows)
    ops.paged_fork(pool, table, lengths, refs, parents, reserve=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forked = ops.paged_fork(pool, table, lengths, refs, parents, reserve=2)
        packed = ops.paged_compact(pool, forked.page_table, forked.refcounts)
    for seed in range(4):
        t, n, c = random_tables(seed, rows, 5, page, pages, True)
        p = np.random.default_rng(seed).integers(-1, rows, rows)
        for dst, src in ((table, t), (lengths, n), (refs, c), (parents, p)):
            dst.copy_(i32(src))
        start = host(pool)
        want = od.paged_fork(start, t, n, c, p, 2)
        want2 = od.paged_compact(want[0], want[1], want[3])
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(host(forked.page_table), want[1])
        np.testing.assert_array_equal(host(packed.page_table), want2[1])
        np.testing.assert_array_equal(host(packed.refcounts), want2[2])
        np.testing.assert_array_equal(host(pool), want2[0])
        pool.copy_(torch.randn(pages, 2, page, 64))


def test_together():
    """As they are used: prompts stored, rows forked, tokens attended and stored, rows dropped, the pool compacted -- against one plain list of tokens per row."""
    g = torch.Generator().manual_seed(0)
    layers, kv, heads, dim, page, pages, slots = 2, 2, 4, 64, 4, 64, 12
    pool = torch.full((pages, layers, 2, kv, page, dim), float("nan")).cuda()
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    state = ops.paged_fork(pool, i32(np.zeros((0, slots), np.int32)), i32([]), refs, i32([-1] * 3), reserve=i32([5, 8, 0]))
    counts = [5, 8, 0]
    rows = [[[] for _ in range(layers)] for _ in range(3)]
    for layer in range(layers):
        k, v = torch.randn(3, 8, kv, dim, generator=g), torch.randn(3, 8, kv, dim, generator=g)
        ops.paged_append(k.cuda(), v.cuda(), pool[:, layer, 0], pool[:, layer, 1], state.page_table, state.lengths, i32(counts))
        for r in range(3):
            rows[r][layer] = [(k[r, j].double(), v[r, j].double()) for j in range(counts[r])]
    state = state._replace(lengths=i32(counts))
    for step in range(20):
        parents = torch.randint(0, len(rows), (5,), generator=g).tolist()
        if step == 9:
            parents = parents[:2] + [-1]
        state = ops.paged_fork(pool, state.page_table, state.lengths, state.refcounts, i32(parents), reserve=1)
        assert int(state.shortage) == 0
        if step % 5 == 4:
            table, counted, live = ops.paged_compact(pool, state.page_table, state.refcounts)
            state = state._replace(page_table=table, refcounts=counted)
            assert int(table.max()) < int(live)
            pool[int(live):] = float("nan")
        rows = [[list(x) for x in rows[p]] if p >= 0 else [[] for _ in range(layers)] for p in parents]
        for layer in range(layers):
            q, k, v = (torch.randn(len(rows), h, dim, generator=g) for h in (heads, kv, kv))
            out = ops.paged_attention(q.cuda(), pool[:, layer, 0], pool[:, layer, 1], state.page_table, state.lengths, k.cuda(), v.cuda())
            for r, row in enumerate(rows):
                row[layer].append((k[r].double(), v[r].double()))
                kk, vv = (torch.stack([t[i] for t in row[layer]]).repeat_interleave(heads // kv, 1) for i in (0, 1))
                w = torch.softmax((kk * q[r].double()).sum(-1) / math.sqrt(dim), 0)
                want = (w[..., None] * vv).sum(0)
                assert float((out[r].double().cpu() - want).abs().max()) < 1e-5
        state = state._replace(lengths=state.lengths + 1)
    used = host(state.page_table)
    np.testing.assert_array_equal(np.bincount(used[used >= 0].ravel(), minlength=pages), host(state.refcounts))


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_traced_by_torch_compile(backend, grad):
    """A decoding step in one graph: the operators store through views of one pool, which a graph without in-place operations (aot_eager) has to keep in order."""
    from multimodal_amd import _torch_ops

    ns = _torch_ops.load()

    def state():
        g = torch.Generator().manual_seed(4)
        pool = torch.randn(9, 3, 2, 2, 16, 64, generator=g).to(BF16).cuda()
        return pool, i32([[0, 1], [2, 3], [4, 5]]), i32([3, 16, 20]), i32([1] * 6 + [0] * 3), i32([2, 2, 0]), torch.randn(3, 8, 64, generator=g).to(BF16).cuda()

    def step(pool, table, lengths, refs, parents, qkv):
        x, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        table, lengths, refs, short = ns.paged_fork(pool, table, lengths, refs, parents, None, 1)
        for layer in range(3):
            x = x + ns.paged_attention(x, pool[:, layer, 0], pool[:, layer, 1], table, lengths, k, v, None)
        ns.paged_append(k[:, None], v[:, None], pool[:, 1, 0], pool[:, 1, 1], table, lengths + 1, None)
        table, refs, live = ns.paged_compact(pool, table, refs)
        y = torch.empty_like(x)
        ns.paged_attention_into(x, pool[:, 1, 0], pool[:, 1, 1], table, lengths + 2, None, None, None, y)
        best = ns.beam_search_step(y.flatten(1).float(), torch.zeros(1, 3, device="cuda"), lengths[None], lengths[None] < 0, None, 5, 0.0)
        return (x, y, table, refs, live, short, *best[:5])

    args = state()
    want, pool = step(*args), args[0]
    torch._dynamo.reset()
    compiled = torch.compile(step, backend=backend, fullgraph=True)
    with torch.set_grad_enabled(grad):  # (nothing here asks for a gradient)
        for _ in range(2):
            args = state()
            for a, b in zip(compiled(*args), want):
                assert torch.equal(a, b)
            assert torch.equal(args[0], pool)
    torch._dynamo.reset()


def test_gradients_are_refused_on_the_device():
    """The same refusals as on meta tensors (tests/test_decoding_no_grad.py), before anything is stored."""
    import torch.autograd.forward_ad as fwad

    kp, vp, table, q, k, v = make(3, 2, 4, 2, 64, 16, [5, 20], F32)
    before, n = (kp.clone(), vp.clone()), i32([5, 20])
    with pytest.raises(ops.MmamdError, match="no gradient"):
        ops.paged_attention(q, kp, vp, table, n, k.clone().requires_grad_(), v)
    with fwad.dual_level(), pytest.raises(ops.MmamdError, match="no gradient"):
        ops.paged_attention(fwad.make_dual(q.contiguous(), q.contiguous()), kp, vp, table, n, k, v)
    with pytest.raises(ops.MmamdError, match="no gradient"):
        torch.func.grad(lambda x: ops.paged_attention(x, kp, vp, table, n, k, v).sum())(q.contiguous())
    with pytest.raises(ops.MmamdError, match="no gradient"):
        ops.paged_append(k[:, None].clone().requires_grad_(), v[:, None], kp, vp, table, n)
    np.testing.assert_array_equal(host(kp), host(before[0]))
    np.testing.assert_array_equal(host(vp), host(before[1]))
    version = kp._version
    ops.paged_attention(q, kp, vp, table, n, k, v)
    assert kp._version > version
