"""Host side of the decoding operators, on the CPU: argument checks of the C-ABI and of the wrappers, the page arithmetic, and the oracle itself."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import decoding_oracle as od

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def L():
    from multimodal_amd import _lib, build

    build.build()
    return _lib.lib()


class _PagedCache(C.Structure):  # mmamd_paged_cache (include/mmamd.h)
    _fields_ = [("key_pages", C.c_void_p), ("value_pages", C.c_void_p), ("page_table", C.c_void_p),
                ("key_page_stride", C.c_int64), ("key_head_stride", C.c_int64), ("key_token_stride", C.c_int64),
                ("value_page_stride", C.c_int64), ("value_head_stride", C.c_int64), ("value_token_stride", C.c_int64), ("table_row_stride", C.c_int64),
                ("dtype", C.c_int32), ("pages", C.c_int32), ("page_size", C.c_int32), ("slots", C.c_int32), ("kv_heads", C.c_int32), ("dim", C.c_int32)]


def cache(**kw):
    d = dict(key_pages=4096, value_pages=8192, page_table=64, key_page_stride=2048, key_head_stride=1024, key_token_stride=64, value_page_stride=2048,
             value_head_stride=1024, value_token_stride=64, table_row_stride=4, dtype=1, pages=8, page_size=16, slots=4, kv_heads=2, dim=64)
    d.update(kw)
    return _PagedCache(**d)


def attention(L, c, lengths=64, q=256, k=None, v=None, out=256, rows=1, heads=2, q_row=128, ws=None, bytes_=0):
    return L.mmamd_paged_attention(C.byref(c) if c is not None else None, lengths, q, q_row, 64, k, 64, 64, v, 64, 64, out, rows, heads, 0.125, ws, bytes_, None)


def test_attention_arguments(L):
    """Every refusal comes before a launch, with a message (addresses here are no memory)."""
    assert attention(L, None) == -1 and b"null cache" in L.mmamd_last_error()
    for kw, code in [(dict(key_pages=None), -1), (dict(page_table=None), -1), (dict(dtype=2), -2), (dict(pages=0), -1), (dict(page_size=0), -1), (dict(slots=-1), -1),
                     (dict(kv_heads=0), -1), (dict(dim=80), -2), (dict(key_pages=4104), -3), (dict(key_token_stride=60), -3), (dict(value_head_stride=-64), -3),
                     (dict(slots=1 << 26, page_size=32), -2)]:
        assert attention(L, cache(**kw)) == code, kw
        assert L.mmamd_paged_attention_workspace(C.byref(cache(**kw)), 1, 2) == code, kw
        assert L.mmamd_paged_append(C.byref(cache(**kw)), 256, 64, 64, 64, 256, 64, 64, 64, 64, None, 1, 1, None) == code, kw
    c = cache()
    assert attention(L, c, heads=3) == -1 and attention(L, c, rows=-1) == -1 and attention(L, c, rows=70000) == -2
    assert attention(L, c, q=None) == -1 and attention(L, c, lengths=None) == -1 and attention(L, c, out=None) == -1
    assert attention(L, c, k=256) == -1 and b"one of k and v" in L.mmamd_last_error()
    assert attention(L, c, q=258) == -3 and attention(L, c, q_row=65) == -3
    big = cache(slots=1000)
    need = L.mmamd_paged_attention_workspace(C.byref(big), 1, 2)
    assert need > 0 and attention(L, big, ws=None, bytes_=need) == -1 and attention(L, big, ws=256, bytes_=need - 1) == -1
    assert b"needed" in L.mmamd_last_error()
    assert attention(L, c, rows=0) == 0  # nothing to do
    assert L.mmamd_paged_append(C.byref(c), 256, 64, 64, 64, 256, 64, 64, 64, None, None, 1, 1, None) == -1
    assert L.mmamd_paged_append(C.byref(c), 256, 64, 60, 64, 256, 64, 64, 64, 64, None, 1, 1, None) == -3
    assert L.mmamd_paged_append(C.byref(c), 256, 64, 64, 64, 256, 64, 64, 64, 64, None, 1, 1 << 28, None) == -2
    assert L.mmamd_paged_append(C.byref(c), None, 64, 64, 64, None, 64, 64, 64, None, None, 0, 4, None) == 0


def test_fork_compact_and_beam_arguments(L):
    def fork(pool=4096, pages=8, blocks=2, page=16, row=128, table=64, lengths=64, refs=64, old=2, slots=4, parents=64, rows=2, new=64, ws=256, size=1 << 20):
        return L.mmamd_paged_fork(pool, pages, blocks, page, row, table, slots, lengths, refs, old, slots, parents, rows, None, 1, new, new, new, new, ws, size, None)

    for kw, code in [(dict(pages=0), -1), (dict(blocks=0), -1), (dict(slots=0), -1), (dict(rows=-1), -1), (dict(pool=None), -1), (dict(refs=None), -1), (dict(table=None), -1),
                     (dict(parents=None), -1), (dict(ws=None), -1), (dict(size=8), -1), (dict(row=120), -3), (dict(pool=4100), -3), (dict(rows=65534), -2),
                     (dict(slots=1 << 27), -2)]:
        assert fork(**kw) == code, kw
    assert L.mmamd_paged_fork_workspace(2, 2, 0, 8) == -1 and L.mmamd_paged_fork_workspace(2, 3, 4, 8) > 0

    def compact(pool=4096, pages=8, size=4096, table=64, rows=2, slots=4, refs=64, new=64, ws=256, bytes_=1 << 20):
        return L.mmamd_paged_compact(pool, pages, size, table, slots, rows, slots, refs, new, new, new, ws, bytes_, None)

    for kw, code in [(dict(pages=0), -1), (dict(size=0), -1), (dict(size=100), -3), (dict(pool=None), -1), (dict(table=None), -1), (dict(ws=None), -1), (dict(bytes_=4), -1)]:
        assert compact(**kw) == code, kw

    def beam(logits=256, dtype=0, ld=100, scores=64, seq=None, out=64, out_seq=None, tokens=0, eos=3, penalty=0.0, groups=1, beams=4, vocab=100, ws=256, size=1 << 20):
        return L.mmamd_beam_search_step(logits, dtype, ld, scores, 64, 64, seq, tokens, eos, penalty, groups, beams, vocab, out, 64, 64, 64, 64, out_seq, ws, size, None)

    for kw, code in [(dict(logits=None), -1), (dict(dtype=3), -2), (dict(beams=33), -2), (dict(beams=0), -1), (dict(groups=30000), -2), (dict(vocab=0), -1), (dict(eos=100), -1),
                     (dict(eos=-1), -1), (dict(seq=64), -1), (dict(penalty=math.nan), -1), (dict(penalty=math.inf), -1), (dict(size=4), -1), (dict(ws=None), -1), (dict(out=None), -1), (dict(ld=-1), -1)]:
        assert beam(**kw) == code, kw
    assert beam(groups=0) == 0


def test_wrappers_refuse_host_tensors_and_wrong_types():
    from multimodal_amd import ops

    q, pages, table, n = torch.zeros(1, 2, 64), torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    calls = [lambda: ops.paged_attention(q, pages, pages, table, n), lambda: ops.paged_attention(q, pages, pages, table, n, out=q),
             lambda: ops.paged_append(q[None], q[None], pages, pages, table, n), lambda: ops.paged_fork(pages, table, n, n, n),
             lambda: ops.paged_compact(pages, table, n), lambda: ops.beam_search_step(torch.zeros(2, 5), torch.zeros(1, 2), table, table.bool(), None, 0)]
    for call in calls:
        with pytest.raises(ops.MmamdError, match="no CPU fallback"):
            call()
    with pytest.raises(ops.MmamdError):
        ops.paged_attention(1.0, 2, 3, table, n)


def test_meta_kernels_infer_shapes():
    from multimodal_amd import _torch_ops

    ns = _torch_ops.load()
    m = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    i = torch.int32
    out = ns.paged_attention(m(3, 4, 64), m(9, 2, 16, 64), m(9, 2, 16, 64), m(3, 5, dtype=i), m(3, dtype=i), None, None, None)
    assert out.shape == (3, 4, 64)
    table, lengths, refs, short = ns.paged_fork(m(9, 2, 16, 64), m(3, 5, dtype=i), m(3, dtype=i), m(9, dtype=i), m(7, dtype=i), None, 1)
    assert table.shape == (7, 5) and lengths.shape == (7,) and refs.shape == (9,) and short.shape == (1,) and table.dtype == i
    assert [tuple(t.shape) for t in ns.paged_compact(m(9, 2, 16, 64), m(3, 5, dtype=i), m(9, dtype=i))] == [(3, 5), (9,), (1,)]
    r = ns.beam_search_step(m(6, 50), m(2, 3), m(2, 3, dtype=i), m(2, 3, dtype=torch.bool), m(2, 3, 8, dtype=torch.int64), 1, 0.0)
    assert [t.dtype for t in r] == [torch.float32, i, torch.bool, torch.int64, i, torch.int64] and r[5].shape == (2, 3, 8)
    assert "Tensor(a!) key_pages" in str(ns.paged_attention.default._schema)


def test_decoding_kernels_do_not_spill():
    from concurrent.futures import ThreadPoolExecutor

    from tools.check_spills import CSRC, check

    with ThreadPoolExecutor(max_workers=3) as ex:
        for name, rc, rows in ex.map(check, [CSRC / f for f in ("paged_attention.hip", "paged_pages.hip", "beam.hip")]):
            assert rc == 0 and rows, name
            assert not [r for r in rows if r[2] > 0 or r[1] > 256], name


def test_page_division(tmp_path):
    """div_by (csrc/paged.h) is the division, for every divisor and the numerators around its multiples."""
    from multimodal_amd import build

    (tmp_path / "e.hip").write_text("namespace mmamd { void set_error(const char*, ...) {} void count_launch(const char*) {} }")
    (tmp_path / "t.hip").write_text(f'''
#include "{ROOT}/multimodal_amd/csrc/paged.h"
int main() {{
  for (uint32_t d = 1; d < 70000; d = d < 300 ? d + 1 : d * 1.37) {{
    const mmamd::FastDiv f = mmamd::fast_div(d);
    for (uint64_t k = 0; k * d < 0xffffffffull; k = k < 100 ? k + 1 : k * 1.1 + 1)
      for (int64_t e = -1; e <= 1; ++e) {{
        const int64_t n = (int64_t)(k * d) + e;
        if (n >= 0 && n <= 0xffffffffll && mmamd::div_by(f, (uint32_t)n) != (uint32_t)n / d) return 1;
      }}
    if (mmamd::div_by(f, 0xffffffffu) != 0xffffffffu / d) return 2;
  }}
  return 0;
}}''')
    subprocess.run([build._hipcc(), "-O1", "-std=c++17", "--offload-arch=gfx950", "--offload-host-only", "-Wno-return-type", str(tmp_path / "t.hip"), str(tmp_path / "e.hip"),
                    "-o", str(tmp_path / "t")], check=True, capture_output=True)
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0


def test_oracle_attention_equals_dense():
    """Pages in order and out of order give what one dense softmax gives; bad pages are as if their tokens were not there."""
    rng = np.random.default_rng(0)
    kp, vp = rng.standard_normal((2, 6, 2, 4, 8))
    q = rng.standard_normal((2, 4, 8))
    table = np.array([[3, 0, 5], [1, 9, 2]], np.int32)
    out, kp2, _, _ = od.paged_attention(q, kp, vp, table, np.array([10, 12]))
    np.testing.assert_array_equal(kp, kp2)
    for r, ids in ((0, [3, 0, 5]), (1, [1, 2])):
        n = 10 if r == 0 else 8
        for h in range(4):
            kk, vv = (np.concatenate([x[i, h // 2] for i in ids])[:n] for x in (kp, vp))
            s = kk @ q[r, h] / math.sqrt(8)
            w = np.exp(s - s.max())
            np.testing.assert_allclose(out[r, h], w @ vv / w.sum(), atol=1e-12)
    out, kp2, vp2, _ = od.paged_attention(q, kp, vp, table, np.array([10, 4]), kp[0, :, :2].transpose(1, 0, 2), vp[0, :, :2].transpose(1, 0, 2))
    np.testing.assert_array_equal(kp2[5, :, 2], kp[0, :, 0])  # position 10 = place 2 of page 5
    np.testing.assert_array_equal(np.delete(kp2, 5, 0), np.delete(kp, 5, 0))  # position 4 of the second row lies on page 9, which is none
    assert not od.paged_attention(q, kp, vp, table, np.array([0, -3]))[0].any()


def test_oracle_fork_keeps_counts():
    rng = np.random.default_rng(1)
    pool = rng.standard_normal((40, 2, 4, 8))
    table, lengths, refs = np.full((0, 6), -1, np.int32), np.zeros(0, np.int32), np.zeros(40, np.int32)
    pool, table, lengths, refs, short = od.paged_fork(pool, table, lengths, refs, [-1, -1], [5, 9])
    lengths = np.array([5, 9])
    for step in range(8):
        parents = rng.integers(0, len(lengths), 4)
        tokens = [[pool[table[p, t // 4]][..., t % 4, :].copy() for t in range(lengths[p])] for p in parents]
        pool, table, lengths, refs, short = od.paged_fork(pool, table, lengths, refs, parents, 1)
        assert short == 0
        np.testing.assert_array_equal(np.bincount(table[table >= 0], minlength=40), refs)
        for r, row in enumerate(tokens):
            for t, x in enumerate(row):
                np.testing.assert_array_equal(pool[table[r, t // 4]][..., t % 4, :], x)
        pool, table, refs, live = od.paged_compact(pool, table, refs)
        assert (refs[:live] > 0).all() and not refs[live:].any()
        for r in range(4):  # a new token of its own for every row
            pool[table[r, lengths[r] // 4]][..., lengths[r] % 4, :] = rng.standard_normal((2, 8))
        lengths = lengths + 1


def test_oracle_beam_equals_sort():
    rng = np.random.default_rng(2)
    logits, scores = rng.standard_normal((6, 11)), -rng.random((2, 3)).cumsum(1)
    res = od.beam_search_step(logits, scores, np.full((2, 3), 4), np.zeros((2, 3), bool), None, 0)
    logp = logits - np.log(np.exp(logits).sum(1, keepdims=True))
    for g in range(2):
        flat = (scores[g][:, None] + logp[3 * g:3 * g + 3]).ravel()
        best = np.argsort(-flat)[:3]
        np.testing.assert_allclose(res[0][g], flat[best])
        np.testing.assert_array_equal(res[3][g], best % 11)
        np.testing.assert_array_equal(res[4][g], best // 11 + 3 * g)


def test_cache_and_captioning_arguments():
    from multimodal_amd import ops
    from multimodal_amd.models.coca.captioning import generate_captions
    from multimodal_amd.models.coca.coca_model import coca_vit
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache
    from tests.golden.make_golden_coca import SMALL

    with pytest.raises(ops.MmamdError, match="wide heads"):
        PagedKVCache(1, 2, 80, 4, 16, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 64, 0, 16, device="cpu")
    cache = PagedKVCache(2, 3, 64, 5, 33, 16, device="cpu")
    assert cache.pages.shape == (5, 2, 2, 3, 16, 64) and cache.page_table.shape == (0, 3) and cache.rows == 0
    assert cache.layer(1)[0].data_ptr() == cache.pages[0, 1, 0].data_ptr()
    with pytest.raises(ops.MmamdError, match="no CPU fallback"):
        cache.add_rows(2, 1)
    model = coca_vit(**SMALL, cascaded_pooler=False)
    images = torch.zeros(1, 3, 64, 64)
    with pytest.raises(ops.MmamdError, match="eval"):
        generate_captions(model, images, 1, 2)
    model.eval()
    for kw in (dict(max_length=1), dict(max_length=13), dict(num_beams=0), dict(begin=96), dict(end=-1)):
        with pytest.raises(ValueError):
            generate_captions(model, images, **{"begin": 1, "end": 2, **kw})


def test_a_view_of_shared_rows_stores_and_moves_nothing():
    """shared_rows() holds no references: what would write or reassign pages through it is refused."""
    from multimodal_amd import ops
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache

    cache = PagedKVCache(1, 2, 64, 5, 33, 16, device="cpu")
    cache.page_table, cache.lengths = torch.tensor([[0, 1, -1], [2, -1, -1]], dtype=torch.int32), torch.tensor([20, 3], dtype=torch.int32)
    view = cache.shared_rows(torch.tensor([1, 1, 0]))
    assert view.page_table.tolist() == [[2, -1, -1], [2, -1, -1], [0, 1, -1]] and view.lengths.tolist() == [3, 3, 20] and view.pages is cache.pages
    kv, rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: view.fork(rows), lambda: view.reserve(1), lambda: view.add_rows(1, 1), lambda: view.append(0, kv[:, None], kv[:, None]),
                 lambda: view.attend(0, kv, kv, kv), view.advance, view.compact, lambda: view.resize(5), view.reset):
        with pytest.raises(ops.MmamdError, match="another cache"):
            call()
    assert view.lengths.tolist() == [3, 3, 20] and cache.lengths.tolist() == [20, 3]


def test_rows_of_encoder_states_follow_a_fork(monkeypatch):
    """fork() takes the rows of `cross` along (on the CPU: the operator is replaced by its oracle's table)."""
    from multimodal_amd import ops
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache

    cache, cross = (PagedKVCache(1, 2, 64, 8, 33, 16, device="cpu") for _ in range(2))

    def fork(pages, table, lengths, refcounts, parents, reserve):
        n = len(parents)
        return ops.PagedState(torch.full((n, 3), -1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32), refcounts, torch.zeros(1, dtype=torch.int32))

    monkeypatch.setattr(ops, "paged_fork", fork)
    cross.page_table, cross.lengths = torch.tensor([[0, 1, -1], [2, -1, -1]], dtype=torch.int32), torch.tensor([20, 3], dtype=torch.int32)
    cache.cross = cross
    with pytest.raises(ValueError, match="2 rows, this one 0"):
        cache.fork(torch.tensor([-1, -1], dtype=torch.int32))
    cache.add_rows(2, 4)
    assert cache.cross is cross and cache.rows == 2
    cache.fork(torch.tensor([1, -1, 0, 7], dtype=torch.int32))
    assert cache.cross.lengths.tolist() == [3, 0, 20, 0] and cache.cross.page_table[[0, 2]].tolist() == [[2, -1, -1], [0, 1, -1]]
    cache.reserve(2)
    assert cache.cross.lengths.tolist() == [3, 0, 20, 0]
    cache.fork(torch.tensor([[2], [0]], dtype=torch.int32))
    assert cache.cross.lengths.tolist() == [20, 3] and cross.lengths.tolist() == [20, 3] and cross.rows == 2
    held = cache.cross
    cache.fork(torch.tensor([0, 0, 0], dtype=torch.int32), cross=False)
    assert cache.cross is held


def test_prompts_beyond_the_table_and_beams_beyond_the_kernel_are_refused():
    from multimodal_amd.models.coca.captioning import generate_captions
    from multimodal_amd.models.coca.coca_model import coca_vit
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache
    from tests.golden.make_golden_coca import SMALL

    cache = PagedKVCache(1, 2, 64, 5, 33, 16, device="cpu")
    with pytest.raises(ValueError, match="49 tokens for rows of 48"):
        cache.add_rows(2, 49)
    model = coca_vit(**SMALL, cascaded_pooler=False).eval()
    with pytest.raises(ValueError, match="between 1 and 32"):
        generate_captions(model, torch.zeros(1, 3, 64, 64), 1, 2, num_beams=33)


def test_out_of_memory_keeps_its_type(monkeypatch):
    """Callers free memory and go on where they catch torch.OutOfMemoryError."""
    from multimodal_amd import ops

    def full(*args):
        raise torch.OutOfMemoryError("out of memory")

    def wrong(*args):
        raise RuntimeError("a reason\nand a trace")

    pages, table, ints = torch.zeros(2, 1, 4, 64, device="meta"), torch.zeros(1, 1, dtype=torch.int32, device="meta"), torch.zeros(1, dtype=torch.int32, device="meta")
    q, logits, scores = torch.zeros(1, 1, 64, device="meta"), torch.zeros(1, 4, device="meta"), torch.zeros(1, 1, device="meta")
    calls = {"paged_attention": lambda: ops.paged_attention(q, pages, pages, table, ints), "paged_attention_into": lambda: ops.paged_attention(q, pages, pages, table, ints, out=q),
             "paged_append": lambda: ops.paged_append(q[None], q[None], pages, pages, table, ints), "paged_fork": lambda: ops.paged_fork(pages, table, ints, ints, ints),
             "paged_compact": lambda: ops.paged_compact(pages, table, ints),
             "beam_search_step": lambda: ops.beam_search_step(logits, scores, ints[None], ints[None].bool(), None, 0)}
    for name, call in calls.items():
        monkeypatch.setattr(ops, "_DECODING", {name: full})
        with pytest.raises(torch.OutOfMemoryError):
            call()
        monkeypatch.setattr(ops, "_DECODING", {name: wrong})
        with pytest.raises(ops.MmamdError, match="^a reason$"):
            call()
