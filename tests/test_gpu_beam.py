"""One step of a beam search (csrc/beam.hip) against a 64-bit restatement (oracle/decoding_oracle.py)."""
import numpy as np
import pytest
import torch

from multimodal_amd import ops
from oracle import decoding_oracle as od

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from multimodal_amd import build

    build.build()


def host(t):
    t = t.detach().cpu()
    return t.float().numpy() if t.is_floating_point() else t.numpy()


def check(logits, scores, lengths, finished, sequences, eos, penalty):
    """Whole numbers are equal; a score is off by half a step of fp32 and what a log-sum-exp of 32-bit exponentials loses (2^-21 of the sum, at most)."""
    want = od.beam_search_step(host(logits), host(scores), host(lengths), host(finished), None if sequences is None else host(sequences), eos, penalty)
    got = ops.beam_search_step(logits, scores, lengths, finished, sequences, eos, length_penalty=penalty)
    for a, b, name in zip(got[1:], want[1:], got._fields[1:]):
        if b is None:
            assert a is None
            continue
        np.testing.assert_array_equal(host(a), b, err_msg=name)
    a, b = host(got.scores).astype(np.float64), want[0]
    live = np.isfinite(b)
    np.testing.assert_array_equal(np.isneginf(a), ~live)
    assert (np.abs(a[live] - b[live]) <= 2.0 ** -24 * np.abs(b[live]) + 2.0 ** -21).all()
    return got


def make(seed, groups, beams, vocab, dtype=torch.float32, step=7, tokens=20, ended=0.2):
    g = torch.Generator().manual_seed(seed)
    scores = -torch.rand(groups, beams, generator=g).cumsum(1) * (1 + step)
    finished = torch.rand(groups, beams, generator=g) < ended
    lengths = torch.where(finished, torch.randint(1, max(2, step + 1), (groups, beams), generator=g), torch.full((groups, beams), step)).to(torch.int32)
    sequences = torch.randint(0, vocab, (groups, beams, tokens), generator=g)
    logits = (torch.randn(groups * beams, vocab, generator=g) * 2.5).to(dtype)
    return [t.cuda() for t in (logits, scores, lengths, finished, sequences)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("penalty", [0.0, 0.6, 1.0, -0.5])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 1, 5), (2, 3, 3), (3, 5, 101), (2, 32, 40), (1, 5, 49408), (4, 7, 2047), (3, 2, 2049), (9, 4, 8191), (2, 32, 70001)])
def test_step(groups, beams, vocab, penalty, dtype):
    for seed in range(3):
        case = make(seed, groups, beams, vocab, dtype)
        check(*case, vocab - 1 if seed else vocab // 2, penalty)


def test_first_step_and_dead_beams():
    """A search begins with one beam; with fewer continuations than beams the rest tie at -inf, lowest first."""
    for vocab in (3, 5, 200):
        logits, scores, lengths, finished, seq = make(1, 2, 5, vocab, step=0, ended=0.0)
        scores.fill_(float("-inf"))
        scores[:, 0] = 0.0
        got = check(logits, scores, lengths, finished, seq, 0, 0.0)
        assert (host(got.parents) // 5 == np.array([[0], [1]])).all()
    check(logits, torch.full_like(scores, float("nan")), lengths, finished, seq, 0, 0.0)
    check(logits, torch.full_like(scores, float("-inf")), lengths, finished, seq, 0, 0.0)
    finished[0] = True
    check(logits, torch.full_like(scores, float("-inf")), lengths, finished, seq, 7, 1.0)
    check(logits, torch.zeros_like(scores), lengths, torch.ones_like(finished), seq, 3, 1.0)
    dead = torch.full_like(scores, float("-inf"))  # -inf over an infinite power has no order of its own: the lowest win
    got = ops.beam_search_step(logits, dead, lengths + 1000, torch.zeros_like(finished), seq, 0, length_penalty=500.0)
    assert host(got.tokens).tolist() == [[0, 1, 2, 3, 4]] * 2 and np.isneginf(host(got.scores)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_special_logits(dtype):
    """Banned words (-inf), nothing but -inf, a NaN, a +inf, all equal, the type's lowest and highest."""
    logits, scores, lengths, finished, seq = make(4, 2, 6, 5003, dtype, ended=0.0)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits[0, 100:] = float("-inf")
    logits[1] = float("-inf")
    logits[2, 4444] = float("nan")
    logits[3, 17] = float("inf")
    logits[4] = 0.0
    logits[5] = low
    logits[6] = high
    logits[7, ::2] = low
    logits[8, 3] = high
    logits[9, 1:] = float("-inf")
    logits[10] = -0.0
    logits[11, 5] = 1e4
    check(logits, scores, lengths, finished, seq, 4, 0.0)
    check(logits, scores, lengths, finished, seq, 4, 1.0)


def test_ties_go_to_the_lowest():
    """Equal logits within a beam, and equal beams."""
    logits, scores, lengths, finished, seq = make(6, 3, 4, 3001, ended=0.0)
    logits[:] = torch.randint(0, 3, logits.shape, generator=torch.Generator().manual_seed(0)).float().cuda()
    logits[4:8] = logits[4]
    scores[1] = -1.5
    check(logits, scores, lengths, finished, seq, 9, 0.0)
    logits[:] = 1.0
    got = check(logits, scores, lengths, finished, seq, 9, 0.0)
    assert host(got.tokens)[1].tolist() == [0, 1, 2, 3]


def test_strides_lengths_and_sequences():
    """Logits as a slice of padded rows that start off any alignment; sequences without room, with length -1, and none at all."""
    wide = torch.randn(10, 1013, generator=torch.Generator().manual_seed(3)).cuda()
    _, scores, lengths, finished, seq = make(8, 2, 5, 1001, tokens=7)
    lengths[0, 0], lengths[0, 1], lengths[1, 2] = 7, 100, -1
    for off in (0, 1, 5):
        check(wide[:, off:off + 1001], scores, lengths, finished, seq, 0, 0.0)
        check(wide[:, off:off + 1001].bfloat16(), scores, lengths, finished, seq, 0, 1.0)
    check(wide, scores, lengths, finished, None, 0, 0.0)
    check(wide, scores, lengths, finished, seq[..., :0].contiguous(), 0, 0.0)
    r = ops.beam_search_step(wide[:0], scores[:0], lengths[:0], finished[:0], seq[:0], 0)
    assert r.scores.shape == (0, 5)


def test_streams_and_graphs():
    cases = [make(s, 3, 5, 30522) for s in (1, 2)]
    firsts = [ops.beam_search_step(*c, 11) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for _ in range(10):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                runs.append(ops.beam_search_step(*c, 11))
    torch.cuda.synchronize()
    for i, r in enumerate(runs):
        assert all(torch.equal(a, b) for a, b in zip(r, firsts[i % 2]))
    live = [t.clone() for t in cases[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_search_step(*live, 11)
    for seed in (5, 6, 7):
        for dst, src in zip(live, make(seed, 3, 5, 30522)):
            dst.copy_(src)
        graph.replay()
        eager = ops.beam_search_step(*live, 11)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        check(*live, 11, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab", [(2, 9, 49408), (1, 16, 49408), (1, 31, 49408), (2, 17, 997), (1, 5, 131072), (1, 5, 131073), (1, 12, 200003), (1, 3, 524289), (1, 20, 600011)])
def test_many_beams_and_words(groups, beams, vocab, dtype):
    """More beams than waves, more lists than lanes, lists longer than their part in LDS."""
    check(*make(11, groups, beams, vocab, dtype), vocab // 3, 0.6)


@pytest.mark.parametrize("beams,vocab", [(4, 140000), (20, 49408), (32, 600011)])
def test_the_best_in_one_stretch_and_ties_far_apart(beams, vocab):
    """All of a row's best words lie beside each other (one list is used up), then all over it at equal logits."""
    logits, scores, lengths, finished, seq = make(12, 1, beams, vocab, ended=0.0)
    logits[:, 30000:30000 + beams] += 50.0
    check(logits, scores, lengths, finished, seq, 9, 1.0)
    logits[:] = -1.0
    logits[:, 777::9001] = 2.0
    logits[:, vocab - 1] = 2.0
    scores[:] = -0.5 - torch.arange(beams, device="cuda") / 64.0  # (ranks of beams differ by more than a rounding)
    check(logits, scores, lengths, finished, seq, 9, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("beams,vocab", [(2, 101), (4, 49408), (9, 30522)])
def test_beams_whose_logits_are_permutations(beams, vocab, dtype):
    """Equal totals across beams in exact arithmetic: the log-sum-exps, each good to 2^-21 for random logits, decide, so each place holds a continuation within two of those of the exact
    one; within a beam the order is that of the logits, whatever the sums are."""
    g = torch.Generator().manual_seed(beams)
    base = (torch.randn(vocab, generator=g) * 2.5).to(dtype)
    logits = torch.stack([base[torch.randperm(vocab, generator=g)] for _ in range(2 * beams)]).cuda()
    scores, done = torch.full((2, beams), -3.25).cuda(), torch.zeros((2, beams), dtype=torch.bool).cuda()
    got = ops.beam_search_step(logits, scores, torch.full((2, beams), 6, dtype=torch.int32).cuda(), done, None, 3, length_penalty=0.0)
    logp = torch.log_softmax(logits.cpu().double(), -1)
    parents, tokens = host(got.parents), host(got.tokens)
    for k in range(2):
        best = torch.sort((logp[k * beams:(k + 1) * beams] - 3.25).flatten(), descending=True).values[:beams].numpy()
        picked = np.array([float(logp[p, t]) - 3.25 for p, t in zip(parents[k], tokens[k])])
        assert (np.abs(picked - best) <= 2 * 2.0 ** -21).all()
        assert (np.abs(host(got.scores)[k] - picked) <= 2.0 ** -24 * np.abs(picked) + 2.0 ** -21).all()
        assert len({(p, t) for p, t in zip(parents[k], tokens[k])}) == beams
        for b in range(beams):
            mine = tokens[k][parents[k] == k * beams + b]
            order = np.lexsort((np.arange(vocab), -logits[k * beams + b].cpu().double().numpy()))
            np.testing.assert_array_equal(mine, order[:len(mine)])


@pytest.mark.parametrize("score", [torch.finfo(torch.float32).min, -1e30])
def test_scores_that_swallow_the_logits(score):
    """Ranks that round to one number: of each beam its highest logits take part, and of those the lowest beam's lowest words come first."""
    logits, scores, lengths, finished, seq = make(9, 2, 5, 5003, ended=0.0)
    scores.fill_(score)
    got = ops.beam_search_step(logits, scores, lengths, finished, seq, 0, length_penalty=1.0)
    best = torch.topk(logits.view(2, 5, -1)[:, 0], 5).indices.sort(1).values
    assert torch.equal(got.tokens, best) and host(got.parents).tolist() == [[0] * 5, [5] * 5]
    assert (host(got.scores) == np.float32(score)).all()
