"""The decoding operators in the models: TransformerDecoder over a paged cache against the reference's fixture and its own full pass, and captions of a CoCa model
against full forwards."""
import numpy as np
import pytest
import torch

from tests.golden.make_golden import seed
from tests.golden.make_golden_coca import POOL96, SMALL, randomize

pytestmark = pytest.mark.gpu

LOGIT_TOL = 3e-2  # of the vocabulary logits, as in test_gpu_coca.py


@pytest.fixture(scope="module", autouse=True)
def _built():
    from multimodal_amd import build

    build.build()


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def cache_for(dec, rows, max_tokens, page_size):
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache

    att = dec.layer[0].attention
    slots = -(-max_tokens // page_size)
    return PagedKVCache(len(dec.layer), att.num_heads, att.q_proj.out_features // att.num_heads, rows * (slots + 2), max_tokens, page_size)


@pytest.mark.parametrize("page_size", [1, 4, 16])
@pytest.mark.parametrize("cross_cached", [False, True])
@torch.no_grad()
def test_decoder_over_a_paged_cache_vs_reference_fixture(golden, page_size, cross_cached):
    """A prompt and two single tokens through pages equal the reference's causal pass, as the concatenated cache does (tests/test_gpu_coca.py)."""
    from multimodal_amd.modules.layers.transformer import TransformerDecoder

    z = golden("kv_cache.npz")
    dec = TransformerDecoder(n_layer=2, d_model=128, n_head=2, dim_feedforward=256, activation=torch.nn.GELU, layer_norm_eps=1e-5, norm_first=True,
                             use_cross_attention=True, dim_kv=128, final_layer_norm_eps=1e-5)
    dec.load_state_dict({k[7:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("dec.sd.")}, strict=True)
    dec = dec.cuda().eval()
    h, enc = torch.from_numpy(z["dec.h"]).cuda(), torch.from_numpy(z["dec.enc"]).cuda()
    full = dec(h, enc, attention_mask=torch.ones(6, 6, dtype=torch.bool).tril().cuda()).last_hidden_state
    cache = cache_for(dec, 2, 6, page_size)
    if cross_cached:
        cache.cross = dec.cross_cache(enc, page_size)
    cache.add_rows(2, 4)
    o = dec(h[:, :4], enc, past_key_values=cache, return_hidden_states=True)
    assert o.current_key_values is cache and len(o.hidden_states) == 3 and host(cache.lengths).tolist() == [4, 4]
    steps = [o.last_hidden_state]
    for t in (4, 5):
        cache.reserve(1)
        steps.append(dec(h[:, t:t + 1], None if cross_cached else enc, past_key_values=cache).last_hidden_state)
    inc = torch.cat(steps, dim=1)
    assert np.abs(host(inc) - z["dec.full"]).max() <= 4e-2
    assert np.abs(host(inc) - host(full)).max() <= 2e-2
    assert int(cache.shortage) == 0
    with pytest.raises(ValueError):
        dec(h[:1, :1], enc, past_key_values=cache)
    with pytest.raises(RuntimeError):
        dec(h[:, :2], enc, past_key_values=cache)  # several tokens behind others
    with pytest.raises(RuntimeError):
        dec(h[:, :1], enc, attention_mask=torch.ones(1, 1, dtype=torch.bool).cuda(), past_key_values=cache)


@torch.no_grad()
def test_decoder_ragged_prompts_forks_and_resize():
    """Prompts of different lengths (padded), one longer than the concatenated cache's attention takes; rows forked and dropped; the pool cut down on the way:
    every row equals the causal pass over its own tokens."""
    from multimodal_amd.modules.layers.transformer import TransformerDecoder

    torch.manual_seed(0)
    dec = TransformerDecoder(n_layer=2, d_model=192, n_head=3, dim_feedforward=256, activation=torch.nn.GELU, layer_norm_eps=1e-5, norm_first=False,
                             use_cross_attention=False).cuda().eval()
    g = torch.Generator().manual_seed(1)
    counts = [300, 1, 17]
    rows = [torch.randn(n, 192, generator=g) for n in counts]
    cache = cache_for(dec, 6, 400, 16)
    cache.add_rows(3, torch.tensor(counts, dtype=torch.int32, device="cuda"))
    prompt = torch.nn.utils.rnn.pad_sequence(rows, batch_first=True)
    out = dec(prompt.cuda(), past_key_values=cache).last_hidden_state
    assert host(cache.lengths).tolist() == counts
    got = [out[r, n - 1] for r, n in enumerate(counts)]
    for step, parents in enumerate([[0, 0, 1, 2], [3, 2, 1, 1, 0], [4, 0, 2]]):
        cache.fork(torch.tensor(parents, dtype=torch.int32, device="cuda"), reserve=1)
        if step == 1:
            cache.resize(60)
        new = torch.randn(len(parents), 1, 192, generator=g)
        rows = [torch.cat([rows[p], x]) for p, x in zip(parents, new)]
        got = dec(new.cuda(), past_key_values=cache).last_hidden_state[:, 0]
        assert int(cache.shortage) == 0
    for r, row in enumerate(rows):
        full = dec(row[None].cuda(), attention_mask=None if len(row) == 1 else causal(len(row))).last_hidden_state[0, -1] if len(row) <= 288 else None
        if full is not None:
            assert np.abs(host(got[r]) - host(full)).max() <= 2e-2
    assert any(len(row) > 288 for row in rows)
    # the long row: its last state again from a prompt of all its tokens
    long = max(rows, key=len)
    again = cache_for(dec, 1, 400, 7)
    again.add_rows(1, len(long))
    want = dec(long[None].cuda(), past_key_values=again).last_hidden_state[0, -1]
    assert np.abs(host(got[[len(r) for r in rows].index(len(long))]) - host(want)).max() <= 2e-2
    with pytest.raises(ValueError):
        cache.resize(3)


def causal(n):
    return torch.ones(n, n, dtype=torch.bool, device="cuda").tril()


def coca(cfg, cascaded, seed_v):
    from multimodal_amd.models.coca.coca_model import coca_vit

    seed(seed_v)
    model = coca_vit(**cfg, cascaded_pooler=cascaded).eval()
    randomize(model, torch.Generator().manual_seed(seed_v + 1))
    with torch.no_grad():
        model.multimodal_decoder.output_projection.weight.mul_(6.0)  # spread the words, so that rounding rarely decides
    return model.cuda()


def full_log_probs(model, images, sequences):
    """log p(next word) [n, tokens, vocab] in 64 bits from the model's own full forward over the sequences [n, tokens]."""
    ids = sequences.clone()
    pad = model.text_decoder.num_positions - 1 - ids.shape[1]
    ids = torch.nn.functional.pad(ids, (0, pad), value=0)
    return torch.log_softmax(model(images, ids).multimodal_embeddings.double(), -1)[:, :sequences.shape[1]]


@pytest.mark.parametrize("cfg,cascaded", [(SMALL, False), (SMALL, True), (POOL96, False)], ids=["parallel", "cascaded", "three-heads"])
@torch.no_grad()
def test_captions_vs_full_forward(cfg, cascaded):
    from multimodal_amd.models.coca.captioning import generate_captions

    model = coca(cfg, cascaded, 61)
    images = torch.randn(3, 3, 64, 64, generator=torch.Generator().manual_seed(5)).cuda()
    end = 2
    greedy = generate_captions(model, images, 1, end, num_beams=1, length_penalty=0.0)
    assert greedy.sequences.shape == (3, 1, 12) and (greedy.sequences[:, :, 0] == 1).all()
    logp = full_log_probs(model, images, greedy.sequences[:, 0])
    for b in range(3):
        total = 0.0
        for t in range(int(greedy.lengths[b, 0])):
            word = int(greedy.sequences[b, 0, t + 1])
            assert float(logp[b, t].max() - logp[b, t, word]) <= 2 * LOGIT_TOL * 6  # the best word, or one that rounding cannot tell from it
            total += float(logp[b, t, word])
        assert abs(total - float(greedy.scores[b, 0])) <= 2 * LOGIT_TOL * 6 * int(greedy.lengths[b, 0])
    for penalty, page in ((0.0, 16), (1.0, 4)):
        beams = generate_captions(model, images, 1, end, num_beams=4, length_penalty=penalty, page_size=page)
        rank = host(beams.scores) / np.maximum(host(beams.lengths), 1) ** penalty
        assert (np.diff(rank, axis=1) <= 1e-6).all()  # best first
        for k in range(4):
            logp = full_log_probs(model, images, beams.sequences[:, k])
            for b in range(3):
                n = int(beams.lengths[b, k])
                words = beams.sequences[b, k, 1:]
                total = sum(float(logp[b, t, int(words[t])]) for t in range(n))
                assert abs(total - float(beams.scores[b, k])) <= 2 * LOGIT_TOL * 6 * n
                assert (words[:n - 1] != end).all() and (n == 11 or int(words[n - 1]) == end) and (words[n:] == end).all()
            for j in range(k):
                assert not (beams.sequences[:, k] == beams.sequences[:, j]).all(-1).any()  # the beams of an image differ
    again = generate_captions(model, images, 1, end, num_beams=4, length_penalty=1.0, page_size=4)
    assert torch.equal(again.sequences, beams.sequences) and torch.equal(again.scores, beams.scores)
    eager = generate_captions(model, images, 1, end, num_beams=4, length_penalty=1.0, page_size=4, graph=False)  # replays equal eager steps, bit for bit
    assert torch.equal(eager.sequences, beams.sequences) and torch.equal(eager.scores, beams.scores) and torch.equal(eager.lengths, beams.lengths)
    none = generate_captions(model, images[:0], 1, end, num_beams=2)
    assert none.sequences.shape == (0, 2, 12) and none.scores.shape == (0, 2)
    short = generate_captions(model, images[:1], 1, end, num_beams=2, max_length=3)
    assert short.sequences.shape == (1, 2, 3)
    model.train()
    with pytest.raises(RuntimeError):
        generate_captions(model, images, 1, end)


@torch.no_grad()
def test_rows_with_their_own_encoder_states_reordered():
    """Forked rows keep attending to their parents' encoder states: each equals the causal pass of its tokens beside the states it began with."""
    from multimodal_amd.modules.layers.transformer import TransformerDecoder

    torch.manual_seed(2)
    dec = TransformerDecoder(n_layer=2, d_model=128, n_head=2, dim_feedforward=256, activation=torch.nn.GELU, layer_norm_eps=1e-5, norm_first=True,
                             use_cross_attention=True, dim_kv=128).cuda().eval()
    g = torch.Generator().manual_seed(3)
    enc, rows = 3.0 * torch.randn(3, 9, 128, generator=g).cuda(), [torch.randn(4, 128, generator=g) for _ in range(3)]
    cache = cache_for(dec, 6, 16, 4)
    cache.add_rows(3, 4)
    dec(torch.stack(rows).cuda(), enc, past_key_values=cache)
    cache.cross, of = dec.cross_cache(enc, 4), [0, 1, 2]
    for parents in ([2, 0, 0, 1], [3, 1, 0]):
        cache.fork(torch.tensor(parents, dtype=torch.int32, device="cuda"))
        new = torch.randn(len(parents), 1, 128, generator=g)
        rows, of = [torch.cat([rows[p], x]) for p, x in zip(parents, new)], [of[p] for p in parents]
        got = dec(new.cuda(), past_key_values=cache).last_hidden_state[:, 0]
        want = dec(torch.stack(rows).cuda(), enc[of], attention_mask=causal(len(rows[0]))).last_hidden_state[:, -1]
        other = dec(torch.stack(rows).cuda(), enc[[(o + 1) % 3 for o in of]], attention_mask=causal(len(rows[0]))).last_hidden_state[:, -1]
        assert np.abs(host(got) - host(want)).max() <= 2e-2
        assert np.abs(host(other) - host(want)).max() > 0.2  # (the states matter)


@torch.no_grad()
def test_prompt_counts_beyond_the_prompt():
    """A count above the prompt's padded length counts what was stored, no places that were never written."""
    from multimodal_amd.modules.layers.transformer import TransformerDecoder

    torch.manual_seed(4)
    dec = TransformerDecoder(n_layer=1, d_model=128, n_head=2, dim_feedforward=256, activation=torch.nn.GELU, layer_norm_eps=1e-5, norm_first=True,
                             use_cross_attention=False).cuda().eval()
    x = torch.randn(3, 6, 128, generator=torch.Generator().manual_seed(5)).cuda()
    last = []
    for counts in ([9, 3, -2], [5, 3, 0]):
        cache = cache_for(dec, 3, 16, 4)
        cache.pages.fill_(float("nan"))
        cache.add_rows(3, torch.tensor(counts, dtype=torch.int32, device="cuda"))
        dec(x[:, :5], past_key_values=cache)
        assert host(cache.lengths).tolist() == [5, 3, 0]
        cache.reserve(1)
        last.append(dec(x[:, 5:], past_key_values=cache).last_hidden_state)
    assert torch.equal(last[0], last[1]) and bool(torch.isfinite(last[0]).all())


@torch.no_grad()
def test_captions_of_two_streams_and_two_threads():
    """Calls that follow each other on different streams without a wait, and calls from two threads, give what single calls give."""
    from threading import Thread

    from multimodal_amd.models.coca.captioning import generate_captions

    model = coca(SMALL, False, 62)
    g = torch.Generator().manual_seed(6)
    images = [torch.randn(2, 3, 64, 64, generator=g).cuda() for _ in range(2)]
    want = [generate_captions(model, x, 1, 2, num_beams=3) for x in images]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]

    def call(i):
        with torch.no_grad(), torch.cuda.stream(streams[i]):
            got[i] = generate_captions(model, images[i], 1, 2, num_beams=3)

    def check():
        torch.cuda.synchronize()
        for w, r in zip(want, got):
            assert torch.equal(w.sequences, r.sequences) and torch.equal(w.scores, r.scores) and torch.equal(w.lengths, r.lengths)
        got[:] = [None, None]

    for i in range(2):
        call(i)
    check()
    threads = [Thread(target=call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    check()


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@torch.no_grad()
def test_captions_that_lost_keys_are_not_returned(graph, monkeypatch):
    """A pool that is too small from some step on, also where that step is a replay: with pages of two tokens and two a row, the fourth step finds at least 6 of the 8
    live (the rows' last pages and a first one per image) and needs 4."""
    from multimodal_amd import ops
    from multimodal_amd.models.coca.captioning import generate_captions
    from multimodal_amd.modules.layers.paged_cache import PagedKVCache

    model = coca(SMALL, False, 63)
    images = torch.randn(2, 3, 64, 64, generator=torch.Generator().manual_seed(7)).cuda()
    generate_captions(model, images, 1, 2, num_beams=2, page_size=2, graph=graph)
    monkeypatch.setattr(PagedKVCache, "pages_for", staticmethod(lambda rows, *a: rows * 2))
    with pytest.raises(ops.MmamdError, match="lost"):
        generate_captions(model, images, 1, 2, num_beams=2, page_size=2, graph=graph)


@torch.no_grad()
def test_steps_without_a_reserve_equal_the_causal_pass():
    """A prompt that fills its page, then single tokens with no fork or reserve between, up to the table's end and one beyond, which is on record."""
    from multimodal_amd.modules.layers.transformer import TransformerDecoder

    torch.manual_seed(6)
    dec = TransformerDecoder(n_layer=2, d_model=128, n_head=2, dim_feedforward=256, activation=torch.nn.GELU, layer_norm_eps=1e-5, norm_first=True,
                             use_cross_attention=False).cuda().eval()
    x = torch.randn(2, 13, 128, generator=torch.Generator().manual_seed(8)).cuda()
    full = dec(x[:, :12], attention_mask=causal(12)).last_hidden_state
    cache = cache_for(dec, 2, 12, 4)
    cache.pages.fill_(float("nan"))
    cache.add_rows(2, 4)
    got = [dec(x[:, :4], past_key_values=cache).last_hidden_state]
    got += [dec(x[:, t:t + 1], past_key_values=cache).last_hidden_state for t in range(4, 12)]
    assert np.abs(host(torch.cat(got, 1)) - host(full)).max() <= 2e-2  # (as in the tests above)
    assert int(cache.lost) == 0 and host(cache.lengths).tolist() == [12, 12]
    dec(x[:, 12:], past_key_values=cache)
    assert int(cache.lost) == 2 and host(cache.lengths).tolist() == [12, 12]


class RoundedOtherwise:
    """multimodal_amd.ops with attention outputs that are moved by up to one step of bf16, at random."""

    def __init__(self, seed_v):
        from multimodal_amd import ops

        self.ops, self.g = ops, torch.Generator(device="cuda").manual_seed(seed_v)

    def __getattr__(self, name):
        return getattr(self.ops, name)

    def _moved(self, att):
        return (att.float() * (1 + 2.0 ** -8 * (2 * torch.rand(att.shape, generator=self.g, device="cuda") - 1))).bfloat16()

    def attention_fwd(self, *args, **kw):
        return self._moved(self.ops.attention_fwd(*args, **kw))

    def attention_x_fwd(self, *args, **kw):
        att, probs = self.ops.attention_x_fwd(*args, **kw)
        return self._moved(att), probs


@pytest.mark.parametrize("penalty", [0.0, 1.0])
@pytest.mark.parametrize("cfg,cascaded", [(SMALL, False), (SMALL, True), (POOL96, False)], ids=["parallel", "cascaded", "three-heads"])
@torch.no_grad()
def test_every_step_of_a_search_selects_what_full_forwards_select(cfg, cascaded, penalty, monkeypatch):
    """Step by step: the model's own full forward over every beam's tokens gives all continuations in 64 bits; the search's beams have to be among the best of them, no two
    alike, with their totals.

    How far two right log-probabilities of a word may lie apart: the two ways differ in how attention weights and attention outputs are rounded to bf16, by at most half a
    step, 2^-9 of each, in either way, and in what follows from that.  So the outputs of all the decoders' attentions are moved by up to 2^-8 at random, and twice what that
    does at most to the log-probabilities of random words is the tolerance."""
    from multimodal_amd.models.coca import captioning
    from multimodal_amd.modules.layers import multi_head_attention as mha

    model, bsz, beams, steps, end = coca(cfg, cascaded, 64), 8, 4, 11, 2
    g = torch.Generator().manual_seed(9)
    images = torch.randn(bsz, 3, 64, 64, generator=g).cuda()
    words = torch.randint(3, 96, (bsz, 12), generator=g).cuda()
    words[:, 0] = 1
    full = full_log_probs(model, images, words)
    with monkeypatch.context() as m:
        m.setattr(mha, "ops", RoundedOtherwise(3))
        tol = 2 * max(float((full - full_log_probs(model, images, words)).abs().max()) for _ in range(3))
    assert tol > 0
    swapped = words.clone()
    swapped[:, [3, 4]] = words[:, [4, 3]]
    shown = float((full_log_probs(model, images, swapped) - full)[:, 6:].abs().amax((1, 2)).min())
    print(f"tolerance {tol:.4f}, two cached words in each other's place change {shown:.4f}")
    assert shown > 4 * tol

    s = captioning._Search(model, captioning.captioning_embeddings(model, images), 1, end, beams, 12, penalty, 4)
    state = lambda: [t.clone().cpu().numpy() for t in (s.scores.double(), s.lengths, s.finished, s.sequences)]  # noqa: E731
    for t in range(steps):
        scores, lengths, finished, seqs = state()
        s.place.copy_(s.positions[t:t + 1])
        s.step()
        scores2, lengths2, finished2, seqs2 = state()
        rows = torch.cat([torch.ones(bsz, beams, 1, dtype=torch.int64), torch.from_numpy(seqs[:, :, :t])], 2).cuda()
        logp = torch.stack([full_log_probs(model, images, rows[:, k].contiguous())[:, t] for k in range(beams)], 1).cpu().numpy()
        total = scores[..., None] + logp
        total[finished] = -np.inf
        total[finished, end] = scores[finished]
        after = lengths + ~finished
        rank = total / np.maximum(after, 1)[..., None] ** penalty
        least = np.sort(rank.reshape(bsz, -1), 1)[:, -beams]
        for b in range(bsz):
            taken = set()
            for k in range(beams):
                for p in range(beams):  # the beam that it continues: its tokens, and its word
                    if finished[b, p]:
                        fits, word = (seqs2[b, k] == seqs[b, p]).all(), end
                    else:
                        fits, word = (seqs2[b, k, :t] == seqs[b, p, :t]).all() and scores[b, p] > -np.inf, seqs2[b, k, t]
                    if fits and lengths2[b, k] == after[b, p] and (p, word) not in taken:
                        break
                else:
                    raise AssertionError((t, b, k, seqs2[b, k], seqs[b]))
                taken.add((p, word))
                assert abs(scores2[b, k] - total[b, p, word]) <= (0 if finished[b, p] else tol), (t, b, k)
                assert rank[b, p, word] >= least[b] - 2 * tol / max(1, after[b, p]) ** penalty, (t, b, k)
                assert finished2[b, k] == (finished[b, p] or word == end)
                assert (seqs2[b, k, after[b, p]:] == end).all()
            place = scores2[b] / np.maximum(lengths2[b], 1) ** penalty
            assert (np.diff(place) <= 1e-6).all()
    got = captioning.generate_captions(model, images, 1, end, num_beams=beams, length_penalty=penalty, page_size=4)
    assert torch.equal(got.sequences[:, :, 1:], s.sequences) and torch.equal(got.scores, s.scores) and torch.equal(got.lengths, s.lengths)
