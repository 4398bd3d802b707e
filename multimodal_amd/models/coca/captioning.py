"""Captions from a CoCa model: the generative read-out of the decoder that the captioning loss trains (models/coca/coca_model.py:434-466 of the reference,
which has none for it).  Beam search, one token of all beams per step, with the keys and values of both decoders in pages."""
from threading import Lock
from typing import Dict, NamedTuple, Optional

import torch
from torch import Tensor

from ... import ops
from ...modules.layers.paged_cache import PagedKVCache
from ...modules.layers.transformer import TransformerOutput
from .coca_model import CoCaModel


class Captions(NamedTuple):
    """Best first: token ids int64 [bsz, beams, max_length] (filled up with the end token), log-probabilities fp32 and lengths int32 [bsz, beams]
    (tokens behind the begin token, the end token among them)."""
    sequences: Tensor
    scores: Tensor
    lengths: Tensor


def captioning_embeddings(model: CoCaModel, images: Tensor) -> Tensor:
    """The pooled image embeddings [bsz, queries, dim] that the multimodal decoder reads (coca_model.py:66-87 of the reference)."""
    out = model.vision_encoder(images)
    states = out.last_hidden_state if isinstance(out, TransformerOutput) else out[0] if isinstance(out, tuple) else out
    pooled = model.vision_pooler(states)
    return pooled[0] if isinstance(pooled, list) else pooled[:, 1:]


# A search with a graph has a stream of its own (the legacy default stream cannot be captured): one per device, since the allocator keeps what was freed per
# stream, and new ones would each hold the caches of a search.  One search at a time is on it.
_SEARCH_STREAMS: Dict[torch.device, torch.cuda.Stream] = {}
_searching = Lock()


class _Search:
    """The state of one search in tensors that stay where they are, so that a step can be captured in a HIP graph and replayed."""

    def __init__(self, model: CoCaModel, states: Tensor, begin: int, end: int, beams: int, max_length: int, length_penalty: float, page_size: int) -> None:
        self.text, self.fusion, self.end, self.length_penalty = model.text_decoder.transformer_decoder, model.multimodal_decoder, end, length_penalty
        emb = model.text_decoder.embeddings
        self.table = emb._packed.get(emb.token_embeddings.weight, torch.float32)
        self.positions = emb._packed.get(emb.position_embeddings, torch.float32)
        bsz, dev = states.shape[0], states.device
        rows = self.rows = bsz * beams
        self.caches = []
        for decoder in (self.text, self.fusion.transformer_decoder):
            att = decoder.layer[0].attention
            pages = PagedKVCache.pages_for(rows, max_length, page_size)
            self.caches.append(PagedKVCache(len(decoder.layer), att.num_heads, att.q_proj.out_features // att.num_heads, pages, max_length, page_size, device=dev))
        # the beams of an image read the same pages, and a beam is only ever continued within its image: one table for the whole search
        cross = self.fusion.transformer_decoder.cross_cache(states.contiguous(), page_size)
        self.caches[1].cross = cross.shared_rows(torch.arange(bsz, device=dev).repeat_interleave(beams))
        for cache in self.caches:
            cache.fork(torch.full((rows,), -1, dtype=torch.int32, device=dev), reserve=1, cross=False)
        self.scores = torch.full((bsz, beams), float("-inf"), device=dev)
        self.scores[:, 0] = 0.0
        self.lengths = torch.zeros((bsz, beams), dtype=torch.int32, device=dev)
        self.finished = torch.zeros((bsz, beams), dtype=torch.bool, device=dev)
        self.sequences = torch.full((bsz, beams, max_length - 1), end, dtype=torch.int64, device=dev)  # what follows the begin token
        self.tokens = torch.full((bsz, beams), begin, dtype=torch.int64, device=dev)
        self.place = self.positions[:1].clone()
        self.held = [[c.page_table, c.lengths, c.refcounts, c.lost] for c in self.caches]

    def step(self) -> None:
        """One more token of every beam."""
        x = ops.embed_tokens(self.tokens.view(self.rows, 1), self.table, self.place).view(self.rows, 1, -1)
        x = self.text(x, past_key_values=self.caches[0]).last_hidden_state
        x = self.fusion.transformer_decoder(x, past_key_values=self.caches[1]).last_hidden_state
        r = ops.beam_search_step(self.fusion.project(x.view(self.rows, -1)), self.scores, self.lengths, self.finished, self.sequences, self.end, self.length_penalty)
        for to, new in zip((self.scores, self.lengths, self.finished, self.tokens, self.sequences), (r.scores, r.lengths, r.finished, r.tokens, r.sequences)):
            to.copy_(new)
        for cache, held in zip(self.caches, self.held):
            cache.fork(r.parents, reserve=1, cross=False)
            cache._held_in(held)

    def run(self, steps: int, graph: bool) -> None:
        replay = None
        for t in range(steps):
            self.place.copy_(self.positions[t:t + 1])
            if graph and replay is None and t == 2 and steps > 4:
                # two steps went before on this stream, with a wait between them: the kernel-ready weights are made and nobody waits for their making
                replay = torch.cuda.CUDAGraph()
                replay.capture_begin(capture_error_mode="thread_local")
                try:
                    self.step()
                finally:
                    replay.capture_end()
            if replay is None:
                self.step()
                if t == 0 and graph:
                    torch.cuda.current_stream().synchronize()
            else:
                replay.replay()
            if t % 8 == 7 and bool(self.finished.all()):
                break
        if replay is not None:
            torch.cuda.current_stream().synchronize()  # the graph's own memory goes with it
        if int(self.caches[0].lost + self.caches[1].lost) != 0:
            raise ops.MmamdError("generate_captions: keys and values had no page to go to (PagedKVCache.lost)")


@torch.no_grad()
def generate_captions(model: CoCaModel, images: Tensor, begin: int, end: int, num_beams: int = 5, max_length: Optional[int] = None,
                      length_penalty: float = 1.0, page_size: int = 16, graph: bool = True) -> Captions:
    """Captions of images [bsz, ...] by beam search from token `begin` until every beam has taken `end` or has max_length tokens (default and at most: the
    text decoder's positions without its CLS).  Ranked by log-probability / length ** length_penalty.  graph: from the third token on a step is a replayed
    HIP graph, in place of some three hundred launches from Python; such calls from several threads take turns."""
    if model.training:
        raise ops.MmamdError("generate_captions: call model.eval() first")
    text, fusion = model.text_decoder, model.multimodal_decoder
    places = text.num_positions - (1 if text.embed_cls else 0)
    max_length = places if max_length is None else max_length
    if not 2 <= max_length <= places:
        raise ValueError(f"max_length must lie between 2 and the decoder's {places} positions, got {max_length}")
    if not 1 <= num_beams <= 32:
        raise ValueError(f"num_beams must lie between 1 and 32 (ops.beam_search_step), got {num_beams}")
    if fusion.output_projection is None:
        raise ValueError("the multimodal decoder has no output projection to the vocabulary")
    vocab = text.embeddings.token_embeddings.num_embeddings
    if not (0 <= begin < vocab and 0 <= end < min(vocab, fusion.output_projection.out_features)) or fusion.output_projection.out_features > vocab:
        raise ValueError(f"begin {begin} and end {end} must be words of the vocabulary of {vocab}, which the output projection must not exceed")
    if not images.is_cuda:
        raise ops.MmamdError(f"generate_captions: the images are on {images.device}: the MI355X path needs HIP device tensors (no CPU fallback)")
    if images.shape[0] == 0:  # (the encoders take no empty batch)
        empty = torch.zeros((0, num_beams), device=images.device)
        return Captions(empty[:, :, None].expand(0, num_beams, max_length).long(), empty, empty.int())

    def search() -> Captions:
        s = _Search(model, states, begin, end, num_beams, max_length, length_penalty, page_size)
        s.run(max_length - 1, graph)
        first = torch.full((states.shape[0], num_beams, 1), begin, dtype=torch.int64, device=states.device)
        return Captions(torch.cat([first, s.sequences], dim=2), s.scores, s.lengths)

    with torch.cuda.device(images.device):
        if not graph:
            states = captioning_embeddings(model, images)
            return search()
        with _searching:
            states = captioning_embeddings(model, images)
            main = torch.cuda.current_stream()
            side = _SEARCH_STREAMS.get(states.device)
            if side is None:
                side = _SEARCH_STREAMS[states.device] = torch.cuda.Stream(states.device)
            side.wait_stream(main)
            try:
                with torch.cuda.stream(side):
                    result = search()
            finally:
                main.wait_stream(side)
        for t in result:
            t.record_stream(main)
        return result
