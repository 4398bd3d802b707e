"""Captions from a CoCa model: the generative read-out of the decoder that the captioning loss trains (models/coca/coca_model.py:434-466 of the reference,
which has none for it).  Beam search, one token of all beams per step, with the keys and values of both decoders in pages."""
from typing import NamedTuple, Optional

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


@torch.no_grad()
def generate_captions(model: CoCaModel, images: Tensor, begin: int, end: int, num_beams: int = 5, max_length: Optional[int] = None,
                      length_penalty: float = 1.0, page_size: int = 16) -> Captions:
    """Captions of images [bsz, ...] by beam search from token `begin` until every beam has taken `end` or has max_length tokens (default and at most: the
    text decoder's positions without its CLS).  Ranked by log-probability / length ** length_penalty."""
    if model.training:
        raise ops.MmamdError("generate_captions: call model.eval() first")
    text, fusion = model.text_decoder, model.multimodal_decoder
    places = text.num_positions - (1 if text.embed_cls else 0)
    max_length = places if max_length is None else max_length
    if not 2 <= max_length <= places:
        raise ValueError(f"max_length must lie between 2 and the decoder's {places} positions, got {max_length}")
    if num_beams < 1:
        raise ValueError(f"num_beams must be at least 1, got {num_beams}")
    if fusion.output_projection is None:
        raise ValueError("the multimodal decoder has no output projection to the vocabulary")
    emb = text.embeddings
    table, positions = emb._packed.get(emb.token_embeddings.weight, torch.float32), emb._packed.get(emb.position_embeddings, torch.float32)
    states = captioning_embeddings(model, images)
    bsz, dev = states.shape[0], states.device
    rows = bsz * num_beams

    def cache_of(decoder) -> PagedKVCache:
        att = decoder.layer[0].attention
        slots = -(-max_length // page_size)
        return PagedKVCache(len(decoder.layer), att.num_heads, att.q_proj.out_features // att.num_heads, max(1, rows * (slots + 2)), max_length, page_size, device=dev)

    caches = [cache_of(text.transformer_decoder), cache_of(fusion.transformer_decoder)]
    # the beams of an image read the same pages, and a beam is only ever continued within its image: one table for the whole search
    cross = fusion.transformer_decoder.cross_cache(states.contiguous(), page_size)
    caches[1].cross = cross.shared_rows(torch.arange(bsz, device=dev).repeat_interleave(num_beams))
    for cache in caches:
        cache.add_rows(rows, 1)
        cache._prompt = None  # the first token is a step like the others

    scores = torch.full((bsz, num_beams), float("-inf"), device=dev)
    scores[:, 0] = 0.0
    lengths = torch.zeros((bsz, num_beams), dtype=torch.int32, device=dev)
    finished = torch.zeros((bsz, num_beams), dtype=torch.bool, device=dev)
    sequences = torch.full((bsz, num_beams, max_length), end, dtype=torch.int64, device=dev)
    sequences[:, :, 0] = begin
    tokens = sequences[:, :, 0].contiguous()
    if rows == 0:
        return Captions(sequences, scores, lengths)
    for t in range(max_length - 1):
        x = ops.embed_tokens(tokens.view(rows, 1), table, positions[t:t + 1].contiguous()).view(rows, 1, -1)
        x = text.transformer_decoder(x, past_key_values=caches[0]).last_hidden_state
        x = fusion.transformer_decoder(x, past_key_values=caches[1]).last_hidden_state
        # what follows the begin token is chosen and reordered; it is the same for every beam
        step = ops.beam_search_step(fusion.project(x.view(rows, -1)), scores, lengths, finished, sequences[:, :, 1:].contiguous(), end, length_penalty)
        scores, lengths, finished, tokens = step.scores, step.lengths, step.finished, step.tokens
        sequences = torch.cat([sequences[:, :, :1], step.sequences], dim=2)  # (data movement)
        if t + 2 >= max_length or (t % 8 == 7 and bool(finished.all())):
            break
        for cache in caches:
            cache.fork(step.parents, reserve=1)
    return Captions(sequences, scores, lengths)
