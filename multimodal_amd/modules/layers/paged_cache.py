"""Key-value cache in pages for serving the decoders (TransformerDecoder, MultiHeadAttentionWithCache): rows (sequences) are continued, forked, dropped and
added without moving their keys and values, where the reference concatenates the whole cache per token and layer
(modules/layers/multi_head_attention.py:158-179) and cannot reorder it.  The operators underneath: ops.paged_attention, paged_append, paged_fork, paged_compact."""
from typing import List, Optional, Tuple, Union

import torch
from torch import Tensor

from ... import ops


class PagedKVCache:
    """Keys and values of `n_layer` attention layers for a changing set of rows.  The decoders serve bfloat16 and 64- or 96-wide heads (prompts of more than 288 tokens: 64);
    append() and attend() by themselves every type and width of ops.paged_attention.

    pages [num_pages, n_layer, 2, num_heads, page_size, head_dim]: a page holds `page_size` tokens of one row for every layer, so that sharing, copying and
    freeing it is one decision.  page_table int32 [rows, slots], lengths int32 [rows], refcounts int32 [num_pages] as in ops.paged_fork; all on the device, and no
    method but compact() waits for it.

        cache = PagedKVCache(...)
        cache.add_rows(batch, prompt_tokens)                # or a tensor of counts
        decoder(prompt, past_key_values=cache)              # stores the prompt, advances the lengths
        cache.fork(parents, reserve=1)                      # rows of the next token: beams reordered, rows dropped or doubled
        decoder(token_states, past_key_values=cache)        # [rows, 1, d]

    A decoder's step takes room for its token by itself where none is left of an int `reserve`; with one per row the room is the caller's.

    num_pages has to cover what is live and, at a fork, what is fresh beside it: pages that were reserved and hold no token yet are taken anew by every fork,
    while the old rows' still count.  pages_for() is always enough, less serves rows that share pages or end early.  What could not be had is counted in
    `shortage` (int32 [1], of the last fork) and added to `lost` (int32 [1], since reset()), and so are tokens beyond a row's table, and those of a decoder's step
    whose row got no room by a `reserve` per row: tokens of those places are gone, the rows' outputs are wrong from there on, and what is done with a search's results
    should look at `lost` first.  (Replays of a captured step advance the lengths unseen: where they pass max_tokens is the caller's to know.)"""

    def __init__(self, n_layer: int, num_heads: int, head_dim: int, num_pages: int, max_tokens: int, page_size: int = 16, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda") -> None:
        if head_dim not in (64, 96, 128):
            raise ops.MmamdError(f"the paged attention kernels are built for 64-, 96- and 128-wide heads, got {head_dim}")
        if min(n_layer, num_heads, num_pages, max_tokens, page_size) < 1:
            raise ValueError("n_layer, num_heads, num_pages, max_tokens and page_size must be at least 1")
        self.page_size, self.max_tokens = page_size, max_tokens
        self.pages = torch.empty((num_pages, n_layer, 2, num_heads, page_size, head_dim), dtype=dtype, device=device)
        self.cross: Optional["PagedKVCache"] = None  # keys and values of encoder states, for decoders with cross-attention, row for row
        self._view = False
        self._moves, self._made = [0], 0  # how often pages were moved or taken from under shared_rows() views, which look at their maker's count; its state at their making
        self.reset()

    @staticmethod
    def pages_for(rows: int, max_tokens: int, page_size: int = 16, reserve: int = 1) -> int:
        """Pages that suffice whatever happens, for at most `rows` rows of max_tokens tokens before and after every fork, none of which asks for more than `reserve`
        tokens a row (nor add_rows, where rows are there already): the old rows' pages, and a fresh row's copy of a partial page and its reserved ones."""
        if min(rows, max_tokens, page_size) < 1 or reserve < 0:
            raise ValueError(f"rows, max_tokens and page_size must be at least 1 and reserve at least 0, got {rows}, {max_tokens}, {page_size}, {reserve}")
        slots = -(-max_tokens // page_size)
        return rows * (slots + min(slots, 1 - (-reserve // page_size)))

    def reset(self) -> None:
        """No rows, every page free."""
        self._owned("reset")
        self._moves[0] += 1
        dev = self.pages.device
        slots = -(-self.max_tokens // self.page_size)
        self.page_table = torch.empty((0, slots), dtype=torch.int32, device=dev)
        self.lengths = torch.empty((0,), dtype=torch.int32, device=dev)
        self.refcounts = torch.zeros((self.pages.shape[0],), dtype=torch.int32, device=dev)
        self.shortage = torch.zeros((1,), dtype=torch.int32, device=dev)
        self.lost = torch.zeros((1,), dtype=torch.int32, device=dev)
        self._prompt: Union[None, int, Tensor] = None
        # what the host knows without asking the device: tokens that every row has room for (None: of each row's own), and the most that a row may hold (None: unknown)
        self._room: Optional[int] = 0
        self._most: Optional[int] = 0
        self._room_of = self.page_table  # the table that _room speaks of: one that was put in its place by hand has the room that its maker knows

    @property
    def rows(self) -> int:
        return self.page_table.shape[0]

    @property
    def n_layer(self) -> int:
        return self.pages.shape[1]

    def _owned(self, what: str) -> None:
        if self._view:
            raise ops.MmamdError(f"{what}: shared_rows() reads the pages of another cache and holds no references to them")

    def layer(self, i: int) -> Tuple[Tensor, Tensor]:
        """(key_pages, value_pages) of layer i, views [num_pages, num_heads, page_size, head_dim]."""
        return self.pages[:, i, 0], self.pages[:, i, 1]

    def add_rows(self, rows: int, tokens: Union[int, Tensor]) -> None:
        """`rows` new rows in the place of the present ones (which must be none, or are dropped), with pages for prompts of `tokens` tokens (an int, or
        int32 [rows]); the next decoder call stores them.  `cross` stays as it is: assign the new rows' before or after."""
        room = self.page_table.shape[1] * self.page_size
        if isinstance(tokens, int) and tokens > room:
            raise ValueError(f"prompts of {tokens} tokens for rows of {room}")
        self.fork(torch.full((rows,), -1, dtype=torch.int32, device=self.pages.device), reserve=tokens, cross=False)
        self._prompt, self._most = tokens, 0
        self._moves[0] += 1

    def fork(self, parents: Tensor, reserve: Union[int, Tensor] = 1, cross: bool = True) -> None:
        """Row r becomes a continuation of the present row parents[r] (int32, any shape, -1: an empty row) with room for `reserve` more tokens.  The rows of
        `cross` follow (the row of an empty one has no states); cross=False leaves them, where a row and its parent have the same states in any case."""
        self._owned("fork")
        if cross and self.cross is not None:
            if self.cross.rows != self.rows:
                raise ValueError(f"the encoder states' cache has {self.cross.rows} rows, this one {self.rows}")
            follow = self.cross._continued(parents.reshape(-1))
        else:
            follow = self.cross
        s = ops.paged_fork(self.pages, self.page_table, self.lengths, self.refcounts, parents.reshape(-1), reserve=reserve)
        self.page_table, self.lengths, self.refcounts, self.shortage = s
        self.lost = self.lost + s.shortage
        self._room, self._room_of = None if isinstance(reserve, Tensor) else int(reserve), self.page_table
        self.cross = follow
        self._prompt = None

    def reserve(self, tokens: Union[int, Tensor] = 1) -> None:
        """Room for `tokens` more tokens in every row."""
        self.fork(torch.arange(self.rows, dtype=torch.int32, device=self.pages.device), reserve=tokens, cross=False)

    def shared_rows(self, parents: Tensor) -> "PagedKVCache":
        """Another view of the same pages: its row r reads what row parents[r] (int64) holds now.  For reading only -- it takes no references, so storing, forking
        and compacting through it are refused, and this cache has to keep the rows where they are: attending through the view is refused after compact, resize,
        reset and add_rows; no fork may drop the rows (the host does not see which it drops)."""
        view = object.__new__(PagedKVCache)
        view.__dict__.update(self.__dict__)
        if not self._view:
            view._made = self._moves[0]
        view.page_table, view.lengths, view._view = self.page_table[parents], self.lengths[parents], True
        return view

    def _continued(self, parents: Tensor) -> "PagedKVCache":
        """shared_rows() for fork's parents: a number outside the rows gives a row without tokens."""
        if self.rows == 0:
            view = self.shared_rows(torch.zeros((0,), dtype=torch.int64, device=parents.device))
            view.page_table, view.lengths = view.page_table.new_full((len(parents), view.page_table.shape[1]), -1), view.lengths.new_zeros((len(parents),))
            return view
        view = self.shared_rows(parents.clamp(0, self.rows - 1).long())
        view.lengths = torch.where((parents >= 0) & (parents < self.rows), view.lengths, 0)
        return view

    def _held_in(self, held: List[Tensor]) -> None:
        """The state moves into tensors that stay where they are: what a captured step reads and what it leaves for its next replay."""
        for to, new in zip(held, (self.page_table, self.lengths, self.refcounts, self.lost)):
            to.copy_(new)
        self._same_room(held[0])
        self.lengths, self.refcounts, self.lost = held[1:]

    def _same_room(self, table: Tensor) -> None:
        """`table` takes the present one's place, with as much room in its rows."""
        if self.page_table is self._room_of:
            self._room_of = table
        self.page_table = table

    def append(self, layer: int, k: Tensor, v: Tensor, counts: Optional[Tensor] = None) -> None:
        """Stores k, v [rows, tokens, num_heads, head_dim] (counts int32 [rows]: the first ones of each row) behind the rows' tokens; advance() is the caller's."""
        self._owned("append")
        kp, vp = self.layer(layer)
        ops.paged_append(k, v, kp, vp, self.page_table, self.lengths, counts)

    def attend(self, layer: int, q: Tensor, k: Optional[Tensor] = None, v: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
        """One token a row: q [rows, heads, head_dim] over the row's tokens in `layer`, and over its new one, which is stored, if k and v are given."""
        if k is not None:
            self._owned("attend with new tokens")
        if self._view and self._made != self._moves[0]:
            raise ops.MmamdError("attend: the pages of this view's rows were moved or freed by the cache that shared_rows() was called on")
        kp, vp = self.layer(layer)
        return ops.paged_attention(q, kp, vp, self.page_table, self.lengths, k, v, scale)

    def advance(self, tokens: Union[int, Tensor] = 1) -> None:
        """Counts tokens that every layer has stored.  A length ends at the table's room; what is beyond it has no place and is counted in `lost`."""
        self._owned("advance")
        if isinstance(tokens, Tensor):
            self._advance(tokens, None, None)
        else:
            self._advance(tokens, self._most + tokens if self._most is not None else None, max(0, self._room - tokens) if self._room is not None else None)

    def _advance(self, tokens: Union[int, Tensor], most: Optional[int], room: Optional[int]) -> None:
        cap = self.page_table.shape[1] * self.page_size
        after = self.lengths + tokens
        if most is None or most > cap:
            self.lengths, most = after.clamp(max=cap), cap
            self.lost = self.lost + (after - self.lengths).sum(dtype=torch.int32)
        else:
            self.lengths = after
        self._prompt, self._most, self._room = None, most, room

    def _stored_prompt(self, tokens: int) -> None:
        """advance() for the prompts [rows, tokens, ...] that add_rows announced (a count beyond the prompt has stored nothing there)."""
        if isinstance(self._prompt, Tensor):
            self._advance(self._prompt.clamp(0, tokens), tokens, 0)
        else:
            self.advance(tokens)

    def _make_room(self) -> None:
        """Before a step: a place for each row's token where the host knows that none was asked for; where it does not know, tokens without one are counted."""
        known = self._room is not None and self.page_table is self._room_of
        if known and self._room == 0:
            self.reserve(1)
        elif not known and self.rows > 0:
            slots = self.page_table.shape[1]
            at = torch.div(self.lengths, self.page_size, rounding_mode="floor").long()
            page = torch.gather(self.page_table, 1, at.clamp(0, slots - 1)[:, None])[:, 0]
            self.lost = self.lost + ((at < slots) & ((page < 0) | (page >= self.pages.shape[0]))).sum(dtype=torch.int32)

    def compact(self) -> int:
        """Moves the live pages to the front and says how many they are (this waits for the device)."""
        self._owned("compact")
        self._moves[0] += 1
        table, self.refcounts, live = ops.paged_compact(self.pages, self.page_table, self.refcounts)
        self._same_room(table)
        return int(live)

    def resize(self, num_pages: int) -> None:
        """Another number of pages: the live ones are moved to the front and kept, the rest of the memory is given back (or added)."""
        live = self.compact()
        if num_pages < max(live, 1):
            raise ValueError(f"{live} pages are live, {num_pages} are too few")
        keep = min(num_pages, self.pages.shape[0])
        pages = torch.empty((num_pages, *self.pages.shape[1:]), dtype=self.pages.dtype, device=self.pages.device)
        refcounts = torch.zeros((num_pages,), dtype=torch.int32, device=self.pages.device)
        pages[:live].copy_(self.pages[:live])
        refcounts[:keep].copy_(self.refcounts[:keep])
        self.pages, self.refcounts = pages, refcounts
