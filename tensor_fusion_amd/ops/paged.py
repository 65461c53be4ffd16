"""A paged KV cache and what writes, reads and attends over it
(native/ops/paged_cache.hip, paged_attention.hip, paged_binding.cpp).

A pool is [pages, kv_heads, page_size, head_dim], one for keys and one for
values. A token's slot is page * page_size + offset; which pages a sequence
owns, and in which order, its row of a block table says:

    cache = paged.make_cache(pages, page_size, kv_heads, head_dim)
    q = paged.rope_kv_write(cache, q_in, k_in, v_in, cos, sin, pos, slots,
                            heads)
    out = paged.paged_attention(q, cache, q_starts, kv_lens, block_table)

A pool is bf16, fp16, or e4m3 with one scale a token and head (`quantized`):
a byte s for 2**(s - 127), the smallest power of two with
max|x| <= 448 * scale. The value that a code stands for is code * scale.

The operators serve: they have no backward pass and no forward mode, and
refuse tensors that ask for either. They run on the current stream of the tensors' device and never
wait for the GPU; lengths, slots and tables stay on the device, so that a
captured graph is replayed while they change. Shapes, types and devices are
checked on the host (ValueError), and that the tensors are plain ones, with
their values in their memory; what lies on the device is checked by the
kernels, which read and write nothing outside of the tensors: see each
operator for what they answer instead.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os
from dataclasses import dataclass

import torch

from . import fused

HEAD_DIMS = (32, 64, 128)

_EXT = None


def _ext():
    """The binding; missing, it is an error, as the library it calls is."""

    global _EXT
    if _EXT is None:
        fused.lib()
        path = os.path.join(fused._native_dir(), "tf_paged.so")
        if not os.path.exists(path):
            raise fused.FusedOpsMissing(
                f"{path} not built — run python build_native.py")
        loader = importlib.machinery.ExtensionFileLoader("tf_paged", path)
        ext = importlib.util.module_from_spec(
            importlib.util.spec_from_loader("tf_paged", loader))
        loader.exec_module(ext)
        _EXT = ext
    return _EXT


class PagedKVCache:
    """One layer's pages: k and v [pages, kv_heads, page_size, head_dim],
    without gaps, bf16, fp16 or float8_e4m3fn; for the last k_scale and
    v_scale, uint8 [pages, kv_heads, page_size]. page_size is a power of two
    from 16 to 1024, head_dim 32, 64 or 128."""

    __slots__ = ("_tensors", "_pools")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        self._pools = _ext().pools(k, v, k_scale, v_scale)
        self._tensors = (k, v, k_scale, v_scale)

    @property
    def k(self):
        return self._tensors[0]

    @property
    def v(self):
        return self._tensors[1]

    @property
    def k_scale(self):
        return self._tensors[2]

    @property
    def v_scale(self):
        return self._tensors[3]

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def dtype(self):
        return self.k.dtype

    @property
    def device(self):
        return self.k.device

    @property
    def quantized(self) -> bool:
        return self.k_scale is not None


def make_cache(pages: int, page_size: int, kv_heads: int, head_dim: int,
               dtype=torch.bfloat16, quantized: bool = False,
               device="cuda") -> PagedKVCache:
    """A cleared cache. dtype is that of the rows; a quantised one takes
    rows of either 16-bit type and holds 8 bits and a scale."""

    shape = (pages, kv_heads, page_size, head_dim)
    if quantized:
        # codes 0, scale 1
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device)
                .view(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.full(shape[:3], 127, dtype=torch.uint8,
                             device=device) for _ in range(2))
        return PagedKVCache(k, v, ks, vs)
    return PagedKVCache(torch.zeros(shape, dtype=dtype, device=device),
                        torch.zeros(shape, dtype=dtype, device=device))


@dataclass
class PagedBatch:
    """New tokens of some sequences, as the operators take them: packed one
    sequence after the other, token i at position pos[i] of its sequence, in
    slot slots[i]; kv_lens counts them. page_size is the one that the slots
    were worked out for, and has to be the caches'; None where they are a
    caller's own."""

    q_starts: torch.Tensor      # int32 [B + 1]
    kv_lens: torch.Tensor       # int32 [B]
    block_table: torch.Tensor   # int32 [B, columns]
    pos: torch.Tensor           # int64 [tokens]
    slots: torch.Tensor         # int64 [tokens]
    page_size: int | None = None

    @classmethod
    def of(cls, block_table, past, new, page_size: int) -> "PagedBatch":
        """`new` tokens (a number, or one for each sequence) behind the
        first `past` (integers [B]) of the sequences of a block table. With
        a number everything is worked out on the device, so that a step that
        is captured goes on from wherever `past` stands at the replay. A list
        is worked out on the host, and its copies wait for the stream."""

        if page_size < 1:
            raise ValueError(f"no page_size of {page_size}")
        (B, cols), device = block_table.shape, block_table.device
        past = past.to(torch.int64)
        if isinstance(new, int):
            starts = torch.arange(B + 1, device=device,
                                  dtype=torch.int32) * new
            pos = past[:, None] + torch.arange(new, device=device)
            seq = torch.arange(B, device=device)[:, None].expand(B, new)
            pos, seq, lens = pos.flatten(), seq.flatten(), past + new
        else:
            if len(new) != B or min(new, default=0) < 0:
                raise ValueError(f"{len(new)} counts {list(new)[:8]} for {B} "
                                 "sequences")
            n = torch.tensor(new, dtype=torch.int64)
            starts = torch.zeros(B + 1, dtype=torch.int64)
            starts[1:] = n.cumsum(0)
            seq = torch.arange(B).repeat_interleave(n)
            pos = torch.arange(len(seq)) - starts[seq]
            seq = seq.to(device)
            pos = pos.to(device) + past[seq]
            lens = past + n.to(device)
            starts = starts.to(torch.int32).to(device)
        if cols == 0 and len(pos):
            raise ValueError("a block table without columns has no slots")
        # a position that the table does not hold has no slot
        col = pos // page_size
        there = (pos >= 0) & (col < cols)
        page = block_table[seq, col.clamp(0, max(cols - 1, 0))]
        slots = page.to(torch.int64) * page_size + pos % page_size
        slots = torch.where(there, slots, -1)
        return cls(starts, lens.to(torch.int32), block_table, pos, slots,
                   page_size)

    def check(self, cache: PagedKVCache) -> None:
        size = self.page_size
        if size is not None and size != cache._tensors[0].shape[2]:
            raise ValueError(f"a batch for pages of {self.page_size} tokens, "
                             f"and a cache with pages of {cache.page_size}")

    def over(self, caches):
        """The layers' caches, as a model takes them with this batch."""

        layers = [(c, self) for c in caches]
        for c, _ in layers:
            self.check(c)
        return layers


def attend(q_in, k_in, v_in, cos, sin, cache: PagedKVCache,
           batch: PagedBatch, heads: int):
    """A layer's attention between its projections: rope_kv_write, then
    paged_attention. Returns [tokens, heads * head_dim]."""

    batch.check(cache)
    q = rope_kv_write(cache, q_in, k_in, v_in, cos, sin, batch.pos,
                      batch.slots, heads)
    out = paged_attention(q, cache, batch.q_starts, batch.kv_lens,
                          batch.block_table)
    return out.flatten(1)


def kv_write(cache: PagedKVCache, k, v, slots) -> None:
    """pages[slots] <- k, v; k and v are [n, kv_heads, head_dim], rows and
    heads at any stride, slots int64 [n].

    A quantised cache rounds each row to e4m3 under its own scale; a row
    that holds an infinity or NaN becomes NaN throughout, and fp16 values
    are held to +-61440, the last e4m3 step that fp16 has. Rows whose slot
    is negative (padding) or past the pool are not written. Slots that are
    written have to differ: of two rows for one slot, parts of either may
    stay. Rows may lie in the cache themselves: they are copied first."""

    (_EXT or _ext()).kv_write(cache._pools, k, v, slots)


def rope_kv_write(cache: PagedKVCache, q_in, k_in, v_in, cos, sin, pos,
                  slots, heads: int):
    """One launch for a layer: q rotated to a fresh [n, heads, head_dim],
    k rotated and v copied into the pages (quantised from the 32-bit
    products), as kv_write has it.

    q_in, k_in, v_in: [n, heads * head_dim] and [n, kv_heads * head_dim],
    which may be column slices of one merged product; cos, sin: float32
    [positions, head_dim / 2] for interleaved pairs; pos, slots: int64 [n].
    A row whose position lies outside of the tables becomes NaN."""

    return (_EXT or _ext()).rope_kv_write(cache._pools, q_in, k_in, v_in,
                                          cos, sin, pos, slots, heads)


def kv_read(cache: PagedKVCache, slots, dtype=None):
    """k, v [n, kv_heads, head_dim] of the slots (int64 [n], any order, any
    of them more than once), dequantised to `dtype` (bfloat16 if not given)
    where the cache is quantised. A negative slot reads 0, one past the
    pool NaN."""

    return (_EXT or _ext()).kv_read(cache._pools, slots, dtype)


def paged_attention(q, cache: PagedKVCache, q_starts, kv_lens, block_table,
                    scale=None, causal: bool = True, out=None):
    """Attention of a packed batch of new tokens over the pages of their
    sequences, the new tokens' own keys (already written) among them.

    q: [tokens, heads, head_dim], tokens and heads at any stride, heads a
    multiple of the cache's; q_starts: int32 [B + 1], sequence b's tokens
    are q_starts[b] .. q_starts[b + 1] - 1, and the starts do not fall (if
    they do, rows of sequences may be left out); kv_lens: int32 [B], its keys
    in the cache; block_table: int32 [B, columns], key j lies in page
    block_table[b, j // page_size]. causal: the tokens are the sequence's
    last, and token t of n sees kv_lens[b] - n + t + 1 keys; otherwise each
    sees all. scale: head_dim ** -0.5 if not given. Returns (or fills)
    out [tokens, heads, head_dim], which may be q or share memory with it (q
    is copied then), but not with the cache or the other tensors.

    A row that sees no key is 0. Rows before q_starts[0] and from
    q_starts[B] on are left as they were. A row that sees a key whose page
    number is outside of the pool is NaN, and so are all rows of a sequence
    whose length is negative or more than its table holds. A quantised
    cache's values enter as q's type; for fp16 a value past 65504, which only
    rows of bf16 can have left there, is an infinity. The weights of the keys
    are rounded to q's type for their product with the values, as the result
    is; sums are 32 bits.

    The host sees sizes only: which kernel runs goes by the mean number of new
    tokens, and how it shares the keys by the table's columns. Many steps next
    to a long chunk are sooner done in two calls, and short sequences in a
    table that is not much wider than they are."""

    return (_EXT or _ext()).attention(cache._pools, q, q_starts, kv_lens,
                                      block_table, scale, causal, out)
