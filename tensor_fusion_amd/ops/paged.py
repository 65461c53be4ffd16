"""A paged KV cache and what writes, reads and attends over it
(native/ops/paged_cache.hip, native/ops/paged_attention.hip).

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

The operators serve: they have no backward pass and refuse inputs that ask
for one. They run on the current stream of the tensors' device and never
wait for the GPU; lengths, slots and tables stay on the device, so that a
captured graph is replayed while they change. Shapes, types and devices are
checked here (ValueError); what lies on the device is checked by the kernels,
which read and write nothing outside of the tensors: see each operator for
what they answer instead.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import fused

HEAD_DIMS = (32, 64, 128)
_WIDE = (torch.bfloat16, torch.float16)
_FP8 = torch.float8_e4m3fn


class PagedKVCache:
    """One layer's pages: k and v [pages, kv_heads, page_size, head_dim],
    without gaps, bf16, fp16 or float8_e4m3fn; for the last k_scale and
    v_scale, uint8 [pages, kv_heads, page_size]. page_size is a power of two
    from 16 to 1024, head_dim 32, 64 or 128."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads",
                 "page_size", "page_log2", "head_dim", "dtype", "quantized",
                 "device", "_ptrs")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(
                "k and v pools are [pages, kv_heads, page_size, head_dim], "
                f"of one shape: got {tuple(k.shape)} and {tuple(v.shape)}")
        pages, kv_heads, page_size, head_dim = k.shape
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim is one of {HEAD_DIMS}: {head_dim}")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError("page_size is a power of two from 16 to 1024: "
                             f"{page_size}")
        if pages < 1 or not 1 <= kv_heads <= 4096:
            raise ValueError(f"no pool of {pages} pages, {kv_heads} heads")
        if pages * page_size >= 2 ** 31:
            raise ValueError(f"{pages} pages of {page_size} tokens: a pool "
                             "holds less than 2**31 tokens")
        dtype = k.dtype
        quantized = dtype is _FP8
        if (not quantized and dtype not in _WIDE) or v.dtype is not dtype:
            raise ValueError("pools are both bfloat16, float16 or "
                             f"float8_e4m3fn: got {dtype}, {v.dtype}")
        parts = [k, v]
        if quantized:
            for s in (k_scale, v_scale):
                if (s is None or s.dtype is not torch.uint8
                        or s.shape != k.shape[:3]):
                    raise ValueError("a float8_e4m3fn pool has a uint8 scale "
                                     f"of shape {tuple(k.shape[:3])}")
            parts += [k_scale, v_scale]
        elif k_scale is not None or v_scale is not None:
            raise ValueError(f"a {dtype} pool has no scales")
        ptrs = []
        for x in parts:
            p = x.data_ptr()
            if not x.is_contiguous() or p % 16 or x.device != k.device:
                raise ValueError("pools and scales lie on one device, "
                                 "without gaps, at multiples of 16 bytes")
            ptrs.append(p)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads = pages, kv_heads
        self.page_size, self.page_log2 = page_size, page_size.bit_length() - 1
        self.head_dim, self.dtype, self.quantized = head_dim, dtype, quantized
        self.device = k.device
        self._ptrs = ptrs if quantized else ptrs + [None, None]


def make_cache(pages: int, page_size: int, kv_heads: int, head_dim: int,
               dtype=torch.bfloat16, quantized: bool = False,
               device="cuda") -> PagedKVCache:
    """A cleared cache. dtype is that of the rows; a quantised one takes
    rows of either 16-bit type and holds 8 bits and a scale."""

    shape = (pages, kv_heads, page_size, head_dim)
    if quantized:
        # codes 0, scale 1
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device)
                .view(_FP8) for _ in range(2))
        ks, vs = (torch.full(shape[:3], 127, dtype=torch.uint8,
                             device=device) for _ in range(2))
        return PagedKVCache(k, v, ks, vs)
    return PagedKVCache(torch.zeros(shape, dtype=dtype, device=device),
                        torch.zeros(shape, dtype=dtype, device=device))


_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_ENTRIES = {
    "tf_paged_write": [_P] * 3 + [_L] * 5 + [_P] * 3 + [_I] + [_P] * 6
                      + [_L] + [_I] * 6 + [_P],
    "tf_paged_read": [_P] * 4 + [_L, _I] + [_P] * 3 + [_I] * 4 + [_P],
    "tf_paged_attention": [_P] * 10 + [_L] * 3 + [_I] * 8
                          + [ctypes.c_float] + [_I] * 5 + [_P],
}
_READY = {}


def _entry(name: str):
    fn = _READY.get(name)
    if fn is None:
        fn = getattr(fused.lib(), name)
        fn.restype, fn.argtypes = ctypes.c_int, _ENTRIES[name]
        _READY[name] = fn
    return fn


def _launch(name: str, device, *args):
    """The entry on the device's own current stream, whichever device is
    current."""

    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        rc = _entry(name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = _entry(name)(*args, stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed: {rc}")


def _on_gpu(device, *tensors):
    for x in tensors:
        if x.device != device:
            raise ValueError(f"tensors on {x.device} and a cache on {device}")
    if device.type != "cuda":
        raise ValueError(f"the paged operators run on a GPU: got {device}")


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for x in tensors:
            if x.requires_grad:
                raise RuntimeError(
                    "the paged operators have no backward pass: call them "
                    "under torch.no_grad()")


def _rows(x):
    """x, or a copy of it where 16-byte loads do not fit its layout."""

    if (x.stride(-1) != 1 or x.data_ptr() % 16
            or any(s % 8 for s in x.stride()[:-1])):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _check_rows(cache, *rows):
    dtype = rows[0].dtype
    if dtype not in _WIDE:
        raise ValueError(f"rows are bfloat16 or float16: got {dtype}")
    if not cache.quantized and dtype is not cache.dtype:
        raise ValueError(f"{dtype} rows for a {cache.dtype} cache")
    for x in rows:
        if x.dtype is not dtype:
            raise ValueError(f"rows of one type: got {dtype}, {x.dtype}")


def _check_index(name, x, n):
    if x.dtype is not torch.int64 or x.shape != (n,) or not x.is_contiguous():
        raise ValueError(f"{name} is int64 [{n}] without gaps: got {x.dtype} "
                         f"{tuple(x.shape)}")


def kv_write(cache: PagedKVCache, k, v, slots) -> None:
    """pages[slots] <- k, v; k and v are [n, kv_heads, head_dim], rows and
    heads at any stride, slots int64 [n].

    A quantised cache rounds each row to e4m3 under its own scale; a row
    that holds an infinity or NaN becomes NaN throughout, and fp16 values
    are held to +-61440, the last e4m3 step that fp16 has. Rows whose slot
    is negative (padding) or past the pool are not written. Slots that are
    written have to differ: of two rows for one slot, parts of either may
    stay."""

    n = k.shape[0]
    shape = (n, cache.kv_heads, cache.head_dim)
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"k and v are {shape}: got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    _check_rows(cache, k, v)
    _check_index("slots", slots, n)
    _no_grad(k, v)
    _on_gpu(cache.device, k, v, slots)
    if n == 0:
        return
    k, v = _rows(k), _rows(v)
    _launch("tf_paged_write", cache.device, None, k.data_ptr(), v.data_ptr(),
            0, k.stride(0), k.stride(1), v.stride(0), v.stride(1), None,
            None, None, 0, slots.data_ptr(), None, *cache._ptrs, cache.pages,
            cache.page_log2, n, 0, cache.kv_heads, cache.head_dim,
            k.dtype is torch.float16)


def rope_kv_write(cache: PagedKVCache, q_in, k_in, v_in, cos, sin, pos,
                  slots, heads: int):
    """One launch for a layer: q rotated to a fresh [n, heads, head_dim],
    k rotated and v copied into the pages (quantised from the 32-bit
    products), as kv_write has it.

    q_in, k_in, v_in: [n, heads * head_dim] and [n, kv_heads * head_dim],
    which may be column slices of one merged product; cos, sin: float32
    [positions, head_dim / 2] for interleaved pairs; pos, slots: int64 [n].
    A row whose position lies outside of the tables becomes NaN."""

    D, Hk = cache.head_dim, cache.kv_heads
    n = q_in.shape[0]
    if heads < 1 or q_in.shape != (n, heads * D):
        raise ValueError(f"q_in is [n, {heads} * {D}]: got "
                         f"{tuple(q_in.shape)}")
    if k_in.shape != (n, Hk * D) or v_in.shape != (n, Hk * D):
        raise ValueError(f"k_in and v_in are {(n, Hk * D)}: got "
                         f"{tuple(k_in.shape)} and {tuple(v_in.shape)}")
    _check_rows(cache, q_in, k_in, v_in)
    for x in (cos, sin):
        if (x.dtype is not torch.float32 or x.dim() != 2 or x.shape[0] < 1
                or x.shape != cos.shape or x.shape[1] != D // 2
                or not x.is_contiguous() or x.data_ptr() % 16):
            raise ValueError("cos and sin are float32 [positions, "
                             f"{D // 2}] without gaps")
    _check_index("pos", pos, n)
    _check_index("slots", slots, n)
    if heads + 2 * Hk > 65535 or cos.shape[0] >= 2 ** 31:
        raise ValueError(f"too many heads ({heads}) or positions")
    _no_grad(q_in, k_in, v_in)
    _on_gpu(cache.device, q_in, k_in, v_in, cos, sin, pos, slots)
    q = torch.empty(n, heads, D, device=q_in.device, dtype=q_in.dtype)
    if n == 0:
        return q
    q_in, k_in, v_in = _rows(q_in), _rows(k_in), _rows(v_in)
    _launch("tf_paged_write", cache.device, q_in.data_ptr(), k_in.data_ptr(),
            v_in.data_ptr(), q_in.stride(0), k_in.stride(0), D,
            v_in.stride(0), D, cos.data_ptr(), sin.data_ptr(),
            pos.data_ptr(), cos.shape[0], slots.data_ptr(), q.data_ptr(),
            *cache._ptrs, cache.pages, cache.page_log2, n, heads, Hk, D,
            q_in.dtype is torch.float16)
    return q


def kv_read(cache: PagedKVCache, slots, dtype=None):
    """k, v [n, kv_heads, head_dim] of the slots (int64 [n], any order, any
    of them more than once), dequantised to `dtype` (bfloat16 if not given)
    where the cache is quantised. A negative slot reads 0, one past the
    pool NaN."""

    if dtype is None:
        dtype = torch.bfloat16 if cache.quantized else cache.dtype
    if dtype not in _WIDE or not (cache.quantized or dtype is cache.dtype):
        raise ValueError(f"a {cache.dtype} cache is not read as {dtype}")
    if slots.dim() != 1:
        raise ValueError(f"slots is int64 [n]: got {tuple(slots.shape)}")
    n = slots.shape[0]
    _check_index("slots", slots, n)
    _on_gpu(cache.device, slots)
    k, v = (torch.empty(n, cache.kv_heads, cache.head_dim, dtype=dtype,
                        device=cache.device) for _ in range(2))
    if n:
        kp, vp, ks, vs = cache._ptrs
        _launch("tf_paged_read", cache.device, kp, vp, ks, vs, cache.pages,
                cache.page_log2, slots.data_ptr(), k.data_ptr(),
                v.data_ptr(), n, cache.kv_heads, cache.head_dim,
                dtype is torch.float16)
    return k, v


def _plan(T: int, B: int, G: int, Hk: int, keys: int):
    """(workers, join, splits). What a batch holds lies on the device; this
    goes by its mean, and is right for any batch. Up to 16 rows (new tokens
    * G) a sequence are work for the kernel for few rows, whose `workers`
    share it out among themselves; 0 workers: the kernel for many rows, with
    the keys of each tile of 128 rows in `splits` parts."""

    rows = T * G
    pieces = max(1, -(-keys // 256))  # of keys that are worth a workgroup
    if rows <= 16 * B:
        # two workgroups fit a unit; neighbouring ones share an XCD of eight
        items = Hk * max(B, rows // 16)
        workers = -(-min(512, items * pieces) // 8) * 8
        return workers, int(keys > 384), 1  # 384: never split
    return 0, 0, min(pieces, max(1, 512 // (Hk * max(B, rows // 128))))


def paged_attention(q, cache: PagedKVCache, q_starts, kv_lens, block_table,
                    scale=None, causal: bool = True, out=None):
    """Attention of a packed batch of new tokens over the pages of their
    sequences, the new tokens' own keys (already written) among them.

    q: [tokens, heads, head_dim], tokens and heads at any stride, heads a
    multiple of the cache's; q_starts: int32 [B + 1], sequence b's tokens
    are q_starts[b] .. q_starts[b + 1] - 1; kv_lens: int32 [B], its keys in
    the cache; block_table: int32 [B, columns], key j lies in page
    block_table[b, j // page_size]. causal: the tokens are the sequence's
    last, and token t of n sees kv_lens[b] - n + t + 1 keys; otherwise each
    sees all. scale: head_dim ** -0.5 if not given. Returns (or fills)
    out [tokens, heads, head_dim].

    A row that sees no key is 0. Rows before q_starts[0] and from
    q_starts[B] on are left as they were. A row that sees a key whose page
    number is outside of the pool is NaN, and so are all rows of a sequence
    whose length is negative or more than its table holds. A quantised
    cache's values enter as q's type; for fp16 a value past 65504, which only
    rows of bf16 can have left there, is an infinity."""

    if q.dim() != 3:
        raise ValueError(f"q is [tokens, heads, head_dim]: {tuple(q.shape)}")
    T, Hq, D = q.shape
    Hk = cache.kv_heads
    if D != cache.head_dim or Hq < 1 or Hq % Hk:
        raise ValueError(f"q {tuple(q.shape)} for a cache of {Hk} heads of "
                         f"{cache.head_dim}")
    _check_rows(cache, q)
    if kv_lens.dim() != 1 or block_table.dim() != 2:
        raise ValueError("kv_lens is [B], block_table [B, columns]")
    B, cols = block_table.shape
    if kv_lens.shape[0] != B or q_starts.shape != (B + 1,):
        raise ValueError(f"for {B} sequences of the table: kv_lens "
                         f"{tuple(kv_lens.shape)}, q_starts "
                         f"{tuple(q_starts.shape)}")
    if not (q_starts.dtype is kv_lens.dtype is block_table.dtype
            is torch.int32):
        raise ValueError("q_starts, kv_lens and block_table are int32")
    if not (q_starts.is_contiguous() and kv_lens.is_contiguous()) or (
            cols > 1 and block_table.stride(1) != 1):
        raise ValueError("q_starts, kv_lens and the table's rows have no "
                         "gaps")
    if cols * cache.page_size > 2 ** 30:
        raise ValueError(f"{cols} pages of {cache.page_size} tokens: a "
                         "sequence has at most 2**30")
    G = Hq // Hk
    if (T * G // 16 + B) * Hk >= 2 ** 31 or T * G + 128 * B >= 2 ** 31:
        raise ValueError(f"{T} tokens of {Hq} heads: too many for a launch")
    scale = D ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale is a finite number: got {scale}")
    _no_grad(q)
    _on_gpu(cache.device, q, q_starts, kv_lens, block_table)
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    elif (out.shape != q.shape or out.dtype is not q.dtype
          or not out.is_contiguous() or out.device != q.device
          or out.data_ptr() % 16):
        raise ValueError("out has q's shape, type and device, without gaps")
    if T == 0 or B == 0:
        return out
    q = _rows(q)
    workers, join, splits = _plan(T, B, G, Hk, cols * cache.page_size)
    parts = None
    if join or splits > 1:
        # its own for every call: two captured graphs never share it
        rows = 2 * workers * 16 if workers else \
            (T * G // 128 + B) * Hk * splits * 128
        parts = torch.empty(rows * (D + 2), dtype=torch.float32,
                            device=q.device)
    kp, vp, ks, vs = cache._ptrs
    _launch("tf_paged_attention", cache.device, q.data_ptr(), kp, vp, ks, vs,
            q_starts.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(),
            out.data_ptr(), None if parts is None else parts.data_ptr(),
            q.stride(0), q.stride(1), block_table.stride(0), cols, T, B, Hq,
            Hk, cache.pages, cache.page_log2, D, scale, causal,
            q.dtype is torch.float16, workers, join, splits)
    return out
