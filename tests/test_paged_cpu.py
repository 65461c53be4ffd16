"""What the paged operators refuse, and their plan: no GPU needed."""
import pytest
import torch

from tensor_fusion_amd.ops import paged

pytestmark = pytest.mark.usefixtures("native_built")


def cache(dtype=torch.bfloat16, quantized=False, D=64, page=16, Hk=2, pages=5):
    return paged.make_cache(pages, page, Hk, D, dtype, quantized,
                            device="cpu")


def rows(n=3, heads=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(n, heads, D, dtype=dtype)


SLOTS = torch.arange(3)


def refuse(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_cache_refusals():
    z = torch.zeros
    refuse("of one shape", paged.PagedKVCache, z(2, 2, 16, 64),
           z(2, 2, 16, 32))
    refuse("of one shape", paged.PagedKVCache, z(2, 16, 64), z(2, 16, 64))
    refuse("head_dim", cache, D=96)
    for page in (8, 24, 2048):
        refuse("page_size", cache, page=page)
    refuse("no pool", cache, pages=0)
    refuse("no pool", cache, Hk=0)
    refuse("bfloat16, float16 or", cache, dtype=torch.float32)
    x = z(2, 2, 16, 64, dtype=torch.bfloat16)
    refuse("bfloat16, float16 or", paged.PagedKVCache, x, x.half())
    s = z(2, 2, 16, dtype=torch.uint8)
    refuse("has no scales", paged.PagedKVCache, x, x, s, s)
    c = z(2, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    refuse("uint8 scale", paged.PagedKVCache, c, c)
    refuse("uint8 scale", paged.PagedKVCache, c, c, s, s.float())
    refuse("uint8 scale", paged.PagedKVCache, c, c, s[:1], s)
    wide = z(2, 2, 16, 128, dtype=torch.bfloat16)
    refuse("without gaps", paged.PagedKVCache, wide[..., :64],
           wide[..., 64:])
    flat = z(2 * 2 * 16 * 64 + 8, dtype=torch.bfloat16)
    moved = flat[4:4 + 2 * 2 * 16 * 64].view(2, 2, 16, 64)
    refuse("multiples of 16", paged.PagedKVCache, moved, moved)
    huge = z(1, dtype=torch.bfloat16).expand(2 ** 27, 1, 16, 64)
    refuse("less than", paged.PagedKVCache, huge, huge)


def test_quantized_cache_starts_at_zero():
    c = cache(quantized=True)
    assert c.quantized and c.k.float().abs().sum() == 0
    assert (c.k_scale == 127).all()
    assert (c.pages, c.kv_heads, c.page_size, c.head_dim) == (5, 2, 16, 64)
    with pytest.raises(AttributeError):
        c.k = c.v  # the operators hold the tensors that it was made with


def test_write_refusals():
    c = cache()
    refuse("k and v are", paged.kv_write, c, rows(), rows(2), SLOTS)
    refuse("k and v are", paged.kv_write, c, rows(heads=3), rows(heads=3),
           SLOTS)
    refuse("k and v are", paged.kv_write, c, rows(D=32), rows(D=32), SLOTS)
    refuse("rows are", paged.kv_write, c, rows(dtype=torch.float32),
           rows(dtype=torch.float32), SLOTS)
    refuse("rows for a", paged.kv_write, c, rows(dtype=torch.float16),
           rows(dtype=torch.float16), SLOTS)
    refuse("of one type", paged.kv_write, cache(quantized=True), rows(),
           rows(dtype=torch.float16), SLOTS)
    refuse("slots is int64", paged.kv_write, c, rows(), rows(), SLOTS.int())
    refuse("slots is int64", paged.kv_write, c, rows(), rows(), SLOTS[:2])
    refuse("slots is int64", paged.kv_write, c, rows(), rows(),
           torch.arange(6)[::2])
    refuse("run on a GPU", paged.kv_write, c, rows(), rows(), SLOTS)
    with pytest.raises(RuntimeError, match="no backward"):
        paged.kv_write(c, rows().requires_grad_(), rows(), SLOTS)


def test_rope_write_refusals():
    c = cache()
    q, k = torch.zeros(3, 256, dtype=torch.bfloat16), rows().flatten(1)
    t = torch.zeros(8, 32)

    def call(q=q, k=k, v=k, cos=t, sin=t, pos=SLOTS, slots=SLOTS, heads=4):
        return paged.rope_kv_write(c, q, k, v, cos, sin, pos, slots, heads)

    refuse("q_in is", call, heads=3)
    refuse("q_in is", call, heads=0)
    refuse("k_in and v_in", call, k=k[:2])
    refuse("k_in and v_in", call, v=k[:, :64])
    refuse("of one type", call, k=k.half())
    refuse("cos and sin", call, cos=t.double())
    refuse("cos and sin", call, sin=t[:4])
    refuse("cos and sin", call, cos=torch.zeros(8, 64)[:, ::2])
    refuse("cos and sin", call, cos=t[:0], sin=t[:0])
    refuse("pos is int64", call, pos=SLOTS.int())
    refuse("slots is int64", call, slots=SLOTS[:2])
    refuse("run on a GPU", call)


def test_read_refusals():
    refuse("not read as", paged.kv_read, cache(), SLOTS, torch.float16)
    refuse("not read as", paged.kv_read, cache(quantized=True), SLOTS,
           torch.float32)
    refuse("slots is int64", paged.kv_read, cache(), SLOTS.int())
    refuse("slots is int64", paged.kv_read, cache(), SLOTS.view(1, 3))
    refuse("run on a GPU", paged.kv_read, cache(), SLOTS)


def test_attention_refusals():
    c = cache()
    i32 = torch.int32
    starts = torch.tensor([0, 1, 3], dtype=i32)
    lens = torch.tensor([5, 9], dtype=i32)
    table = torch.zeros(2, 3, dtype=i32)

    def call(q=rows(heads=4), cache=c, starts=starts, lens=lens, table=table,
             **kw):
        return paged.paged_attention(q, cache, starts, lens, table, **kw)

    refuse("tokens, heads", call, q=rows()[0])
    refuse("for a cache of", call, q=rows(heads=3))
    refuse("for a cache of", call, q=rows(heads=4, D=32))
    refuse("for a cache of", call, q=rows(heads=0))
    refuse("rows are", call, q=rows(heads=4).float())
    refuse("rows for a", call, q=rows(heads=4).half())
    refuse("kv_lens is", call, table=table[0])
    refuse("sequences of the table", call, lens=lens[:1])
    refuse("sequences of the table", call, starts=starts[:2])
    refuse("are int32", call, starts=starts.long())
    refuse("are int32", call, table=table.long())
    refuse("no gaps", call, table=torch.zeros(2, 6, dtype=i32)[:, ::2])
    refuse("no gaps", call, lens=torch.zeros(4, dtype=i32)[::2])
    refuse("at most 2", call,
           table=torch.zeros(2 ** 26 + 1, dtype=i32).expand(2, -1))
    refuse("finite", call, scale=float("nan"))
    refuse("run on a GPU", call)
    with pytest.raises(RuntimeError, match="no backward"):
        call(q=rows(heads=4).requires_grad_())
    with torch.no_grad():
        refuse("run on a GPU", call, q=rows(heads=4).requires_grad_())


@pytest.mark.parametrize("T,B,G", [(1, 1, 1), (64, 64, 8), (8192, 1, 4),
                                   (613, 9, 1), (60, 12, 4), (33, 1, 1),
                                   (5000, 300, 7), (2, 2, 128)])
def test_plan_covers_every_row(T, B, G):
    """Whatever the lengths, each sequence's tiles fit the grid."""

    workers, join, splits = paged._ext().plan(T, B, G, 8, 128, 4096)
    assert 1 <= splits <= 16
    assert workers == 0 or (join and 8 <= workers <= 512
                            and workers % 8 == 0)
    BM = 16 if workers else 128
    tiles = T * G // BM + B
    gen = torch.Generator().manual_seed(T)
    for _ in range(20):
        cuts = torch.randint(0, T + 1, (B - 1,), generator=gen).sort()[0]
        starts = [0, *cuts.tolist(), T]
        end = 0
        for i in range(B):
            first = starts[i] * G // BM + i
            assert first >= end
            end = first + -(-(starts[i + 1] - starts[i]) * G // BM)
        assert end <= tiles


def test_plan_refuses_what_is_no_size():
    plan = paged._ext().plan
    assert plan(1, 1, 1, 1, 128, 0)
    for i in range(6):
        sizes = [4, 2, 2, 2, 64, 100]
        for bad in (-1, 2 ** 40) + ((0,) if i < 5 else ()):
            sizes[i] = bad
            with pytest.raises(ValueError, match="no plan"):
                plan(*sizes)
    with pytest.raises(ValueError, match="whole number"):
        plan(1, 1, "x", 1, 1, 1)
