"""The paged KV-cache operators against their definitions in 64 bits."""
import pytest
import torch

from tensor_fusion_amd.ops import paged

from paged_oracle import Batch, cache_values, check, e4m3

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
WIDE = pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
KEPT = pytest.mark.parametrize("quantized", [False, True],
                               ids=["wide", "e4m3"])
DIMS = pytest.mark.parametrize("D", [32, 64, 128])


# ---- writing and reading ---------------------------------------------------


def edge_rows(n, Hk, D, dtype, seed):
    """Rows whose maxima lie on and next to the scales' borders, tiny, huge,
    empty and broken ones among them."""

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, Hk, D, generator=g)
    x *= torch.exp2(torch.randint(-12, 12, (n, Hk, 1), generator=g).float())
    flat = x.view(-1, D)
    flat[0] = 0
    tops = [448.0, 450.0, 1.75, 1.7578125, 3.0, 65504.0, 63488.0, 2.0 ** -14,
            2.0 ** -24, float("inf"), float("-inf"), float("nan"), 7.0,
            57344.0, 1e-7]
    for i, top in enumerate(tops):
        if i + 1 < len(flat):
            flat[i + 1] = flat[i + 1].clamp(-1, 1) * min(top, 6e4) / 2 \
                if top == top and abs(top) < 1e30 else flat[i + 1]
            flat[i + 1, (7 * i) % D] = top
    return x.to(dtype)


@WIDE
@KEPT
@DIMS
@pytest.mark.parametrize("n,Hk,page", [(1, 1, 16), (17, 3, 32), (40, 8, 16),
                                       (259, 2, 64)])
def test_write_then_read(n, Hk, page, D, dtype, quantized):
    """Bit for bit, at slots in any order, the others left as they were."""

    cache = paged.make_cache(n // page + 3, page, Hk, D, dtype, quantized)
    before = cache_values(cache)
    k, v = (edge_rows(n, Hk, D, dtype, s) for s in (1, 2))
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(cache.pages * page, generator=g)[:n]
    slots[n // 2] = -1
    if n > 4:
        slots[3] = cache.pages * page  # past the pool
    # rows as columns of one wider product
    wide = torch.zeros(n, 2 * Hk * D + 8, dtype=dtype)
    wide[:, :Hk * D], wide[:, Hk * D:2 * Hk * D] = k.flatten(1), v.flatten(1)
    wide = wide.cuda()
    kd = wide[:, :Hk * D].unflatten(1, (Hk, D))
    vd = wide[:, Hk * D:2 * Hk * D].unflatten(1, (Hk, D))
    paged.kv_write(cache, kd, vd, slots.cuda())
    got = paged.kv_read(cache, slots.cuda(), dtype)
    kept = (slots >= 0) & (slots < cache.pages * page)
    pools = cache_values(cache)
    for x, r, pool, old in zip((k, v), got, pools, before):
        want = e4m3(x, dtype is FP16)[0] if quantized else x.double()
        r = r.cpu().double()
        assert torch.equal(r[kept].nan_to_num(9e9), want[kept].nan_to_num(9e9))
        assert (r[slots < 0] == 0).all()
        assert torch.isnan(r[slots >= cache.pages * page]).all()
        rows = pool.transpose(1, 2).flatten(0, 1)  # [slots, Hk, D]
        assert torch.equal(rows[slots[kept]].nan_to_num(9e9),
                           want[kept].nan_to_num(9e9))
        rest = torch.ones(len(rows), dtype=torch.bool)
        rest[slots[kept]] = False
        assert torch.equal(rows[rest],
                           old.transpose(1, 2).flatten(0, 1)[rest])
    if quantized:
        byte = e4m3(k)[1]
        rows = cache.k_scale.cpu().transpose(1, 2).flatten(0, 1)
        assert torch.equal(rows[slots[kept]], byte[kept])


def test_read_the_same_slot_twice_and_none():
    cache = paged.make_cache(2, 16, 2, 64, quantized=True)
    k = torch.randn(4, 2, 64, device="cuda", dtype=BF16)
    paged.kv_write(cache, k, -k, torch.tensor([5, 6, 20, 31], device="cuda"))
    a, b = paged.kv_read(cache, torch.tensor([20, 5, 20], device="cuda"))
    assert torch.equal(a[0], a[2]) and torch.equal(a, -b)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert paged.kv_read(cache, none)[0].shape == (0, 2, 64)
    paged.kv_write(cache, k[:0], k[:0], none)


def test_read_scales_at_the_ends():
    """255 stands for no value, 0 for 2^-127; fp16 has no value past 65504,
    which rows of bf16 may have left in a quantised cache."""

    cache = paged.make_cache(1, 16, 1, 32, quantized=True)
    slots = torch.arange(3, device="cuda")
    k = torch.full((3, 1, 32), 448.0, device="cuda", dtype=BF16)
    paged.kv_write(cache, k * 1024, k, slots)
    assert (cache.k_scale[0, 0, :3] == 137).all()
    cache.k_scale[0, 0, 1], cache.k_scale[0, 0, 2] = 255, 0
    got = paged.kv_read(cache, slots)[0].float()
    assert (got[0] == 448 * 1024).all() and torch.isnan(got[1]).all()
    assert (got[2] == 448 * 2.0 ** -127).all()
    half = paged.kv_read(cache, slots, FP16)[0]
    assert torch.isinf(half[0]).all() and (half[2] == 0).all()


@pytest.mark.parametrize("n", [1, 40], ids=["few", "many"])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@WIDE
def test_attention_scale_without_a_value(which, n, dtype):
    """A key or value whose scale byte is 255 makes the rows that see it
    NaN, and no other."""

    b = Batch([(n, 70), (n, 50)], 4, 2, 64, 16, dtype, True, seed=20)
    at = int(b.table[0, 69 // 16])
    getattr(b.cache, which)[at, 1, 69 % 16] = 255
    got = b.run()
    assert torch.isnan(got[n - 1, 2:].float()).all()
    want, tol, mine = Batch([(n, 70), (n, 50)], 4, 2, 64, 16, dtype, True,
                            seed=20).want()
    rest = torch.ones_like(want, dtype=torch.bool)
    rest[n - 1, 2:] = False
    off = (got.cpu().double() - want).abs() - tol
    assert off[rest].max() <= 0


@pytest.mark.parametrize("layout", ["heads first", "odd start", "odd row"])
def test_write_any_layout(layout):
    """Strides and addresses that 16-byte loads do not fit."""

    n, Hk, D = 9, 2, 64
    k = torch.randn(n, Hk, D, device="cuda", dtype=BF16)
    if layout == "heads first":
        x = k.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "odd start":
        flat = torch.empty(n * Hk * D + 3, device="cuda", dtype=BF16)
        x = flat[3:].view(n, Hk, D)
        x.copy_(k)
    else:
        x = torch.empty(n, Hk * D + 5, device="cuda", dtype=BF16)[
            :, :Hk * D].unflatten(1, (Hk, D))
        x.copy_(k)
    cache = paged.make_cache(1, 16, Hk, D)
    slots = torch.arange(n, device="cuda")
    paged.kv_write(cache, x, x, slots)
    a, b = paged.kv_read(cache, slots)
    assert torch.equal(a, k) and torch.equal(b, k)


@WIDE
@KEPT
@DIMS
@pytest.mark.parametrize("n,heads,Hk", [(1, 4, 2), (35, 6, 3), (130, 16, 2)])
def test_rope_write(n, heads, Hk, D, dtype, quantized):
    page = 16
    cache = paged.make_cache(n // page + 2, page, Hk, D, dtype, quantized)
    g = torch.Generator().manual_seed(n)
    qkv = torch.randn(n, (heads + 2 * Hk) * D, generator=g).to(dtype)
    angle = torch.rand(300, D // 2, generator=g) * 6.3
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, 300, (n,), generator=g)
    if n > 1:
        pos[1] = 300  # outside of the tables
    slots = torch.randperm(cache.pages * page, generator=g)[:n]
    d = qkv.cuda()
    parts = d.split([heads * D, Hk * D, Hk * D], 1)
    q = paged.rope_kv_write(cache, *parts, cos.cuda(), sin.cuda(),
                            pos.cuda(), slots.cuda(), heads)
    known = pos < 300
    c, s = (x.double()[pos.clamp(max=299)].unsqueeze(1) for x in (cos, sin))

    def turned(x):
        x = x.double().unflatten(1, (-1, D))
        a, b = x[..., ::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), \
            torch.stack([a.abs() * c.abs() + b.abs() * s.abs()] * 2,
                        -1).flatten(-2)

    u = 2.0 ** -8 if dtype is BF16 else 2.0 ** -11
    parts = qkv.split([heads * D, Hk * D, Hk * D], 1)
    want, mag = turned(parts[0])
    # one rounding of a 32-bit value that is off by two of its own
    tol = u * 1.01 * want.abs() + 2.0 ** -22 * mag + 2.0 ** -25
    assert (((q.cpu().double() - want).abs() - tol)[known] <= 0).all()
    assert torch.isnan(q.cpu()[~known]).all()
    k, v = paged.kv_read(cache, slots.cuda(), dtype)
    want, mag = turned(parts[1])
    k = k.cpu().double()
    assert torch.isnan(k[~known]).all()
    if quantized:
        # an e4m3 step is 2^-3 of the binade: off by half of one, 2^-4 of
        # the value, or by half of the smallest, 2^-10 of the scale
        scale = torch.exp2(torch.ceil(torch.log2(
            want.abs().amax(-1, keepdim=True) * (1 + 2.0 ** -20) / 448)))
        tol = 2.0 ** -4 * 1.01 * want.abs() + 2.0 ** -10 * scale \
            + 2.0 ** -22 * mag
        wv = e4m3(parts[2].unflatten(1, (Hk, D)), dtype is FP16)[0]
    else:
        tol = u * 1.01 * want.abs() + 2.0 ** -22 * mag + 2.0 ** -25
        wv = parts[2].unflatten(1, (Hk, D)).double()
    assert (((k - want).abs() - tol)[known] <= 0).all()
    assert torch.equal(v.cpu().double(), wv)


# ---- attention --------------------------------------------------------------

# (new tokens, keys) of each sequence
STEP = [(1, 1), (1, 16), (1, 17), (1, 300), (1, 31), (1, 1000), (1, 64)]
FEW = [(3, 3), (5, 90), (2, 33), (7, 513), (1, 5), (4, 260)]
MANY = [(129, 129), (65, 700), (200, 260), (128, 1025)]
MIXED = [(1, 77), (150, 150), (2, 400), (1, 1), (70, 333), (0, 50), (33, 64)]
EMPTY = [(0, 0), (1, 0), (5, 2), (0, 9), (3, 3), (1, 12)]
EMPTY_MANY = [(200, 60), (0, 0), (130, 0), (140, 140)]
SHAPES = pytest.mark.parametrize("seqs", [
    STEP, FEW, MANY, MIXED, EMPTY, EMPTY_MANY, [(1, 1)], [(1, 4097)],
    [(40, 40)], [(300, 2000)]], ids=[
    "step", "few", "many", "mixed", "empty", "empty_many", "one", "split",
    "prompt", "chunk"])


@WIDE
@KEPT
@DIMS
@SHAPES
def test_attention(seqs, D, quantized, dtype):
    b = Batch(seqs, 8, 2, D, 16, dtype, quantized, seed=D)
    check(b.run(), *b.want())


@pytest.mark.parametrize("heads,Hk", [(1, 1), (3, 3), (8, 8), (7, 1),
                                      (15, 3), (40, 1), (64, 8), (20, 10)])
@pytest.mark.parametrize("seqs", [STEP, MIXED, [(1, 2000)], [(60, 200)]],
                         ids=["step", "mixed", "split", "chunk"])
def test_attention_heads(seqs, heads, Hk):
    b = Batch(seqs, heads, Hk, 64, 32, BF16, heads % 2 == 0, seed=heads)
    check(b.run(), *b.want())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("seqs", [STEP, MIXED, [(140, 1500)]],
                         ids=["step", "mixed", "chunk"])
@KEPT
def test_attention_pages(seqs, page, quantized):
    b = Batch(seqs, 8, 4, 128, page, BF16, quantized, seed=page)
    check(b.run(), *b.want())


@SHAPES
@WIDE
def test_attention_not_causal(seqs, dtype):
    b = Batch(seqs, 6, 2, 64, 16, dtype, False, seed=4)
    check(b.run(causal=False), *b.want(causal=False))


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-4])
def test_attention_scale(scale):
    b = Batch(MIXED, 4, 2, 64, 16, BF16, False, seed=6)
    check(b.run(scale=scale), *b.want(scale=scale))


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-4])
@pytest.mark.parametrize("seqs", [STEP, [(1, 9000)], [(2, 9000)]],
                         ids=["step", "shared", "split"])
@KEPT
def test_attention_scale_of_steps(seqs, scale, quantized):
    heads = 16 if seqs == STEP else 8 * seqs[0][0] ** 3
    b = Batch(seqs, heads, 4, 128, 64, FP16, quantized, seed=16)
    check(b.run(scale=scale), *b.want(scale=scale))


@pytest.mark.parametrize("seqs", [[(1, 700), (1, 90)], [(3, 400), (0, 8)],
                                  [(1, 3000)] * 2], ids=str)
@pytest.mark.parametrize("heads,Hk", [(256, 1), (384, 2), (130, 1)])
def test_attention_more_heads_than_a_tile_has_rows(seqs, heads, Hk):
    b = Batch(seqs, heads, Hk, 64, 16, BF16, heads == 384, seed=17)
    check(b.run(), *b.want())


@pytest.mark.parametrize("seqs", [STEP, MANY], ids=["step", "many"])
def test_attention_far_scores(seqs):
    """Scores of some hundreds: one key takes all, the running maximum
    moves a long way."""

    b = Batch(seqs, 8, 2, 128, 16, BF16, False, seed=8, spread=30.0)
    check(b.run(), *b.want())


def test_attention_rows_outside_of_the_sequences():
    b = Batch(MIXED, 8, 2, 64, 16, BF16, False, seed=9)
    T = len(b.q)
    b.q = torch.cat([b.q, torch.randn(9, 8, 64).to(BF16)])
    first = b.q_starts.clone()
    out = torch.full(b.q.shape, 7.0, dtype=BF16, device="cuda")
    assert b.run(out=out) is out
    want, tol, mine = b.want()
    check(out, want, tol, mine)
    assert (out[T:] == 7).all()
    # rows before the first sequence
    b.q_starts = first + 9
    b.q = torch.cat([b.q[T:], b.q[:T]])
    out = torch.full(b.q.shape, 7.0, dtype=BF16, device="cuda")
    b.run(out=out)
    check(out, *b.want())
    assert (out[:9] == 7).all()


def test_attention_strided_rows():
    b = Batch(MIXED, 8, 2, 64, 16, FP16, False, seed=10)
    want = b.run()
    wide = torch.zeros(len(b.q), 8 * 64 + 128, dtype=FP16, device="cuda")
    view = wide[:, 64:64 + 512].unflatten(1, (8, 64))
    view.copy_(b.q)
    swapped = b.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(b.q.numel() + 1, dtype=FP16, device="cuda")[1:].view(
        b.q.shape)
    odd.copy_(b.q)
    for q in (view, swapped, odd):
        got = paged.paged_attention(q, b.cache, b.q_starts.cuda(),
                                    b.kv_lens.cuda(), b.table.cuda())
        assert torch.equal(got, want)
    # a table whose rows are longer than it
    table = torch.full((len(MIXED), b.table.shape[1] + 7), 10 ** 6,
                       dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    got = paged.paged_attention(b.q.cuda(), b.cache, b.q_starts.cuda(),
                                b.kv_lens.cuda(),
                                table[:, :b.table.shape[1]])
    assert torch.equal(got, want)


@pytest.mark.parametrize("seqs", [[(3, 50), (5, 5)], [(200, 200), (70, 300)],
                                  [(1, 40), (64, 64), (2, 2)]],
                         ids=["few", "many", "mixed"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"),
                                   float("-inf")])
@WIDE
def test_attention_broken_values_in_masked_places(seqs, value, dtype):
    """A key or value that is not finite reaches the rows that see it, and
    no other; a broken query row stays alone."""

    b = Batch(seqs, 4, 2, 64, 16, dtype, False, seed=11)
    for i, (n, kv) in enumerate(seqs):
        for back in (1, n // 2 + 1):
            j = kv - back
            at, off = int(b.table[i, j // 16]), j % 16
            b.cache.v[at, 0, off, 5] = value
            if back > 1:
                b.cache.v[at, 1, off, 63] = value
                b.cache.v[at, 0, off, 6] = -value
    b.q[0, 1] = float("nan")
    check(b.run(), *b.want())
    i, (n, kv) = 0, seqs[0]
    at, off = int(b.table[i, (kv - 1) // 16]), (kv - 1) % 16
    b.cache.k[at, 1, off, 3] = float("nan")
    got = b.run()
    want, tol, mine = b.want()
    last = int(b.q_starts[1]) - 1
    assert torch.isnan(got[last, 2:].float()).all()
    check(got, want, tol, mine)


@pytest.mark.parametrize("seqs", [[(3, 6000), (2, 900)],
                                  [(60, 4000), (70, 2000)]],
                         ids=["shared", "split"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_broken_values_where_keys_are_split(seqs, value):
    workers, _, splits = paged._ext().plan(
        sum(n for n, _ in seqs), 2, 2, 2, 64, max(k for _, k in seqs))
    assert workers or splits > 1
    test_attention_broken_values_in_masked_places(seqs, value, BF16)


@pytest.mark.parametrize("seqs", [[(1, 60), (2, 50)], [(150, 150), (40, 90)]],
                         ids=["few", "many"])
def test_attention_bad_pages_and_lengths(seqs):
    """A page outside of the pool: the rows that see one of its keys are
    NaN. A length that the table does not hold: the sequence's rows are."""

    for bad in (-1, 10 ** 6, 2 ** 31 - 1):
        b = Batch(seqs, 4, 2, 64, 16, BF16, False, seed=12)
        good, tol, mine = b.want()
        b.table[0, 2] = bad  # keys 32 .. 47
        got = b.run()
        n, kv = seqs[0]
        for t in range(n):
            if kv - n + t + 1 > 32:
                assert torch.isnan(got[t].float()).all()
                mine[t] = False
        check(got, good, tol, mine)
    for length in (-1, b.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        b = Batch(seqs, 4, 2, 64, 16, BF16, False, seed=12)
        good, tol, mine = b.want()
        b.kv_lens[0] = length
        got = b.run()
        n = seqs[0][0]
        assert torch.isnan(got[:n].float()).all()
        mine[:n] = False
        check(got, good, tol, mine)


def test_attention_bad_starts_stay_inside():
    """Starts that are not in order or not in the batch write nothing
    outside of it."""

    b = Batch([(2, 20), (3, 30), (4, 40)], 4, 2, 64, 16, BF16, False, seed=3)
    for starts in ([0, -5, 7, 9], [5, 3, 8, 100], [9, 9, 9, 9],
                   [2 ** 31 - 1, 0, -2 ** 31, 4]):
        b.q_starts = torch.tensor(starts, dtype=torch.int32)
        out = torch.zeros(11, 4, 64, dtype=BF16, device="cuda")
        b.run(out=out[:9])
        assert (out[9:] == 0).all()


def test_attention_past_32_bits():
    """Pages that lie behind the first 2**32 bytes and 2**31 values."""

    D, Hk, page = 128, 8, 64
    pages = 2 ** 31 // (Hk * page * D) + 40
    cache = paged.make_cache(pages, page, Hk, D)
    small = Batch([(1, 200), (3, 130), (100, 180)], 16, Hk, D, page, BF16,
                  False, seed=14)
    width = small.table.shape[1]
    far = torch.arange(pages - 3 * width, pages).view(3, width)
    for i in range(3):
        for j in range(width):
            cache.k[far[i, j]] = small.cache.k[int(small.table[i, j])]
            cache.v[far[i, j]] = small.cache.v[int(small.table[i, j])]
    got = paged.paged_attention(
        small.q.cuda(), cache, small.q_starts.cuda(), small.kv_lens.cuda(),
        far.to(torch.int32).cuda())
    assert torch.equal(got, small.run())
    slots = torch.tensor([pages * page - 1, 0], device="cuda")
    k = torch.randn(2, Hk, D, device="cuda", dtype=BF16)
    paged.kv_write(cache, k, -k, slots)
    a, b = paged.kv_read(cache, slots)
    assert torch.equal(a, k) and torch.equal(b, -k)


WHOLE = [(1, 700)] * 30 + [(9, 900), (40, 60), (0, 5), (1, 1)]
SHORT = [(1, 500)] * 30 + [(9, 600), (40, 60), (0, 5), (1, 1)]
SHARED = [(1, 3000), (2, 2500), (1, 0), (8, 1000), (0, 40)]


@pytest.mark.parametrize("seqs,Hk,D,workers", [
    (WHOLE, 2, 64, 108), (WHOLE, 3, 128, 162), (SHORT, 1, 128, 54),
    (WHOLE * 6, 2, 64, 648), (WHOLE * 6, 2, 128, 648), (SHARED, 2, 64, 120),
    (SHARED * 2, 6, 128, 256)],
    ids=["two an item", "two an item, 128", "four an item", "one an item",
         "one an item, 128", "shared", "shared, many"])
@KEPT
@WIDE
def test_attention_few_rows_shared_or_whole(seqs, Hk, D, workers, quantized,
                                            dtype):
    """Each way of giving workgroups their work, sequences of several tiles
    and without tokens among them."""

    b = Batch(seqs, 4 * Hk, Hk, D, 32, dtype, quantized, seed=5)
    plan = paged._ext().plan(len(b.q), len(seqs), 4, Hk, D,
                             b.table.shape[1] * 32)
    assert plan == (workers, seqs[0] == SHARED[0], 1)
    out = torch.full(b.q.shape, 7.0, dtype=dtype, device="cuda")
    b.run(out=out)
    check(out, *b.want())
    assert torch.equal(b.run(), out)


@KEPT
def test_attention_sorted_tiles_in_parts(quantized):
    """More workgroups than places: the longest sequences' tiles first, each
    in parts; sequences of equal length and without tokens among them."""

    seqs = [(80, 1900), (76, 1500), (95, 300), (0, 50), (80, 80)] * 4
    b = Batch(seqs, 8, 8, 64, 32, BF16, quantized, seed=6)
    assert paged._ext().plan(len(b.q), len(seqs), 1, 8, 64,
                             b.table.shape[1] * 32) == (0, 0, 4)
    out = torch.full(b.q.shape, 7.0, dtype=BF16, device="cuda")
    b.run(out=out)
    check(out, *b.want())
    assert torch.equal(b.run(), out)


@pytest.mark.parametrize("most", [3, 200], ids=["few", "many"])
@pytest.mark.parametrize("count", [65, 300, 2500])
def test_attention_many_sequences(count, most):
    """More sequences than a wave has lanes, empty ones among them."""

    g = torch.Generator().manual_seed(count)
    new = torch.randint(0, 4, (count,), generator=g)
    new[5], new[-2] = most, most
    past = torch.randint(0, 60, (count,), generator=g)
    past[7] = 3000
    seqs = [(int(n), int(n + p)) for n, p in zip(new, past)]
    b = Batch(seqs, 4, 2, 32, 64, BF16, False, seed=count, extra_cols=0)
    check(b.run(), *b.want())


@KEPT
def test_attention_a_very_long_sequence(quantized):
    b = Batch([(2, 40000)], 4, 1, 64, 64, BF16, quantized, seed=15)
    check(b.run(), *b.want())


@pytest.mark.parametrize("seqs", [STEP, MIXED, [(2, 5000)], [(130, 4000)]],
                         ids=["step", "mixed", "split", "chunk"])
def test_attention_repeats_bit_for_bit(seqs):
    b = Batch(seqs, 8, 2, 128, 16, BF16, True, seed=16)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)


# ---- streams, graphs, the operators together ----------------------------------


def test_on_another_stream():
    b = Batch([(1, 3000), (2, 700)], 8, 2, 128, 16, BF16, False, seed=17)
    want = b.run()
    q, starts = b.q.cuda(), b.q_starts.cuda()
    lens, table = b.kv_lens.cuda(), b.table.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.paged_attention(q, b.cache, starts, lens, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_steps_replay_as_eager():
    """Two captured graphs, replayed in turn with the program's own work
    between, while lengths, tables and rows change on the device."""

    torch.manual_seed(0)
    Hq, Hk, D, page, B = 8, 2, 64, 16, 3
    table = torch.randperm(60, device="cuda")[:B * 20].view(B, 20).to(
        torch.int32)
    starts = torch.arange(B + 1, device="cuda", dtype=torch.int32)
    angle = torch.rand(400, D // 2, device="cuda")
    cos, sin = angle.cos(), angle.sin()
    caches = [paged.make_cache(60, page, Hk, D, BF16, q8)
              for q8 in (False, True)]
    spare = [paged.make_cache(60, page, Hk, D, BF16, q8)
             for q8 in (False, True)]
    qkv = torch.zeros(B, (Hq + 2 * Hk) * D, device="cuda", dtype=BF16)
    pos = torch.zeros(B, dtype=torch.int64, device="cuda")

    def step(cache):
        slots = table.gather(1, (pos // page)[:, None])[:, 0].long() * page \
            + pos % page
        lens = (pos + 1).to(torch.int32)
        q = paged.rope_kv_write(
            cache, *qkv.split([Hq * D, Hk * D, Hk * D], 1), cos, sin, pos,
            slots, Hq)
        return paged.paged_attention(q, cache, starts, lens, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in caches:
            step(c)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in caches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for i in range(150):
        qkv.copy_(torch.randn_like(qkv))
        pos.copy_(torch.tensor([i, i + 3, 2 * i], device="cuda"))
        for g in graphs:
            g.replay()
        want = [step(c) for c in spare]
        torch.cuda.synchronize()
        for a, w in zip(outs, want):
            assert torch.equal(a, w), i


@pytest.mark.parametrize("n", [1, 40], ids=["few", "many"])
def test_captured_joins_keep_their_own_parts(n):
    """Two captured graphs whose keys are split, replayed in turn with eager
    calls between, while lengths and rows change on the device."""

    torch.manual_seed(1)
    Hq, Hk, D, page, B = 16, 4, 128, 32, 2
    table = torch.randperm(512, device="cuda").view(B, 256).to(torch.int32)
    starts = torch.arange(B + 1, device="cuda", dtype=torch.int32) * n
    lens = torch.full((B,), 5000, device="cuda", dtype=torch.int32)
    caches = []
    for q8 in (False, True):
        c = paged.make_cache(512, page, Hk, D, BF16, q8)
        k, v = torch.randn(2, 512 * page, Hk, D, device="cuda").to(BF16)
        paged.kv_write(c, k, v, torch.arange(512 * page, device="cuda"))
        caches.append(c)
    rows, workers, splits = n * B * Hq // Hk, *paged._ext().plan(
        n * B, B, Hq // Hk, Hk, D, 256 * page)[::2]
    assert workers if rows <= 16 * B else splits > 1
    qs = [torch.randn(n * B, Hq, D, device="cuda").to(BF16) for _ in caches]

    def call(i):
        return paged.paged_attention(qs[i], caches[i], starts, lens, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for a, b in [(8192, 8100), (n, n), (3000, 8000), (8192, 41), (600, 700)]:
        lens.copy_(torch.tensor([a, b]))
        for q in qs:
            q.copy_(torch.randn_like(q))
        for g in graphs:
            g.replay()
        want = [call(0), call(1)]
        graphs[0].replay()
        torch.cuda.synchronize()
        for x, w in zip(outs, want):
            assert torch.equal(x, w), (a, b)


@KEPT
@WIDE
def test_a_prompt_in_chunks_and_steps(dtype, quantized):
    """The operators as they are used: the prompts go in in ragged chunks,
    then token by token; each row against the whole sequence at once."""

    torch.manual_seed(1)
    Hq, Hk, D, page = 8, 2, 64, 16
    lengths = [75, 140]
    cache = paged.make_cache(40, page, Hk, D, dtype, quantized)
    table = torch.randperm(40, device="cuda")[:20].view(2, 10).to(torch.int32)
    angle = torch.rand(160, D // 2, device="cuda") * 6
    cos, sin = angle.cos(), angle.sin()
    rows = [torch.randn(n, (Hq + 2 * Hk) * D, device="cuda").to(dtype)
            for n in lengths]
    done, outs, qs = [0, 0], [[], []], [[], []]
    chunks = [(30, 64), (0, 33), (41, 1)] + [(1, 1)] * 4 + [(0, 38)]
    for chunk in chunks:
        pos, slots, x = [], [], []
        for b, n in enumerate(chunk):
            p = torch.arange(done[b], done[b] + n, device="cuda")
            pos.append(p)
            slots.append(table[b, p // page].long() * page + p % page)
            x.append(rows[b][done[b]:done[b] + n])
            done[b] += n
        x, pos, slots = (torch.cat(t) for t in (x, pos, slots))
        q = paged.rope_kv_write(
            cache, *x.split([Hq * D, Hk * D, Hk * D], 1), cos, sin, pos,
            slots, Hq)
        starts = torch.tensor([0, chunk[0], sum(chunk)], dtype=torch.int32,
                              device="cuda")
        lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        out = paged.paged_attention(q, cache, starts, lens, table)
        for b, (o, r) in enumerate(zip(out.split(list(chunk)),
                                       q.split(list(chunk)))):
            outs[b].append(o)
            qs[b].append(r)
    assert done == lengths
    whole = Batch([(n, n) for n in lengths], Hq, Hk, D, page, dtype,
                  False, seed=0)
    whole.cache, whole.table = cache, table.cpu()
    whole.q = torch.cat([torch.cat(x) for x in qs]).cpu()
    check(torch.cat([torch.cat(x) for x in outs]), *whole.want())
