"""The paged operators' answers to unusual arguments."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tensor_fusion_amd.ops import paged

from paged_oracle import Batch, check

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
KEPT = pytest.mark.parametrize("quantized", [False, True],
                               ids=["wide", "e4m3"])


def test_results_under_a_mode_that_fakes_tensors():
    """Real arguments, but what would be allocated for the result has no
    memory: refused, and nothing is launched."""

    b = Batch([(1, 40), (2, 30)], 4, 2, 64, 16, BF16, False, seed=1)
    q, starts = b.q.cuda(), b.q_starts.cuda()
    lens, table = b.kv_lens.cuda(), b.table.cuda()
    slots = torch.arange(4, device="cuda")
    with FakeTensorMode():
        with pytest.raises(ValueError, match="plain tensor"):
            paged.paged_attention(q, b.cache, starts, lens, table)
        with pytest.raises(ValueError, match="plain tensor"):
            paged.kv_read(b.cache, slots)
    check(paged.paged_attention(q, b.cache, starts, lens, table), *b.want())


# ---- results over what is read ------------------------------------------------


@pytest.mark.parametrize("heads,D,seqs", [
    (8, 64, [(1, 300), (1, 90), (1, 500)]),
    (8, 128, [(1, 300), (1, 90), (1, 500)]),
    (8, 64, [(1, 300)] * 40), (16, 128, [(2, 300)] * 40),
    (8, 64, [(1, 4000), (2, 3000)]), (8, 128, [(150, 150), (70, 400)]),
    (8, 64, [(40, 3000), (30, 2900)])],
    ids=["two an item", "four an item", "two, 40", "one an item", "shared",
         "many", "many in parts"])
@KEPT
def test_out_is_q(heads, D, seqs, quantized):
    """In place, and moved by some rows to either side: several workgroups
    read the rows that one of them writes."""

    b = Batch(seqs, heads, 2 if heads == 8 else 4, D, 16, BF16, quantized,
              seed=D)
    want = b.run()
    starts, lens, table = b.q_starts.cuda(), b.kv_lens.cuda(), b.table.cuda()
    T = len(b.q)
    flat = torch.empty(3 * T, heads, D, dtype=BF16, device="cuda")
    for first in (T, T - 1, T + 1, T - 1 - T // 2):
        flat.fill_(7.0)
        q, out = flat[T:2 * T], flat[first:first + T]
        q.copy_(b.q)
        assert paged.paged_attention(q, b.cache, starts, lens, table,
                                     out=out) is out
        assert torch.equal(out, want)
        assert (flat[:min(first, T)] == 7).all()
        assert (flat[max(first, T) + T:] == 7).all()


# ---- rows that lie in the cache themselves --------------------------------------


@pytest.mark.parametrize("heads,D", [(2, 64), (8, 128), (1, 32)])
def test_write_rows_of_the_cache(heads, D):
    """Tokens moved on by some slots, over each other: every row is written
    as it was before the call."""

    page, pages = 64, 40
    cache = paged.make_cache(pages, page, heads, D)
    n = pages * page
    k, v = torch.randn(2, n, heads, D, device="cuda").to(BF16)
    slots = torch.arange(n, device="cuda")
    for by in (1, 17, -3, 700):
        paged.kv_write(cache, k, v, slots)
        to = (slots + by) % n
        # the first page's rows, in order
        rows = [x[0].transpose(0, 1) for x in (cache.k, cache.v)]
        paged.kv_write(cache, *rows, to[:page])
        got = paged.kv_read(cache, slots)
        for x, new in zip(got, (k, v)):
            want = new.clone()
            want[to[:page]] = new[:page]
            assert torch.equal(x, want), by


def test_rope_rows_of_the_cache():
    """q and k of a product that lies where the pages are."""

    D, Hk, heads, n = 64, 2, 4, 512
    angle = torch.rand(n, D // 2, device="cuda")
    cos, sin = angle.cos(), angle.sin()
    pos = torch.arange(n, device="cuda")
    x = torch.randn(n, (heads + 2 * Hk) * D, device="cuda").to(BF16)
    apart, over = (paged.make_cache(n // 16 * 4, 16, Hk, D) for _ in "ab")
    rows = over.k.view(-1, (heads + 2 * Hk) * D)[:n]
    rows.copy_(x)
    slots = torch.randperm(4 * n, device="cuda")[:n]
    outs = [paged.rope_kv_write(c, *r.split([heads * D, Hk * D, Hk * D], 1),
                                cos, sin, pos, slots, heads)
            for c, r in ((apart, x), (over, rows))]
    assert torch.equal(*outs)
    for a, b in zip(paged.kv_read(apart, slots), paged.kv_read(over, slots)):
        assert torch.equal(a, b)


# ---- what autograd has kept ---------------------------------------------------


def test_a_tensor_kept_for_a_backward_pass_is_missed():
    """What is written in place counts as changed: a backward pass that had
    kept it is refused, and not computed from what lies there now."""

    b = Batch([(1, 40), (2, 30)], 4, 2, 64, 16, BF16, True, seed=1)
    q, starts = b.q.cuda(), b.q_starts.cuda()
    lens, table = b.kv_lens.cuda(), b.table.cuda()
    out, w = torch.zeros_like(q), torch.ones_like(q, requires_grad=True)
    y = (out * w).sum()
    paged.paged_attention(q, b.cache, starts, lens, table, out=out)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    c, slots = b.cache, torch.arange(3, device="cuda")
    k = torch.randn(3, 2, 64, device="cuda").to(BF16)
    cos = torch.ones(3, 32, device="cuda")
    kept = [c.k, c.v, c.k_scale, c.v_scale]
    for write in (lambda: paged.kv_write(c, k, k, slots),
                  lambda: paged.rope_kv_write(
                      c, k.flatten(1), k.flatten(1), k.flatten(1), cos, cos,
                      slots, slots, 2)):
        before = [x._version for x in kept]
        write()
        assert all(x._version > v for x, v in zip(kept, before))
    before = [x._version for x in kept]
    paged.kv_read(c, slots)
    paged.paged_attention(q, c, starts, lens, table)
    assert [x._version for x in kept] == before


def test_under_inference_mode():
    with torch.inference_mode():
        b = Batch([(1, 40), (2, 30)], 4, 2, 64, 16, BF16, False, seed=1)
        out = torch.empty(3, 4, 64, dtype=BF16, device="cuda")
        check(b.run(out=out), *b.want())
        k = torch.randn(3, 2, 64, device="cuda").to(BF16)
        slots = torch.arange(3, device="cuda")
        paged.kv_write(b.cache, k, k, slots)
        assert torch.equal(paged.kv_read(b.cache, slots)[0], k)


# ---- scales -----------------------------------------------------------------------


@pytest.mark.parametrize("seqs", [[(1, 90), (3, 40)], [(2, 5000)],
                                  [(130, 200)]],
                         ids=["few", "shared", "many"])
@KEPT
def test_no_scale_of_large_scores(seqs, quantized):
    """Scores of up to 2^128 and a scale of 0, or of less than 32 bits hold:
    every key has the same weight. (2^128 times the 2^-149 that stands for it
    is 2^-21, far below half a step of p.)"""

    b = Batch(seqs, 8, 2, 64, 16, BF16, quantized, seed=2)
    if quantized:
        b.cache.k_scale.add_(58)
    else:
        b.cache.k.mul_(2.0 ** 58)
    b.q = b.q * 2.0 ** 60  # products of up to 64 * 4 * 4 * 2^118 < 2^128
    for scale in (0.0, 1e-60, -0.0):
        check(b.run(scale=scale), *b.want(scale=0.0))
