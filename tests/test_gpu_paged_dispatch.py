"""The paged attention's variants that its other tests do not reach."""
import pytest
import torch

from tensor_fusion_amd.ops import paged

from paged_oracle import Batch, check

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
KEPT = pytest.mark.parametrize("quantized", [False, True],
                               ids=["wide", "e4m3"])


def dispatch(b, quantized):
    c = b.cache
    return paged._ext().dispatch(
        len(b.q), len(b.kv_lens), b.q.shape[1] // c.kv_heads, c.kv_heads,
        c.head_dim, b.table.shape[1] * c.page_size, quantized)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_whole_items_of_eight_waves(D, dtype):
    """8 bits, an item a workgroup: more items than would be shared by value,
    and no more than there are units."""

    seqs = [(1, 500), (1, 1), (9, 600), (0, 7), (1, 33)] * 5
    b = Batch(seqs, 32, 8, D, 32, dtype, True, seed=5)
    assert dispatch(b, True)[1:] == (8, 0, 1)
    assert 128 < 8 * len(seqs) <= 256
    out = torch.full(b.q.shape, 7.0, dtype=dtype, device="cuda")
    b.run(out=out)
    check(out, *b.want())
    assert torch.equal(b.run(), out)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_broken_values_in_shared_items(value, dtype):
    """Values that are not finite, in keys that some rows of a tile see, where
    a row's parts are joined."""

    seqs = [(3, 6000), (2, 900)]
    b = Batch(seqs, 4, 2, 64, 16, dtype, False, seed=11)
    assert dispatch(b, False)[2]
    for i, (n, kv) in enumerate(seqs):
        for back in (1, n // 2 + 1, 700):
            j = kv - back
            at, off = int(b.table[i, j // 16]), j % 16
            b.cache.v[at, 0, off, 5] = value
            b.cache.v[at, 1, off, 63] = -value
    check(b.run(), *b.want())


FALLING = [[0, 9, 4, 12], [7, 3, 0, 12], [12, 0, 0, 5], [5, -5, 900, 2],
           [2 ** 31 - 1, 0, -2 ** 31, 4]]


@pytest.mark.parametrize("seqs,heads,D,kind", [
    ([(4, 3000), (2, 2500), (6, 2800)], 8, 64, "shared"),
    ([(4, 40), (2, 30), (6, 70)], 8, 64, "whole"),
    ([(150, 150), (40, 90), (60, 60)], 8, 64, "many"),
    ([(60, 4000), (70, 2000), (9, 3000)], 4, 64, "split"),
    ([(150, 400)] * 3, 256, 32, "sorted")], ids=lambda x: x
    if isinstance(x, str) else "")
@KEPT
def test_starts_that_fall_stay_inside(seqs, heads, D, kind, quantized):
    """Rows may be left out; nothing on either side of them is written."""

    Hk = 2 if heads < 100 else 64
    b = Batch(seqs, heads, Hk, D, 16, BF16, quantized, seed=3)
    T = len(b.q)
    workers, _, join, splits = dispatch(b, quantized)
    assert kind == ("shared" if join else "whole" if workers else
                    "split" if splits > 1 else
                    "sorted" if Hk == 64 else "many")
    if kind == "sorted":  # more workgroups than places
        assert (T * heads // Hk // 128 + 3) * Hk > 768
    for starts in FALLING:
        starts = [s * T // 12 if 0 <= s <= 12 else s for s in starts]
        b.q_starts = torch.tensor(starts, dtype=torch.int32)
        flat = torch.full((T + 64, heads, D), 7.0, dtype=BF16, device="cuda")
        out = flat[32:32 + T]
        b.run(out=out)
        assert (flat[:32] == 7).all() and (flat[32 + T:] == 7).all()
    b.q_starts = torch.tensor([0, seqs[0][0], seqs[0][0] + seqs[1][0], T],
                              dtype=torch.int32)
    out = torch.full((T, heads, D), 7.0, dtype=BF16, device="cuda")
    if kind != "sorted":  # the oracle takes long for that many heads
        check(b.run(out=out), *b.want())
