"""Arguments of the paged operators that look right and are not: no GPU
needed. Each is refused before anything is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from tensor_fusion_amd.ops import paged

pytestmark = pytest.mark.usefixtures("native_built")

BF16, I32 = torch.bfloat16, torch.int32
SLOTS = torch.arange(3)


def cache(**kw):
    return paged.make_cache(5, 16, 2, 64, device="cpu", **kw)


def rows(n=3, heads=2):
    return torch.zeros(n, heads, 64, dtype=BF16)


def attend(c, q=None, **kw):
    q = rows(heads=4) if q is None else q
    return paged.paged_attention(
        q, c, torch.tensor([0, 1, 3], dtype=I32),
        torch.tensor([5, 9], dtype=I32), torch.zeros(2, 3, dtype=I32), **kw)


def rope(c, **kw):
    t = torch.zeros(8, 32)
    a = dict(q_in=rows(heads=4).flatten(1), k_in=rows().flatten(1),
             v_in=rows().flatten(1), cos=t, sin=t, pos=SLOTS, slots=SLOTS)
    a.update(kw)
    return paged.rope_kv_write(c, *a.values(), 4)


# ---- tensors whose values are not what lies at their address ---------------


class Wrapper(torch.Tensor):
    """A tensor around another, as distributed and quantised tensors are."""

    @staticmethod
    def __new__(cls, x):
        return torch.Tensor._make_wrapper_subclass(
            cls, x.shape, dtype=x.dtype, device=x.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError("not asked for")


def emptied(x):
    x = x.clone()
    x.untyped_storage().resize_(0)
    return x


@pytest.mark.parametrize("broken", [Wrapper, torch._neg_view, emptied],
                         ids=["wrapper", "negated", "emptied"])
def test_tensors_without_memory_of_their_own(broken):
    c = cache()
    for call in (lambda: paged.kv_write(c, broken(rows()), rows(), SLOTS),
                 lambda: paged.kv_write(c, rows(), broken(rows()), SLOTS),
                 lambda: rope(c, q_in=broken(rows(heads=4).flatten(1))),
                 lambda: rope(c, cos=broken(torch.zeros(8, 32))),
                 lambda: attend(c, broken(rows(heads=4))),
                 lambda: attend(c, out=broken(rows(heads=4))),
                 lambda: paged.PagedKVCache(broken(c.k), c.v)):
        with pytest.raises(ValueError, match="plain tensor"):
            call()


def test_transformed_functions():
    c, x = cache(), rows()

    def write(k):
        paged.kv_write(c, k, x, SLOTS)
        return k

    for call in (lambda: torch.func.vmap(write)(x[None]),
                 lambda: torch.func.jvp(write, (x,), (x,)),
                 lambda: torch.func.functionalize(write)(x)):
        with pytest.raises(ValueError, match="plain tensor"):
            call()


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fake_tensors(device):
    """They claim a device and have no memory there."""

    c = cache()
    with FakeTensorMode():
        with pytest.raises(ValueError, match="plain tensor"):
            paged.make_cache(5, 16, 2, 64, device=device)
        q = torch.zeros(3, 4, 64, dtype=BF16, device=device)
    with pytest.raises(ValueError, match="plain tensor"):
        attend(c, q)


# ---- results over what is read ------------------------------------------------


@pytest.mark.parametrize("pool", ["k", "v", "k_scale", "v_scale"])
def test_out_over_the_cache(pool):
    """From the byte behind it to the byte before it, and not next to it."""

    c = cache(quantized=True)
    parts = {p: getattr(c, p) for p in ("k", "v", "k_scale", "v_scale")}
    x, size = parts[pool], 3 * 4 * 64 * 2
    flat = torch.zeros(2 * size + x.numel(), dtype=torch.uint8)
    parts[pool] = flat[size:size + x.numel()].view(x.dtype).view(x.shape)
    c = paged.PagedKVCache(*parts.values())
    last = size + x.numel()
    for first, match in ((0, "run on a GPU"), (16, "shares"),
                         (last - 16, "shares"), (last, "run on a GPU")):
        out = flat[first:first + size].view(BF16).view(3, 4, 64)
        with pytest.raises(ValueError, match=match):
            attend(c, out=out)


def test_out_over_the_lengths():
    flat = torch.zeros(3 * 4 * 64, dtype=BF16)
    ints = flat.view(I32)
    out = flat.view(3, 4, 64)
    a = dict(starts=torch.zeros(3, dtype=I32), lens=torch.zeros(2, dtype=I32),
             table=torch.zeros(2, 3, dtype=I32))
    over = dict(starts=ints[8:11], lens=ints[-2:], table=ints[:6].view(2, 3))
    for name, x in over.items():
        with pytest.raises(ValueError, match="shares"):
            paged.paged_attention(rows(heads=4), cache(),
                                  *{**a, name: x}.values(), out=out)


# ---- gradients in either direction ------------------------------------------


ASKED = {
    "write k": lambda c, g: paged.kv_write(c, g(rows()), rows(), SLOTS),
    "write v": lambda c, g: paged.kv_write(c, rows(), g(rows()), SLOTS),
    "rope q": lambda c, g: rope(c, q_in=g(rows(heads=4).flatten(1))),
    "rope k": lambda c, g: rope(c, k_in=g(rows().flatten(1))),
    "rope v": lambda c, g: rope(c, v_in=g(rows().flatten(1))),
    "rope cos": lambda c, g: rope(c, cos=g(torch.zeros(8, 32))),
    "rope sin": lambda c, g: rope(c, sin=g(torch.zeros(8, 32))),
    "attend q": lambda c, g: attend(c, g(rows(heads=4))),
    "attend out": lambda c, g: attend(c, out=g(rows(heads=4))),
    "attend cache": lambda c, g: attend(paged.PagedKVCache(c.k, g(c.v))),
    "read cache": lambda c, g: paged.kv_read(
        paged.PagedKVCache(g(c.k), c.v), SLOTS),
    "write cache": lambda c, g: paged.kv_write(
        paged.PagedKVCache(g(c.k), c.v), rows(), rows(), SLOTS),
}


@pytest.mark.parametrize("call", ASKED.values(), ids=ASKED.keys())
def test_no_gradient_in_either_direction(call):
    def leaf(x):
        return x.detach().requires_grad_()

    with pytest.raises(RuntimeError, match="no backward"):
        call(cache(), leaf)
    with torch.no_grad(), pytest.raises(ValueError, match="run on a GPU"):
        call(cache(), leaf)
    with fw.dual_level():
        def dual(x):
            return fw.make_dual(x.detach(), torch.ones_like(x))

        with pytest.raises(RuntimeError, match="no backward"):
            call(cache(), dual)
        # no_grad does not end forward mode
        with torch.no_grad(), pytest.raises(RuntimeError,
                                            match="no backward"):
            call(cache(), dual)


# ---- a cache whose tensors were changed under it ----------------------------


@pytest.mark.parametrize("change,match", [
    (lambda x: x.resize_(1, 2, 16, 64), "of one shape"),
    (lambda x: x.set_(torch.zeros(5, 2, 16, 32, dtype=BF16)), "of one shape"),
    (lambda x: x.swapaxes_(1, 2), "of one shape"),
    (lambda x: setattr(x, "data", torch.zeros(5, 2, 16, 64)), "bfloat16"),
    (lambda x: setattr(x, "data", torch.zeros(5, 2, 64, 16, dtype=BF16).mT),
     "without gaps"),
    (lambda x: setattr(x, "data", torch.zeros(5 * 2 * 16 * 64 + 1, dtype=BF16)
                       [1:].view(5, 2, 16, 64)), "multiples of 16"),
    (lambda x: x.untyped_storage().resize_(0), "plain tensor"),
    (lambda x: x.untyped_storage().resize_(4096), "plain tensor"),
], ids=["resize", "set", "swapaxes", "type", "gaps", "address", "emptied",
        "cut"])
def test_a_cache_that_was_changed(change, match):
    """What is read is what the tensors are at the call."""

    for which in "kv":
        c = cache()
        change(getattr(c, which))
        for call in (lambda: paged.kv_write(c, rows(), rows(), SLOTS),
                     lambda: paged.kv_read(c, SLOTS), lambda: rope(c),
                     lambda: attend(c)):
            with pytest.raises(ValueError, match=match):
                call()


def test_a_cache_that_was_moved():
    """Other memory of the same kind is taken as it is."""

    c = cache()
    for x in (c.k, c.v):
        x.data = torch.zeros(9, 2, 16, 64, dtype=BF16)
    with pytest.raises(ValueError, match="run on a GPU"):
        attend(c)


# ---- more than one launch takes ---------------------------------------------


def steps(B, heads, cols=1):
    """B steps over as many heads, without memory of that size."""

    c = paged.make_cache(1, 16, heads, 32, device="cpu")
    return paged.paged_attention(
        torch.zeros(1, 1, 32, dtype=BF16).expand(B, heads, 32), c,
        torch.zeros(B + 1, dtype=I32), torch.zeros(B, dtype=I32),
        torch.zeros(cols, dtype=I32).expand(B, cols))


def test_more_than_a_launch_takes():
    """A launch has less than 2**32 lanes, 2**24 workgroups of 256: here one
    for each of the B + B / 16 places of tiles, and head. Shared out by
    length, the places for tiles have 5 numbers each at least, of 2**30."""

    for fits, cols in ((493447, 1), (5263440, 1024)):
        with pytest.raises(ValueError, match="run on a GPU"):
            steps(fits, 32, cols)
        with pytest.raises(ValueError, match="too many"):
            steps(fits + 1, 32, cols)
    row = torch.zeros(1, 1, 1, dtype=BF16)
    c = paged.make_cache(1, 16, 1, 128, device="cpu")
    n = 2 ** 28  # 16 a workgroup
    k = row.expand(n, 1, 128)
    huge = torch.empty(n, dtype=torch.int64)  # never touched
    with pytest.raises(ValueError, match="run on a GPU"):
        paged.kv_write(c, k[16:], k[16:], huge[16:])
    for call in (lambda: paged.kv_write(c, k, k, huge),
                 lambda: paged.kv_read(c, huge),
                 lambda: paged.rope_kv_write(
                     c, k[:, 0], k[:, 0], k[:, 0], torch.zeros(1, 64),
                     torch.zeros(1, 64), huge, huge, 1)):
        with pytest.raises(ValueError, match="too many"):
            call()


# ---- a batch for pages of another size ----------------------------------------


def batch_of(page, new=3):
    return paged.PagedBatch.of(torch.zeros(1, 4, dtype=I32),
                               torch.zeros(1, dtype=torch.int64), new, page)


def test_a_batch_of_another_page_size():
    """Its slots would lie in pages of other sequences."""

    c, t = cache(), torch.zeros(8, 32)
    q, k = rows(heads=4).flatten(1), rows().flatten(1)
    for new in (3, [3]):
        for page in (8, 32, 64):
            b = batch_of(page, new)
            assert b.page_size == page
            with pytest.raises(ValueError, match="pages of"):
                paged.attend(q, k, k, t, t, c, b, 4)
            with pytest.raises(ValueError, match="pages of"):
                b.over([c])
        b = batch_of(16, new)
        with pytest.raises(ValueError, match="run on a GPU"):
            paged.attend(q, k, k, t, t, c, b, 4)
        assert [*map(id, sum(b.over(iter([c, c])), ()))] == [id(c), id(b)] * 2
    # slots of a caller's own
    own = paged.PagedBatch(b.q_starts, b.kv_lens, b.block_table, b.pos,
                           b.slots)
    with pytest.raises(ValueError, match="run on a GPU"):
        paged.attend(q, k, k, t, t, c, own, 4)
    for page in (0, -16):
        with pytest.raises(ValueError, match="page_size"):
            batch_of(page)


def test_scales_that_32_bits_do_not_hold():
    """Exponentials are of base 2: the scale times log2(e) has to be finite."""

    for scale in (2.4e38, -3e38, 1e39, float("inf")):
        with pytest.raises(ValueError, match="finite"):
            attend(cache(), scale=scale)
    for scale in (2.3e38, -2.3e38, 0.0, 1e-45, 1e-60):
        with pytest.raises(ValueError, match="run on a GPU"):
            attend(cache(), scale=scale)
