"""Arguments of the paged operators that look right and are not: no GPU
needed. Each is refused before anything is launched."""
import pytest
import torch
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
