"""The merged and shuffled copies of weights that the fused path keeps, which
follow the weights; and what the models refuse over pages. No GPU needed."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tensor_fusion_amd.models import llama as L

pytestmark = pytest.mark.usefixtures("native_built")


def attention(dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return L.Attention(L.CONFIGS["tiny"]).to(dtype).requires_grad_(False)


def doubled(a):
    return {k: v * 2 for k, v in a.state_dict().items()}


def in_place(a):
    for w in (a.wq.weight, a.wk.weight, a.wv.weight):
        w.mul_(2)


CHANGES = {
    "loaded": lambda a: a.load_state_dict(doubled(a)),
    "assigned": lambda a: a.load_state_dict(doubled(a), assign=True),
    "one loaded": lambda a: a.wk.load_state_dict(doubled(a.wk)),
    "in place": in_place,
    "one in place": lambda a: a.wv.weight.add_(1),
    "double": lambda a: a.double(),
    "there and back": lambda a: a.half().float(),
    "parameter": lambda a: setattr(a.wq, "weight",
                                   nn.Parameter(a.wq.weight * 3)),
    "data": lambda a: setattr(a.wq.weight, "data", a.wq.weight * 3),
    "layer": lambda a: setattr(a, "wk", nn.Linear(128, 64, bias=False)),
}


@pytest.mark.parametrize("change", CHANGES.values(), ids=CHANGES.keys())
@torch.no_grad()
def test_merged_weights_follow(change):
    a = attention()
    x = torch.randn(2, 3, 128)
    for _ in range(2):
        for y, w in zip(a._merged_qkv(x), (a.wq, a.wk, a.wv)):
            torch.testing.assert_close(y, w(x), rtol=1e-5, atol=1e-5)
        change(a)
        x = x.to(a.wq.weight.dtype)


@torch.no_grad()
def test_merged_weights_are_kept():
    """Laid out once, and again in the same memory: a captured graph may read
    it."""

    a = attention()
    x = torch.randn(1, 2, 128)
    calls = []
    real = torch.cat
    try:
        torch.cat = lambda *b, **kw: calls.append(1) or real(*b, **kw)
        for _ in range(3):
            a._merged_qkv(x)
        assert len(calls) == 1
        at = a._wqkv.value.data_ptr()
        in_place(a)
        a.to("cpu").float()  # nothing to convert
        a._merged_qkv(x)
        assert len(calls) == 2 and a._wqkv.value.data_ptr() == at
    finally:
        torch.cat = real


@torch.no_grad()
def test_a_copy_of_a_model_has_its_own():
    a = attention()
    x = torch.randn(1, 2, 128)
    a._merged_qkv(x)
    b = copy.deepcopy(a)
    in_place(b)
    for m in (a, b):
        assert torch.allclose(m._merged_qkv(x)[0], m.wq(x), atol=1e-5)


def test_weights_made_under_inference_mode():
    """They do not count their changes: loading and conversions are seen."""

    with torch.inference_mode():
        a = attention()
        x = torch.randn(1, 2, 128)
        for _ in range(2):
            assert torch.allclose(a._merged_qkv(x)[0], F.linear(
                x, a.wq.weight), atol=1e-5)
            a.load_state_dict(doubled(a))
        a.double()
        a._merged_qkv(x.double())
    with torch.no_grad():
        a._merged_qkv(x.double())


def test_merged_weights_ask_for_gradients():
    """Over pages too: a weight that asks for a gradient is not served from a
    copy that does not."""

    from tensor_fusion_amd.ops import paged
    a = attention(torch.bfloat16)
    cache = paged.make_cache(4, 16, 2, 32, device="cpu")
    batch = paged.PagedBatch.of(torch.zeros(1, 4, dtype=torch.int32),
                                torch.zeros(1, dtype=torch.int64), 3, 16)
    t = torch.zeros(8, 16)
    x = torch.zeros(1, 3, 128, dtype=torch.bfloat16)
    fused, L._FUSED_OPS = L._FUSED_OPS, True
    try:
        with pytest.raises(ValueError, match="run on a GPU"):
            a(x, t, t, batch.pos, (cache, batch))
        for w in (a.wq.weight, a.wk.weight, a.wv.weight):
            w.requires_grad_()
            with pytest.raises(RuntimeError, match="no backward"):
                a(x, t, t, batch.pos, (cache, batch))
            with torch.no_grad(), pytest.raises(ValueError,
                                                match="run on a GPU"):
                a(x, t, t, batch.pos, (cache, batch))
            w.requires_grad_(False)
    finally:
        L._FUSED_OPS = fused


def test_a_mask_over_pages():
    """Attention over pages takes none: it is not passed over."""

    from tensor_fusion_amd.ops import paged
    from tensor_fusion_amd.parallel.tp import TPAttention
    cfg = L.CONFIGS["tiny"]
    cache = paged.make_cache(4, 16, 2, 32, device="cpu")
    batch = paged.PagedBatch.of(torch.zeros(1, 4, dtype=torch.int32),
                                torch.zeros(1, dtype=torch.int64), 3, 16)
    t, x = torch.zeros(8, 16), torch.zeros(1, 3, 128, dtype=torch.bfloat16)
    for a in (attention(torch.bfloat16),
              TPAttention(cfg, 1).bfloat16().requires_grad_(False)):
        with pytest.raises(ValueError, match="mask"):
            a(x, t, t, batch.pos, (cache, batch),
              mask=torch.zeros(1, 1, 1, 64))
        with pytest.raises(ValueError, match="run on a GPU"):
            a(x, t, t, batch.pos, (cache, batch))


def test_a_decode_benchmark_past_the_positions():
    """Rows past the rotation's tables are NaN: no time is given for them."""

    m = L.build_model("tiny", device="cpu")
    for graphs, most in ((False, 512 - 12), (True, 512 - 15)):
        def run(ctx):
            L.decode_bench_paged(m, 1, ctx, 10, 2, graphs=graphs,
                                 device="cpu")

        with pytest.raises(ValueError, match="run on a GPU"):
            run(most)
        with pytest.raises(ValueError, match="positions"):
            run(most + 1)
