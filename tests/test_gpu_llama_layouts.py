"""The fused path after its weights have changed: as a model that never had
others."""
import copy

import pytest
import torch

from tensor_fusion_amd.models import llama as L
from tensor_fusion_amd.ops.paged import PagedBatch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def other_weights(m, seed=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {k: torch.randn(w.shape, device="cuda", generator=g).to(w.dtype)
            * 0.05 + (w.dim() == 1) for k, w in m.state_dict().items()}


def paged_run(m, dtype, quantized=False):
    """A prompt and two steps."""

    caches = m.make_paged_cache(8, 16, "cuda", dtype, quantized)
    table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
    past = torch.zeros(2, dtype=torch.int64, device="cuda")
    outs = []
    for n in (20, 1, 1):
        toks = (torch.arange(2 * n, device="cuda") * 37 % 256).view(2, n)
        b = PagedBatch.of(table, past, n, 16)
        outs.append(m(toks, pos=b.pos, caches=b.over(caches)))
        past += n
    return outs


def dense_run(m, dtype):
    caches = m.make_kv_cache(2, 64, "cuda", dtype)
    outs, at = [], 0
    for n in (20, 1, 1):
        toks = (torch.arange(2 * n, device="cuda") * 37 % 256).view(2, n)
        pos = torch.arange(at, at + n, device="cuda")
        at += n
        outs.append(m(toks, pos=pos, caches=caches, pos_end=at))
    return outs


@pytest.mark.parametrize("run", [paged_run, dense_run])
@pytest.mark.parametrize("small", ["0", "1"], ids=["", "all packed"])
@torch.no_grad()
def test_reloaded_weights(run, small, monkeypatch):
    monkeypatch.setattr(L, "_FUSED_OPS", True)
    monkeypatch.setenv("TF_PACKED_SMALL", small)
    m = L.build_model("tiny", dtype=BF16)
    first = run(m, BF16)
    new = other_weights(m)
    fresh = L.build_model("tiny", dtype=BF16, seed=3)
    fresh.load_state_dict(new)
    want = run(fresh, BF16)
    m.load_state_dict(new)
    got = run(m, BF16)
    for g, w, f in zip(got, want, first):
        assert torch.equal(g, w) and not torch.equal(g, f)
    for p in m.parameters():
        p.mul_(0.5)
    for p in fresh.parameters():
        p.mul_(0.5)
    for g, w in zip(run(m, BF16), run(copy.deepcopy(fresh), BF16)):
        assert torch.equal(g, w)


@torch.no_grad()
def test_converted_weights(monkeypatch):
    monkeypatch.setattr(L, "_FUSED_OPS", True)
    m = L.build_model("tiny", dtype=BF16)
    m.load_state_dict(other_weights(m))
    first = paged_run(m, BF16)
    m.half()
    fresh = L.build_model("tiny", dtype=torch.float16, seed=3)
    fresh.load_state_dict(m.state_dict())
    for g, w in zip(paged_run(m, torch.float16),
                    paged_run(fresh, torch.float16)):
        assert torch.equal(g, w)
    m.bfloat16()  # bf16 to fp16 and back: these weights keep their values
    for g, w in zip(paged_run(m, BF16), first):
        assert (g - w).norm() <= 2.0 ** -5 * w.norm()


@torch.no_grad()
def test_a_captured_step_after_its_weights_changed(monkeypatch):
    """The graph reads what the eager step has laid out again."""

    monkeypatch.setattr(L, "_FUSED_OPS", True)
    m = L.build_model("tiny", dtype=BF16)
    m.load_state_dict(other_weights(m))
    caches = m.make_paged_cache(8, 16, "cuda", BF16)
    table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
    past = torch.full((2,), 5, dtype=torch.int64, device="cuda")
    cur = torch.full((2, 1), 9, device="cuda")

    def step():
        b = PagedBatch.of(table, past, 1, 16)
        return m(cur, pos=b.pos, caches=b.over(caches))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    last = None
    for seed in (1, 2, 3):
        m.load_state_dict(other_weights(m, seed))
        cur.fill_(seed)
        want = step()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        assert last is None or not torch.equal(want, last)
        last = want


@torch.no_grad()
def test_a_first_step_that_is_captured(monkeypatch):
    """What a capture lays out is its own: the next eager step does not read
    memory that only a replay fills."""

    monkeypatch.setattr(L, "_FUSED_OPS", True)
    warm = L.build_model("tiny", dtype=BF16)
    paged_run(warm, BF16)  # libraries, outside of the capture
    m = L.build_model("tiny", dtype=BF16, seed=1)
    m.load_state_dict(other_weights(m))
    x = torch.randn(2, 1, 128, device="cuda").to(BF16)
    a = m.blocks[0].attn
    want = torch.nn.functional.linear(x, torch.cat(
        [a.wq.weight, a.wk.weight, a.wv.weight]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.cat(a._merged_qkv(x), -1)
    got = torch.cat(a._merged_qkv(x), -1)
    assert torch.equal(got, want)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    a.wq.weight.mul_(2)  # laid out at each replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, torch.cat(a._merged_qkv(x), -1))
