"""The models over paged caches: against their dense caches, captured, and
from the command line."""
import json
import os
import subprocess
import sys

import pytest
import torch

from tensor_fusion_amd.models import llama as L
from tensor_fusion_amd.ops.paged import PagedBatch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAGE = 16


def model(dtype=torch.bfloat16):
    m = L.build_model("tiny", device="cuda", dtype=dtype)
    for p in m.parameters():  # scores of some size, and norms about 1
        p.data.mul_(2.0) if p.dim() > 1 else p.data.add_(1.0)
    return m


def table_of(B, cols, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randperm(B * cols, device="cuda", generator=g).view(
        B, cols).to(torch.int32)


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype,fused", [
    (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False)],
    ids=["bf16", "bf16 fused", "fp16"])
@pytest.mark.parametrize("quantized", [False, True], ids=["wide", "e4m3"])
@torch.no_grad()
def test_paged_decode_against_the_whole_forward(dtype, quantized, fused,
                                                monkeypatch):
    """A prompt in two chunks, then token by token. The paged model rounds
    no more often than the dense one, so it may be no further from the same
    weights in 64 bits than half as much again; in 8 bits a key or value is
    off by up to 2^-4, which is less than 2^-3 of the logits."""

    m = model(dtype)
    B, T = 3, 41
    toks = torch.randint(0, 256, (B, T), device="cuda")
    exact = model(dtype).double()
    exact._cos, exact._sin = L.precompute_rope(exact.cfg, "cuda")
    want = exact(toks)
    dense = m.make_kv_cache(B, 64, "cuda", dtype)
    ref = [m(toks[:, :32], pos=torch.arange(32, device="cuda"),
             caches=dense, pos_end=32)]
    for t in range(32, T):
        ref.append(m(toks[:, t:t + 1], pos=torch.tensor([t], device="cuda"),
                     caches=dense, pos_end=t + 1))
    ref = torch.cat(ref, 1)

    monkeypatch.setattr(L, "_FUSED_OPS", fused)
    caches = m.make_paged_cache(B * 4, PAGE, "cuda", dtype, quantized)
    table = table_of(B, 4)
    got, past = [], torch.zeros(B, dtype=torch.int64, device="cuda")
    for n in [20, 12] + [1] * (T - 32):
        at = int(past[0])
        b = PagedBatch.of(table, past, n, PAGE)
        got.append(m(toks[:, at:at + n], pos=b.pos, caches=b.over(caches)))
        past += n
    got = torch.cat(got, 1)
    assert got.shape == ref.shape
    bound = 2.0 ** -3 if quantized else 1.5 * off(ref, want)
    assert off(got, want) <= bound, (off(got, want), off(ref, want))


@torch.no_grad()
def test_ragged_batch_is_its_sequences():
    """Prompts of different lengths and decode steps packed in one pass."""

    m = model()
    table = table_of(4, 5, seed=1)
    caches = m.make_paged_cache(20, PAGE, "cuda", torch.bfloat16)
    alone = m.make_paged_cache(20, PAGE, "cuda", torch.bfloat16)
    past = torch.zeros(4, dtype=torch.int64, device="cuda")
    for new in ([7, 33, 0, 20], [1, 1, 40, 1], [5, 0, 1, 17]):
        toks = [torch.randint(0, 256, (1, n), device="cuda") for n in new]
        b = PagedBatch.of(table, past, new, PAGE)
        got = m(torch.cat(toks, 1), pos=b.pos, caches=b.over(caches))
        for i, (n, part) in enumerate(zip(new, got[0].split(new))):
            if n == 0:
                continue
            one = PagedBatch.of(table[i:i + 1], past[i:i + 1], n, PAGE)
            want = m(toks[i], pos=one.pos, caches=one.over(alone))[0]
            # the kernels may take other tiles, with one more rounding of p
            assert off(part, want.double()) < 2.0 ** -7
        past += torch.tensor(new, device="cuda")


def test_batch_of():
    table = torch.tensor([[5, 2], [1, 9]], dtype=torch.int32, device="cuda")
    past = torch.tensor([3, 15], device="cuda")
    b = PagedBatch.of(table, past, 2, PAGE)
    assert b.q_starts.tolist() == [0, 2, 4] and b.kv_lens.tolist() == [5, 17]
    assert b.pos.tolist() == [3, 4, 15, 16]
    assert b.slots.tolist() == [83, 84, 31, 144]
    c = PagedBatch.of(table, past, [2, 2], PAGE)
    for x, y in zip((b.q_starts, b.kv_lens, b.pos, b.slots),
                    (c.q_starts, c.kv_lens, c.pos, c.slots)):
        assert torch.equal(x, y) and x.dtype == y.dtype
    # past the table: no slot
    d = PagedBatch.of(table, past + 16, 2, PAGE)
    assert d.slots.tolist() == [35, 36, 159, -1]
    assert PagedBatch.of(table, past, 0, PAGE).q_starts.tolist() == [0] * 3
    assert PagedBatch.of(table, past, [0, 1], PAGE).slots.tolist() == [31]
    with pytest.raises(ValueError, match="counts"):
        PagedBatch.of(table, past, [1], PAGE)
    with pytest.raises(ValueError, match="without columns"):
        PagedBatch.of(table[:, :0], past, 1, PAGE)


def test_a_pass_that_asks_for_gradients_is_refused():
    m = model()
    caches = m.make_paged_cache(4, PAGE, "cuda", torch.bfloat16)
    b = PagedBatch.of(table_of(1, 4), torch.zeros(1, device="cuda"), 3, PAGE)
    with pytest.raises(RuntimeError, match="no backward"):
        m(torch.zeros(1, 3, dtype=torch.int64, device="cuda"), pos=b.pos,
          caches=b.over(caches))


@pytest.mark.parametrize("quantized", [False, True], ids=["wide", "e4m3"])
@torch.no_grad()
def test_captured_decode_step(quantized):
    """One graph, replayed over a page's end, with the program's own work
    between: the logits of each step are the eager ones."""

    m = model()
    B = 2
    table = table_of(B, 4, seed=2)
    runs = []
    for _ in range(2):
        caches = m.make_paged_cache(B * 4, PAGE, "cuda", torch.bfloat16,
                                    quantized)
        past = torch.tensor([9, 14], device="cuda")
        prompt = PagedBatch.of(table, past * 0, [9, 14], PAGE)
        g = torch.Generator(device="cuda").manual_seed(5)
        toks = torch.randint(0, 256, (1, 23), device="cuda", generator=g)
        m(toks, pos=prompt.pos, caches=prompt.over(caches))
        cur = torch.full((B, 1), 7, device="cuda")
        runs.append((caches, past, cur))

    def step(caches, past, cur):
        b = PagedBatch.of(table, past, 1, PAGE)
        logits = m(cur, pos=b.pos, caches=b.over(caches))
        cur.copy_(logits.argmax(-1))
        past.add_(1)
        return logits

    warm = (m.make_paged_cache(B * 4, PAGE, "cuda", torch.bfloat16,
                               quantized), runs[0][1].clone(),
            runs[0][2].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*runs[0])
    for i in range(30):
        graph.replay()
        want = step(*runs[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(runs[0][2], runs[1][2])


@torch.no_grad()
def test_tensor_parallel_model_of_one_rank():
    from tensor_fusion_amd.parallel.tp import TPLlama
    m = model()
    tp = TPLlama(m.cfg, 1).to(torch.bfloat16).cuda()
    names = dict(m.named_parameters())
    for name, p in tp.named_parameters():
        p.data.copy_(names[name.replace(".linear.", ".")].data)
    toks = torch.randint(0, 256, (2, 30), device="cuda")
    table, past = table_of(2, 2), torch.zeros(2, device="cuda")
    outs = []
    for x in (m, tp):
        caches = x.make_paged_cache(4, PAGE, "cuda", torch.bfloat16)
        b = PagedBatch.of(table, past, 30, PAGE)
        outs.append(x(toks, pos=b.pos, caches=b.over(caches)))
    assert torch.equal(*outs)


@pytest.mark.parametrize("flags", [[], ["--graphs"],
                                   ["--graphs", "--kv-e4m3", "--page-size",
                                    "16"]], ids=["eager", "graph", "e4m3"])
def test_decode_from_the_command_line(flags):
    out = subprocess.run(
        [sys.executable, "-m", "tensor_fusion_amd.models.llama", "--model",
         "tiny", "--batch", "2", "--ctx", "40", "--steps", "20", "--warmup",
         "2", "--paged"] + flags, cwd=REPO, capture_output=True, text=True,
        timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert json.loads(out.stdout.strip().splitlines()[-1])["tok_s"] > 0
