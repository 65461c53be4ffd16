"""Tensor parallelism over paged caches: each rank has its kv heads' pages."""
import threading

import pytest
import torch

from tensor_fusion_amd.models import llama as L
from tensor_fusion_amd.ops.paged import PagedBatch
from tensor_fusion_amd.parallel import tp as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
ROWS = ("wo.", "down.")  # split by columns; other products by rows


def run(m, toks):
    """A prompt in two ragged chunks, then steps."""

    table = torch.randperm(12, generator=torch.Generator().manual_seed(4)).to(
        torch.int32).view(3, 4).cuda()
    caches = m.make_paged_cache(12, 16, "cuda", BF16)
    past = torch.zeros(3, dtype=torch.int64, device="cuda")
    outs = []
    for new in ([20, 7, 33], [4, 17, 0], [1, 1, 1], [1, 1, 1]):
        at = past.tolist()
        x = torch.cat([toks[i, a:a + n] for i, (a, n) in
                       enumerate(zip(at, new))])[None]
        b = PagedBatch.of(table, past, new, 16)
        outs.append(m(x, pos=b.pos, caches=b.over(caches))[0])
        past += torch.tensor(new, device="cuda")
    return torch.cat(outs)


def sharded(m, tp, rank):
    names = dict(m.named_parameters())
    part = P.TPLlama(m.cfg, tp).to(BF16).cuda()
    with torch.no_grad():
        for name, p in part.named_parameters():
            w = names[name.replace(".linear.", ".")]
            if p.shape != w.shape:
                w = w.chunk(tp, 1 if any(r in name for r in ROWS) else 0)[rank]
            p.copy_(w)
    return part


def test_two_ranks_are_one_model(monkeypatch):
    """Two ranks in one process, in lock step, their reductions through a
    barrier. A reduction rounds two halves and their sum, where one rank
    rounds once: the variance of its roundings at most doubles, so the distance
    from the same weights in 64 bits is at most sqrt(2) as large, bounded by
    half as much again."""

    torch.manual_seed(2)
    m = L.build_model("tiny", dtype=BF16)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(2.0) if p.dim() > 1 else p.add_(1.0)
    toks = torch.randint(0, 256, (3, 64), device="cuda")
    barrier, halves = threading.Barrier(2, timeout=60), [None, None]
    rank = threading.local()

    def all_reduce(x):
        halves[rank.id] = x
        barrier.wait()
        y = halves[0] + halves[1]
        barrier.wait()
        return y

    monkeypatch.setattr(P, "_all_reduce", all_reduce)
    parts, outs = [sharded(m, 2, r) for r in range(2)], [None, None]
    for part in parts:
        assert part.make_paged_cache(1, 16, "cuda", BF16)[0].kv_heads == 1

    def work(r):
        rank.id = r
        try:
            with torch.no_grad():
                outs[r] = run(parts[r], toks)
        except BaseException:
            barrier.abort()
            raise

    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert torch.equal(*outs)
    with torch.no_grad():
        one = run(m, toks)
        # the same rows of whole forward passes in 64 bits
        exact = L.build_model("tiny", dtype=BF16)
        exact.load_state_dict(m.state_dict())
        exact = exact.double()
        exact._cos, exact._sin = L.precompute_rope(exact.cfg, "cuda")
        whole = exact(toks)
    rows, past = [], [0, 0, 0]
    for new in ([20, 7, 33], [4, 17, 0], [1, 1, 1], [1, 1, 1]):
        for i, n in enumerate(new):
            rows.append(whole[i, past[i]:past[i] + n])
            past[i] += n
    want = torch.cat(rows)

    def off(x):
        return ((x.double() - want).norm() / want.norm()).item()

    assert off(outs[0]) <= 1.5 * off(one), (off(outs[0]), off(one))
