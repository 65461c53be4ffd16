"""The paged operators' definitions in 64 bits on the CPU, and how far a
kernel may be from them."""
import torch

from tensor_fusion_amd.ops import paged

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step


def e4m3(x, half=False):
    """Rows of values -> (the values a quantised cache stands for, scale
    bytes); a row that is not finite is NaN."""

    x = x.double()
    top = x.abs().amax(-1)
    broken = ~torch.isfinite(x).all(-1)
    m, e = torch.frexp(torch.where(broken, 1.0, top))
    # 448 = 0.875 * 2**9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(top > 0, e, -126).clamp(min=-126)
    if half:
        x = x.clamp(-61440, 61440)
    y = torch.ldexp(x, -e.unsqueeze(-1))
    q = y.float().to(torch.float8_e4m3fn).double()
    v = torch.ldexp(q, e.unsqueeze(-1))
    v[broken] = float("nan")
    byte = torch.where(broken, 127, e + 127).to(torch.uint8)
    return v, byte


def cache_values(cache):
    """The pools' values, float64 on the CPU."""

    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = x.cpu().float().double()
        if s is not None:
            x = torch.ldexp(x, s.cpu().to(torch.int32).unsqueeze(-1) - 127)
        out.append(x)
    return out


def attend(q, cache, q_starts, kv_lens, table, scale, causal, dtype):
    """(out, tolerance) of the rows that belong to sequences, and which rows
    those are.

    Tolerance, for each value: the result's rounding, u |o|; p's rounding,
    at most u of every term, u A with A = sum p |v| / sum p (fp16 also has a
    smallest step, 2**-25 a key, against a sum of at least 1); the 32-bit
    score, a sum of D products and 4 roundings more, which enters p as a
    relative error; 32-bit sums over the n keys; 4 steps of 2**-23 for the
    exponential and the quotient."""

    T, Hq, D = q.shape
    q = q.cpu().double()
    pools = cache_values(cache)
    Hk, page = cache.kv_heads, cache.page_size
    G = Hq // Hk
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    mine = torch.zeros(T, dtype=torch.bool)
    u = EPS[dtype]
    for b in range(len(kv_lens)):
        first, last = int(q_starts[b]), int(q_starts[b + 1])
        n, length = last - first, int(kv_lens[b])
        mine[first:last] = True
        pages = table[b, :-(-length // page)].long().cpu()
        k, v = (x[pages].transpose(0, 1).flatten(1, 2)[:, :length]
                for x in pools)  # [Hk, length, D]
        for t in range(n):
            see = min(max(length - n + t + 1, 0), length) if causal \
                else length
            if see == 0:
                continue
            row = q[first + t].view(Hk, G, D)
            s = row @ k[:, :see].transpose(1, 2) * scale  # [Hk, G, see]
            mag = (row.abs() @ k[:, :see].abs().transpose(1, 2)).amax(-1)
            p = torch.softmax(s, -1)
            o = p @ v[:, :see]
            A = p @ v[:, :see].abs()
            ds = (D + 8) * 2.0 ** -24 * mag * abs(scale)
            rel = u + 2 * ds + (see + 64) * 2.0 ** -24 + 4 * 2.0 ** -23
            least = 2.0 ** -25 * v[:, :see].abs().sum(1, keepdim=True) \
                if dtype is torch.float16 else 0.0
            out[first + t] = o.reshape(Hq, D)
            tol[first + t] = (u * 1.01 * o.abs() + rel.unsqueeze(-1) * A
                              + least + 2.0 ** -24).reshape(Hq, D)
    return out, tol, mine


def check(got, want, tol, mine):
    got = got.cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got)[mine], nan[mine])
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = mine.view(-1, 1, 1) & ~nan & ~inf
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


class Batch:
    """A ragged batch over pages in any order. `seqs`: (new tokens, keys) of
    each. Slots that belong to nobody hold NaN."""

    def __init__(self, seqs, heads, kv_heads, D, page, dtype, quantized,
                 seed=0, device="cuda", spread=1.0, extra_cols=1):
        g = torch.Generator().manual_seed(seed)
        width = max(-(-kv // page) for _, kv in seqs) + extra_cols
        pages = width * len(seqs) + 3
        perm = torch.randperm(pages, generator=g)[:width * len(seqs)]
        self.table = perm.view(len(seqs), width).to(torch.int32)
        shape = (pages, kv_heads, page, D)
        k = torch.full(shape, float("nan"))
        v = torch.full(shape, float("nan"))
        for b, (_, kv) in enumerate(seqs):
            for j in range(-(-kv // page)):
                n = min(page, kv - j * page)
                at = int(self.table[b, j])
                k[at, :, :n] = torch.randn(kv_heads, n, D, generator=g) \
                    * spread
                v[at, :, :n] = torch.randn(kv_heads, n, D, generator=g)
        if quantized:
            parts = []
            for x in (k, v):
                x = x.to(dtype).float()
                val, byte = e4m3(torch.nan_to_num(x), dtype is torch.float16)
                codes = torch.ldexp(val.float(), 127 - byte.to(
                    torch.int32).unsqueeze(-1)).to(torch.float8_e4m3fn)
                bits = codes.view(torch.uint8)
                bits[torch.isnan(x)] = 0x7f
                parts.append((bits.to(device).view(torch.float8_e4m3fn),
                              byte.to(device)))
            self.cache = paged.PagedKVCache(parts[0][0], parts[1][0],
                                            parts[0][1], parts[1][1])
        else:
            self.cache = paged.PagedKVCache(k.to(dtype).to(device),
                                            v.to(dtype).to(device))
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.q_starts = torch.tensor(starts, dtype=torch.int32)
        self.kv_lens = torch.tensor([kv for _, kv in seqs],
                                    dtype=torch.int32)
        self.q = torch.randn(starts[-1], heads, D, generator=g).to(dtype)
        self.dtype, self.device = dtype, device

    def run(self, **kw):
        d = self.device
        return paged.paged_attention(
            self.q.to(d), self.cache, self.q_starts.to(d),
            self.kv_lens.to(d), self.table.to(d), **kw)

    def want(self, scale=None, causal=True):
        scale = self.q.shape[-1] ** -0.5 if scale is None else scale
        return attend(self.q, self.cache, self.q_starts, self.kv_lens,
                      self.table, scale, causal, self.dtype)
