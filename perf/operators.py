"""The paged KV-cache operators on sizes of real use.

Three kinds of case, one for each operator of a serving step over a paged
key/value cache (pages of [kv_heads, page, head_dim], 16-bit or 8-bit e4m3
with a power-of-two scale for every token and head):

  write   new keys and values go into the pages; a quantised cache is read
          back, so that what comes out are the values that it stands for
  rope    q and k are rotated, k and v go into the pages in the same pass
  attend  a packed, ragged batch of new tokens attends over its pages
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0


def _write(name, seqs, tokens, kv_heads, head_dim, page, dtype, quantized,
           padding):
    return {"name": name, "kind": "write", "seqs": seqs, "tokens": tokens,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "dtype": dtype, "quantized": quantized, "padding": padding}


def _rope(name, seqs, tokens, heads, kv_heads, head_dim, page, dtype,
          quantized):
    return {"name": name, "kind": "rope", "seqs": seqs, "tokens": tokens,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "quantized": quantized}


def _attend(name, seqs, q_min, q_max, past_min, past_max, heads, kv_heads,
            head_dim, page, dtype, quantized, causal=True):
    return {"name": name, "kind": "attend", "seqs": seqs, "q_min": q_min,
            "q_max": q_max, "past_min": past_min, "past_max": past_max,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "quantized": quantized,
            "causal": causal}


def listed():
    return [
        # one decode step of a batch of 8 (the flagship's batch): latency
        _write("write step", 8, 1, 8, 128, 16, "bf16", True, 0),
        # a prefill chunk of 8192 tokens from 4 prompts goes in quantised
        _write("write chunk", 4, 2048, 8, 128, 64, "fp16", True, 0),
        # odd lengths, few heads, a padded batch, a 16-bit cache
        _write("write odd", 7, 1021, 3, 64, 32, "bf16", False, 5),
        # one decode step with the rotation, 32 query heads over 8
        _rope("rope step", 8, 1, 32, 8, 128, 16, "bf16", False),
        # a prefill chunk with the rotation, 64 query heads, quantised
        _rope("rope chunk", 2, 4095, 64, 8, 128, 16, "bf16", True),
        # the flagship's decode step: batch 8 at a context of 512
        _attend("step short", 8, 1, 1, 512, 560, 32, 8, 128, 16, "bf16",
                False),
        # a full server's decode step: 64 ragged sequences, 8-bit cache
        _attend("step batch", 64, 1, 1, 700, 8191, 64, 8, 128, 16, "bf16",
                True),
        # one user with a very long document: the cache's axis is split
        _attend("step long", 1, 1, 1, 131000, 131071, 32, 8, 128, 64, "fp16",
                False),
        # few new tokens a sequence (drafted tokens checked together)
        _attend("draft check", 12, 3, 7, 90, 4000, 32, 8, 128, 32, "bf16",
                False),
        # a later chunk of a long prompt over what is there already
        _attend("chunk", 2, 1500, 2048, 3000, 6000, 32, 8, 128, 16, "bf16",
                False),
        # prompts and decode steps in one batch, odd sizes, 8-bit cache,
        # as many kv heads as query heads
        _attend("mixed", 9, 1, 613, 0, 1800, 12, 12, 64, 32, "fp16", True),
        # a whole prompt at the model's longest context: compute bound
        _attend("prefill", 1, 8192, 8192, 0, 0, 32, 8, 128, 64, "bf16",
                False),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of its range."""
    return min(high, max(low, int(round(
        math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["write", "rope", "attend", "attend"])
    head_dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64])
    dtype = rng.choice(["bf16", "fp16"])
    quantized = rng.random() < 0.5
    if kind == "attend":
        kv_heads, group = rng.choice([(8, 4), (8, 8), (2, 4), (4, 1), (3, 5)])
        form = rng.choice(["step", "few", "chunk"])
        if form == "chunk":
            seqs = rng.randint(1, 4)
            past_max = _spread(rng, 1, 6000)
            # no more products than a whole prompt at the longest context
            most = 2 ** 28 * 4 / (seqs * kv_heads * group)
            q_max = _spread(rng, 17, 4000)
            while q_max * (past_max + q_max) > most:
                q_max = q_max * 3 // 4
        else:
            seqs = _spread(rng, 1, 64)
            q_max = 1 if form == "step" else rng.randint(2, 16)
            past_max = _spread(rng, 100, 8000)
        q_min = rng.randint(1, q_max)
        return _nameless(_attend(
            "", seqs, q_min, q_max, past_max // 4, past_max,
            kv_heads * group, kv_heads, head_dim, page, dtype, quantized,
            rng.random() < 0.8))
    seqs = rng.randint(1, 16)
    tokens = max(1, _spread(rng, 1, 8192) // seqs)
    kv_heads = rng.choice([1, 2, 5, 8])
    if kind == "write":
        return _nameless(_write("", seqs, tokens, kv_heads, head_dim, page,
                                dtype, quantized, rng.choice([0, 3])))
    return _nameless(_rope("", seqs, tokens, kv_heads * rng.choice([1, 4, 8]),
                           kv_heads, head_dim, page, dtype, quantized))


def _nameless(case):
    del case["name"]
    return case


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: the
    case's own, whatever the seed of its values."""

    sizes = [v for k, v in sorted(case.items())
             if k != "name" and isinstance(v, int)]
    rng = random.Random(":".join(str(int(v)) for v in sizes))
    new = [rng.randint(case["q_min"], case["q_max"])
           for _ in range(case["seqs"])]
    past = [rng.randint(case["past_min"], case["past_max"])
            for _ in range(case["seqs"])]
    new[0], past[-1] = case["q_max"], case["past_max"]
    return new, [n + p for n, p in zip(new, past)]


def _values(gen, *shape, spread=1.0):
    return torch.randn(*shape, device="cuda", generator=gen) * spread


def _exponent(amax):
    """The smallest e with amax <= 448 * 2**e; 448 is 0.875 * 2**9."""

    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, -126).clamp(min=-126)


def _quantise(x, dtype):
    """e4m3 codes and biased exponents of rows of 32-bit values."""

    e = _exponent(x.abs().amax(-1))
    if dtype is torch.float16:  # the largest e4m3 value that fp16 holds
        x = x.clamp(-61440.0, 61440.0)
    codes = torch.ldexp(x, -e.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values_of(codes, exponents):
    return torch.ldexp(codes.float(), exponents.to(torch.int32).unsqueeze(-1)
                       - 127)


def _pools(gen, pages, kv_heads, page, head_dim, dtype, quantized):
    """The pages as earlier tokens left them. Keys have a few large
    channels, as trained models' keys do."""

    k = _values(gen, pages, kv_heads, page, head_dim)
    k *= 1 + 3 * (torch.arange(head_dim, device="cuda") % 29 == 7)
    v = _values(gen, pages, kv_heads, page, head_dim, spread=0.5)
    if not quantized:
        return {"k": k.to(dtype), "v": v.to(dtype), "k_scale": None,
                "v_scale": None}
    k, ke = _quantise(k.to(dtype).float(), dtype)
    v, ve = _quantise(v.to(dtype).float(), dtype)
    return {"k": k, "v": v, "k_scale": ke, "v_scale": ve}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    D, Hk = case["head_dim"], case["kv_heads"]
    s = {"kind": case["kind"], "quantized": case["quantized"]}
    if case["kind"] == "attend":
        new, total = _lengths(case)
    else:
        # where each sequence already stands: anywhere in its page
        new = [case["tokens"]] * case["seqs"]
        total = [n + (37 * i + 11) % (3 * page) for i, n in enumerate(new)]
    width = -(-max(total) // page)
    # page 0 belongs to nobody; the others are handed out in any order
    pages = 1 + width * len(new)
    s["table"] = (1 + torch.randperm(pages - 1, device="cuda", generator=gen)
                  ).view(len(new), width).to(torch.int32)
    s.update(_pools(gen, pages, Hk, page, D, dtype, case["quantized"]))
    if case["kind"] == "attend":
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["q"] = _values(gen, starts[-1], case["heads"], D).to(dtype)
        s["q_starts"] = torch.tensor(starts, dtype=torch.int32,
                                     device="cuda")
        s["kv_lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
        s["max_q"], s["causal"] = max(new), case["causal"]
        return s
    seq = torch.arange(len(new), device="cuda").repeat_interleave(
        case["tokens"])
    first = torch.tensor([t - n for t, n in zip(total, new)], device="cuda")
    pos = first[seq] + torch.arange(case["tokens"],
                                    device="cuda").repeat(len(new))
    s["slots"] = s["table"][seq, pos // page].long() * page + pos % page
    N = len(pos)
    if case["kind"] == "write":
        if case["padding"]:
            s["slots"] = torch.cat([s["slots"], torch.full(
                (case["padding"],), -1, device="cuda")])
            N += case["padding"]
        # the rows are columns of one product's output, as a model has them
        kv = _values(gen, N, 2 * Hk * D).to(dtype)
        s["k_new"] = kv[:, :Hk * D].unflatten(1, (Hk, D))
        s["v_new"] = kv[:, Hk * D:].unflatten(1, (Hk, D))
        return s
    Hq = case["heads"]
    qkv = _values(gen, N, (Hq + 2 * Hk) * D).to(dtype)
    s["q_in"], s["k_in"], s["v_in"] = qkv.split(
        [Hq * D, Hk * D, Hk * D], dim=1)
    s["pos"], s["heads"] = pos, Hq
    inv = 500000.0 ** (-torch.arange(0, D, 2, device="cuda",
                                     dtype=torch.float64) / D)
    angle = torch.arange(8192 + 256, device="cuda",
                         dtype=torch.float64)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ---- the plain forms -------------------------------------------------------


def _put(s, k, v, dtype):
    """Rows of 32-bit values into the pages; slot -1 is no slot, and page 0,
    which belongs to nobody, takes its own value again in its place."""

    page = s["k"].shape[2]
    keep = (s["slots"] >= 0).view(-1, 1, 1)
    slots = s["slots"].clamp(min=0)
    at = (slots // page, slice(None), slots % page)
    for pool, scale, x in (("k", "k_scale", k), ("v", "v_scale", v)):
        if not s["quantized"]:
            s[pool][at] = torch.where(keep, x.to(dtype), s[pool][at])
            continue
        codes, e = _quantise(x, dtype)
        bits, old = codes.view(torch.uint8), s[pool].view(torch.uint8)
        old[at] = torch.where(keep, bits, old[at])
        s[scale][at] = torch.where(keep[..., 0], e, s[scale][at])


def _get(s, dtype):
    page = s["k"].shape[2]
    keep = (s["slots"] >= 0).view(-1, 1, 1)
    slots = s["slots"].clamp(min=0)
    at = (slots // page, slice(None), slots % page)
    out = []
    for pool, scale in (("k", "k_scale"), ("v", "v_scale")):
        codes = s[pool].view(torch.uint8)[at].view(torch.float8_e4m3fn)
        x = _values_of(codes, s[scale][at])
        out.append(torch.where(keep, x, 0.0).to(dtype))
    return out


def _rotate(x, cos, sin):
    c, n = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)


def _plain_write(s):
    dtype = s["k_new"].dtype
    _put(s, s["k_new"].float(), s["v_new"].float(), dtype)
    return _get(s, dtype) if s["quantized"] else [s["k"], s["v"]]


def _plain_rope(s):
    dtype, D = s["q_in"].dtype, s["k"].shape[-1]
    cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
    q, k, v = (s[x].float().unflatten(1, (-1, D))
               for x in ("q_in", "k_in", "v_in"))
    _put(s, _rotate(k, cos, sin), v, dtype)
    kept = _get(s, dtype) if s["quantized"] else [s["k"], s["v"]]
    return [_rotate(q, cos, sin).to(dtype)] + kept


def _plain_attend(s):
    q, starts, total, table = s["q"], s["q_starts"], s["kv_lens"], s["table"]
    T, Hq, D = q.shape
    Hk, page = s["k"].shape[1:3]
    G, most = Hq // Hk, s["max_q"]
    keys = torch.arange(table.shape[1] * page, device=q.device)

    def gathered(pool, scale):
        x = s[pool]
        if s["quantized"]:
            x = x.view(torch.uint8)[table.long()].view(x.dtype)
            x = _values_of(x, s[scale][table.long()])
        else:
            x = x[table.long()].float()
        # [B, pages, Hk, page, D] -> [B, Hk, 1, keys, D], 0 past the end
        x = x.transpose(1, 2).flatten(2, 3)
        there = keys < total[:, None]
        return torch.where(there[:, None, :, None], x, 0.0).unsqueeze(2)

    # the packed rows as [B, most, Hq, D]; row t of a sequence that is
    # shorter than that is some other row, and is dropped at the end
    new = starts[1:] - starts[:-1]
    t = torch.arange(most, device=q.device)
    at = (starts[:-1, None] + t).clamp(max=T - 1)
    qs = q.float()[at].view(-1, most, Hk, G, D).permute(0, 2, 3, 1, 4)
    score = (qs * D ** -0.5) @ gathered("k", "k_scale").transpose(-1, -2)
    last = (total - 1)[:, None].expand(-1, most)
    if s["causal"]:
        last = (total - new)[:, None] + t
    seen = keys <= last[..., None]  # [B, most, keys]
    seen &= keys < total[:, None, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.exp_()
    out = (p @ gathered("v", "v_scale")) / p.sum(-1, keepdim=True)
    out = torch.where(seen.any(-1)[:, None, None, :, None], out, 0.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, most, Hq, D]
    row = torch.arange(T, device=q.device)
    seq = (row[:, None] >= starts[1:]).sum(1)
    return out[seq, row - starts[seq]].to(q.dtype)


def run(s):
    if not own:
        return {"write": _plain_write, "rope": _plain_rope,
                "attend": _plain_attend}[s["kind"]](s)
    from tensor_fusion_amd.ops import paged
    cache = paged.PagedKVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["kind"] == "attend":
        return paged.paged_attention(s["q"], cache, s["q_starts"],
                                     s["kv_lens"], s["table"],
                                     causal=s["causal"])
    if s["kind"] == "write":
        paged.kv_write(cache, s["k_new"], s["v_new"], s["slots"])
        if s["quantized"]:
            return list(paged.kv_read(cache, s["slots"],
                                      s["k_new"].dtype))
        return [s["k"], s["v"]]
    q = paged.rope_kv_write(cache, s["q_in"], s["k_in"], s["v_in"], s["cos"],
                            s["sin"], s["pos"], s["slots"], s["heads"])
    if s["quantized"]:
        return [q, *paged.kv_read(cache, s["slots"], s["q_in"].dtype)]
    return [q, s["k"], s["v"]]


def work(case):
    D, Hk, quantized = case["head_dim"], case["kv_heads"], case["quantized"]
    row = 2 * Hk * (D + 1 if quantized else 2 * D)  # K and V in the cache
    if case["kind"] == "attend":
        new, total = _lengths(case)
        pairs = sum(n * t - (n * (n - 1) // 2 if case["causal"] else 0)
                    for n, t in zip(new, total))
        return {"bytes": sum(total) * row + 4 * sum(new) * case["heads"] * D,
                "flops": 4 * D * case["heads"] * pairs}
    N = case["seqs"] * case["tokens"]
    # new rows in, cache rows out, and 8-bit rows read and returned again
    moved = N * (4 * Hk * D + row + 8)
    if quantized:
        moved += N * (row + 4 * Hk * D)
    if case["kind"] == "write":
        return {"bytes": moved, "flops": 6 * N * Hk * D}
    q = case["heads"] * D
    return {"bytes": moved + N * (4 * q + 4 * D + 8),
            "flops": 3 * N * (q + Hk * D) + 6 * N * Hk * D}


# ---- the definitions in 64 bits --------------------------------------------


def _e4m3_exact(x, half):
    """Rows of 64-bit values as an e4m3 cache stands for them, by its
    definition: a scale 2**e, 3 bits of fraction, steps of 2**-9 at the
    bottom, ties to even."""

    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / E4M3_MAX))
    # the logarithm is near enough for all but a whole number
    e = torch.where(top <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > E4M3_MAX * torch.exp2(e), e + 1, e).clamp(min=-126)
    if half:
        x = x.clamp(-61440.0, 61440.0)
    y = x / torch.exp2(e)
    binade = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20)))
    binade = torch.where(y.abs() >= torch.exp2(binade + 1), binade + 1,
                         binade)
    step = torch.exp2(binade.clamp(min=-6) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_cache(s, case, rows_k, rows_v):
    """What a case that writes returns of its cache."""

    half = case["dtype"] == "fp16"
    page = case["page"]
    there = s["slots"] >= 0
    out = []
    for pool, rows in (("k", rows_k), ("v", rows_v)):
        if case["quantized"]:
            x = _e4m3_exact(rows, half)
            x[~there] = 0
        else:
            x = s[pool].double()
            at = s["slots"][there]
            x[at // page, :, at % page] = rows[there]
        out.append(x)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    D = case["head_dim"]
    if case["kind"] == "write":
        return _exact_cache(s, case, s["k_new"].double(),
                            s["v_new"].double())
    if case["kind"] == "rope":
        z = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"]]

        def turned(x):
            pairs = x.double().view(len(x), -1, D // 2, 2)
            return torch.view_as_real(torch.view_as_complex(
                pairs.contiguous()) * z[:, None]).flatten(-2)

        return [turned(s["q_in"])] + _exact_cache(
            s, case, turned(s["k_in"]),
            s["v_in"].double().unflatten(1, (-1, D)))
    new, total = _lengths(case)
    Hk, G = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, kv) in enumerate(zip(new, total)):
        use = s["table"][b, :-(-kv // case["page"])].long()

        def cached(pool, h):
            x = s[pool].view(torch.uint8)[use, h].view(s[pool].dtype) \
                if case["quantized"] else s[pool][use, h]
            x = x.double()
            if case["quantized"]:
                x = x * torch.exp2(s[pool + "_scale"][use, h].double()
                                   - 127).unsqueeze(-1)
            return x.flatten(0, 1)[:kv]

        for h in range(Hk):
            k, v = cached("k", h), cached("v", h)
            for t in range(0, n, 1024):
                rows = s["q"][first + t:first + min(t + 1024, n),
                              h * G:(h + 1) * G].double()
                w = rows.flatten(0, 1) @ k.T / math.sqrt(D)
                if case["causal"]:
                    at = torch.arange(t, t + len(rows), device="cuda")
                    at = (at + kv - n).repeat_interleave(G)
                    w[torch.arange(kv, device="cuda") > at[:, None]] = \
                        -math.inf
                out[first + t:first + t + len(rows), h * G:(h + 1) * G] = (
                    torch.softmax(w, -1) @ v).view(len(rows), G, D)
        first += n
    return out
