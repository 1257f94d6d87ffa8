"""Timed cases of the paged-serving operators: appending rotated keys and values to a paged cache (16-bit pages, or e4m3
pages with a scale for each page and head), attention over that cache (causal; optionally a sliding window with sink
tokens), and drawing tokens from logits (temperature, top-k, top-p, min-p).

Each case runs in two forms on the same inputs: a plain form of elementary torch operations, and the framework's
kernels (`own`). `exact` gives the operators' values from their definitions in 64 bits.
"""
import math

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _append(name, dtype, kv, batch, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim, page, rotary, interleaved):
    return {"name": name, "op": "append", "dtype": dtype, "kv": kv, "batch": batch, "new_lo": new_lo, "new_hi": new_hi,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "rotary": rotary, "interleaved": interleaved}


def _attend(name, dtype, kv, batch, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim, page, window, sinks):
    return {"name": name, "op": "attend", "dtype": dtype, "kv": kv, "batch": batch, "new_lo": new_lo, "new_hi": new_hi,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "sinks": sinks}


def _sample(name, dtype, rows, vocab, top_k, top_p, min_p):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "top_k": top_k, "top_p": top_p,
            "min_p": min_p}


def listed():
    return [
        # one user's next token in an 8B-width model, 16-bit pages: nothing but latency
        _append("append_one_token", "f16", "16bit", 1, 1, 1, 300, 300, 32, 8, 128, 16, 128, False),
        # 64 users' next tokens into e4m3 pages that are partly full: page scales grow, old rows are rescaled
        _append("append_batch_e4m3", "bf16", "e4m3", 64, 1, 1, 77, 3001, 32, 8, 128, 64, 128, False),
        # ragged prompts of a Scout-width model (5 query heads to a KV head), interleaved rotation of half the head
        _append("append_prompts_e4m3", "bf16", "e4m3", 3, 1021, 2801, 0, 517, 40, 8, 128, 32, 64, True),
        # many prompts at once, 16-bit pages: the largest append
        _append("append_prompts_16bit", "f16", "16bit", 9, 700, 2500, 0, 1300, 32, 8, 128, 64, 128, False),
        # one user, short context: latency
        _attend("decode_one_short", "f16", "16bit", 1, 1, 1, 300, 300, 32, 8, 128, 16, 0, 0),
        # a serving batch of mixed lengths over 16-bit pages
        _attend("decode_batch_16bit", "bf16", "16bit", 24, 1, 1, 150, 6500, 32, 8, 128, 64, 0, 0),
        # the same kind of batch over e4m3 pages
        _attend("decode_batch_e4m3", "bf16", "e4m3", 32, 1, 1, 413, 8111, 32, 8, 128, 64, 0, 0),
        # one user with a long document, 70B width: few rows, a long axis
        _attend("decode_long_e4m3", "f16", "e4m3", 1, 1, 1, 131000, 131000, 64, 8, 128, 64, 0, 0),
        # long chats served with a window and four sink tokens
        _attend("decode_window_sinks", "bf16", "16bit", 16, 1, 1, 3300, 40000, 40, 8, 128, 32, 4096, 4),
        # chunks of prompts behind what is cached already, causal
        _attend("prompt_chunks", "bf16", "16bit", 3, 1023, 2049, 0, 2100, 32, 8, 128, 64, 0, 0),
        # one row of logits with the usual top-k and top-p
        _sample("sample_one", "f16", 1, 128256, 50, 0.9, 0.0),
        # a large batch without top-k: the nucleus of a wide vocabulary, fp32 logits
        _sample("sample_batch_nucleus", "f32", 128, 202048, 0, 0.95, 0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        dtype = rng.choice(["f16", "bf16", "f32"])
        vocab = _log(rng, 500, 202048)
        rows = _log(rng, 1, max(1, min(256, 25_000_000 // vocab)))
        c = _sample("", dtype, rows, vocab, rng.choice([0, 0, _log(rng, 1, 2000)]), rng.choice([1.0, 0.5, 0.9, 0.99]),
                    rng.choice([0.0, 0.0, 0.05, 0.3]))
    else:
        heads, kv_heads = rng.choice([(32, 8), (64, 8), (40, 8), (8, 8), (16, 2), (6, 1), (32, 32)])
        dim = rng.choice([64, 128, 128])
        dtype, kv = rng.choice(["f16", "bf16"]), rng.choice(["16bit", "e4m3"])
        page = rng.choice([16, 32, 64, 128])
        if op == "append":
            if rng.random() < 0.5:
                batch = _log(rng, 1, 200)
                new_lo = new_hi = 1
                ctx_hi = _log(rng, 10, 3000)
            else:
                batch = _log(rng, 1, 12)
                new_hi = _log(rng, 2, max(3, 9000 // batch))
                new_lo = max(1, new_hi // 3)
                ctx_hi = _log(rng, 1, 1500)
            c = _append("", dtype, kv, batch, new_lo, new_hi, ctx_hi // 5, ctx_hi, heads, kv_heads, dim, page,
                        rng.choice([dim, dim, dim // 2, dim // 4]), rng.random() < 0.4)
        else:
            window = rng.choice([0, 0, _log(rng, 1, 6000)])
            sinks = rng.choice([0, 4, _log(rng, 1, 100)]) if window else 0
            if rng.random() < 0.65:
                batch = _log(rng, 1, 64)
                new_lo = new_hi = 1
                ctx_hi = _log(rng, 1, max(2, 2_000_000 // (batch * kv_heads * (dim // 64))))
            else:
                batch = _log(rng, 1, 6)
                new_hi = _log(rng, 2, max(3, 3600 // batch))
                new_lo = max(1, new_hi // 2)
                ctx_hi = _log(rng, 1, max(2, 3000 // batch))
            c = _attend("", dtype, kv, batch, new_lo, new_hi, ctx_hi // 4, ctx_hi, heads, kv_heads, dim, page, window,
                        sinks)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, in a mixed order; the last one is hi."""
    return [hi if n == 1 or i == n - 1 else lo + (hi - lo) * ((i * 37 + 11) % n) // n for i in range(n)]


def _lengths(case):
    """(cached tokens, new tokens) of each sequence."""
    n = case["batch"]
    return _spread(case["ctx_lo"], case["ctx_hi"], n), _spread(case["new_lo"], case["new_hi"], n)[::-1]


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 2 * case["rows"] * case["vocab"]}
    ctx, new = _lengths(case)
    total, D = sum(new), case["dim"]
    kv_size = 1 if case["kv"] == "e4m3" else 2
    pages = sum((c + n - 1) // case["page"] - c // case["page"] + 1 for c, n in zip(ctx, new))
    scales = 2 * 4 * pages * case["kv_heads"] if case["kv"] == "e4m3" else 0
    if case["op"] == "append":
        moved = total * D * ((case["heads"] + 2 * case["kv_heads"]) * 2 + case["heads"] * 2 + 2 * case["kv_heads"] * kv_size)
        table = 8 * (case["rotary"] // 2) * len({c + i for c, n in zip(ctx, new) for i in range(n)})
        return {"bytes": moved + table + 2 * scales,
                "flops": 3 * total * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    seen, pairs = 0, 0
    W, S = case["window"], case["sinks"]
    for c, n in zip(ctx, new):
        first = max(0, c - W + 1) if W else 0  # first token inside the window of the first new one
        seen += c + n - first + min(S, first)
        for p in range(c, c + n):
            lo = max(0, p - W + 1) if W else 0
            pairs += p + 1 - lo + min(S, lo)
    moved = seen * case["kv_heads"] * D * 2 * kv_size + 2 * total * case["heads"] * D * 2
    if scales:
        moved += 2 * 4 * case["kv_heads"] * (seen // case["page"])
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * D}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _page_scale(amax):
    """The smallest power of two s with amax <= 448 s (2^-100 at least)."""
    m, e = torch.frexp(amax)  # amax = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(min=-100)
    return torch.ldexp(torch.ones_like(amax), e)


def _pages(g, num_pages, case):
    """One pool of pages as (pages, scales): keys and values with channels of different size."""
    shape = (num_pages, case["kv_heads"], case["page"], case["dim"])
    size = torch.exp(0.5 * torch.randn(1, case["kv_heads"], 1, case["dim"], device=DEV, generator=g))
    dt = DT[case["dtype"]]
    x = torch.empty(shape, dtype=dt, device=DEV)
    x.normal_(generator=g).mul_(size.to(dt))
    if case["kv"] != "e4m3":
        return x, None
    scales = _page_scale(x.abs().amax(dim=(2, 3)).float())
    return (x / scales.to(dt)[:, :, None, None]).to(E4M3), scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)
    s = {"op": case["op"], "case": dict(case)}
    if case["op"] == "sample":
        rows, V = case["rows"], case["vocab"]
        x = torch.empty(rows, V, dtype=torch.float32, device=DEV).normal_(generator=g).mul_(2.2)
        # a language model's rows: a few likely tokens above the bulk, more or less of them from row to row
        top = torch.randint(0, V, (rows, 40), device=DEV, generator=g)
        x.scatter_add_(1, top, 9.0 * torch.rand(rows, 40, device=DEV, generator=g))
        s["logits"] = x.to(DT[case["dtype"]])
        s["uniforms"] = torch.rand(rows, device=DEV, generator=g)
        s["temperature"] = 0.5 + torch.rand(rows, device=DEV, generator=g)
        if rows > 4:
            s["temperature"][rows // 2] = 0.0  # one greedy user in the batch
        vary = 0.5 + torch.rand(3, rows, device=DEV, generator=g)
        s["top_k"] = (case["top_k"] * vary[0]).ceil().to(torch.int32) if case["top_k"] else None
        s["top_p"] = (case["top_p"] ** vary[1]) if case["top_p"] < 1 else None
        s["min_p"] = (case["min_p"] * vary[2]) if case["min_p"] > 0 else None
        return s
    ctx, new = _lengths(case)
    page, D, dt = case["page"], case["dim"], DT[case["dtype"]]
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    num_pages = sum(need) + 3
    order = torch.randperm(num_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    order_host, at = order.cpu(), 0
    for b, n in enumerate(need):
        table[b, :n] = order_host[at: at + n]
        at += n
    s["block_table"] = table.to(DEV)
    s["context_lens"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["total"], s["max_new"], s["max_context"] = cu[-1], max(new), max(c + n for c, n in zip(ctx, new))
    s["cu_tokens"] = None if max(new) == 1 else torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["k_pages"], s["k_scales"] = _pages(g, num_pages, case)
    s["v_pages"], s["v_scales"] = _pages(g, num_pages, case)
    H, Hkv = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        # the packed projection of the new tokens; q, k and v are views of it
        qkv = torch.empty(s["total"], H + 2 * Hkv, D, dtype=dt, device=DEV).normal_(generator=g)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H: H + Hkv], qkv[:, H + Hkv:]
        half = case["rotary"] // 2
        inv = 500000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        angle = torch.arange(s["max_context"], device=DEV, dtype=torch.float64)[:, None] * inv
        s["freqs"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
    else:
        s["q"] = torch.empty(s["total"], H, D, dtype=dt, device=DEV).normal_(generator=g).mul_(1.5)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from muillm_b200 import ops
        if s["op"] == "append":
            q_out = ops.paged_kv_append(s["k_pages"], s["v_pages"], s["block_table"], s["context_lens"], s["q"], s["k"],
                                        s["v"], freqs=s["freqs"], cu_tokens=s["cu_tokens"], rotary_dim=c["rotary"],
                                        interleaved=c["interleaved"], k_scales=s["k_scales"], v_scales=s["v_scales"])
            return [q_out, s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]
        if s["op"] == "attend":
            return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["context_lens"],
                                       cu_tokens=s["cu_tokens"], max_new_tokens=s["max_new"],
                                       max_context=s["max_context"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                                       window=c["window"], sinks=c["sinks"])
        return list(ops.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"]))
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    return _plain_sample(s)


def _owners(s):
    """(sequence, place among its new tokens) of each new token."""
    n = torch.arange(s["total"], device=DEV)
    if s["cu_tokens"] is None:
        return n, torch.zeros_like(n)
    seq = torch.searchsorted(s["cu_tokens"][1:].long(), n, right=True)
    return seq, n - s["cu_tokens"].long()[seq]


def _plain_rotate(x, cs, rotary, interleaved):
    """x [total, heads, dim] in fp32; the first `rotary` elements of each head turned by cs [total, rotary/2, 2]."""
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    r = x[..., :rotary]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = r[..., : rotary // 2], r[..., rotary // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rotary:]], dim=-1)


def _plain_store(pages, scales, x, s, seq, pos):
    """Writes rows x [total, kv heads, dim] (fp32) at their positions."""
    ps = s["case"]["page"]
    page = s["block_table"].long()[seq, pos // ps]
    slot = pos % ps
    if scales is None:
        pages[page, :, slot] = x.to(pages.dtype)
        return
    heads = torch.arange(pages.shape[1], device=DEV)
    amax = torch.zeros_like(scales)
    amax.index_reduce_(0, page, x.abs().amax(dim=2), "amax")
    need = _page_scale(amax)
    written = torch.zeros(pages.shape[0], dtype=torch.bool, device=DEV)
    written[page] = True
    ctx = s["context_lens"].long()
    # a page whose rows before the new ones count keeps at least its scale, and those rows are rescaled
    seqs = torch.arange(ctx.shape[0], device=DEV)
    old_rows = ctx % ps
    last = s["block_table"].long()[seqs, (ctx // ps).clamp(max=s["block_table"].shape[1] - 1)].clamp(min=0)
    partial = (old_rows > 0) & written[last]
    held = torch.zeros_like(scales)
    held[last] = torch.where(partial[:, None], scales[last], held[last])
    new = torch.where(written[:, None], torch.maximum(need, held), scales)
    ratio = torch.where(partial[:, None], scales[last] / new[last], torch.ones_like(scales[last]))
    rows = pages[last]
    keep = (torch.arange(ps, device=DEV) < old_rows[:, None]) & partial[:, None]
    pages[last] = torch.where(keep[:, None, :, None], (rows.float() * ratio[:, :, None, None]).to(E4M3).float(),
                              rows.float()).to(E4M3)
    pages[page[:, None], heads[None, :], slot[:, None]] = (x / new[page][:, :, None]).to(E4M3)
    scales.copy_(new)


def _plain_append(s):
    c = s["case"]
    seq, i = _owners(s)
    pos = s["context_lens"].long()[seq] + i
    cs = s["freqs"][pos]
    q = _plain_rotate(s["q"].float(), cs, c["rotary"], c["interleaved"]).to(s["q"].dtype)
    _plain_store(s["k_pages"], s["k_scales"], _plain_rotate(s["k"].float(), cs, c["rotary"], c["interleaved"]), s, seq, pos)
    _plain_store(s["v_pages"], s["v_scales"], s["v"].float(), s, seq, pos)
    return [q, s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]


def _plain_gather(pages, scales, table, length):
    """[sequences, kv heads, length, dim] in fp32."""
    x = pages[table].float()  # [sequences, pages, kv heads, page, dim]
    if scales is not None:
        x = x * scales[table][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :length]


def _plain_attend(s):
    c = s["case"]
    H, Hkv, D = c["heads"], c["kv_heads"], c["dim"]
    B, T, L = s["context_lens"].shape[0], s["max_new"], s["max_context"]
    seq, i = _owners(s)
    q = torch.zeros(B, T, H, D, dtype=torch.float32, device=DEV)
    q[seq, i] = s["q"].float()
    table = s["block_table"].long().clamp(min=0)
    k = _plain_gather(s["k_pages"], s["k_scales"], table, L)
    v = _plain_gather(s["v_pages"], s["v_scales"], table, L)
    q = q.view(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, (H // Hkv) * T, D)
    a = (q @ k.transpose(2, 3)).view(B, Hkv, H // Hkv, T, L) / math.sqrt(D)
    p = s["context_lens"].long()[:, None, None] + torch.arange(T, device=DEV)[None, :, None]
    j = torch.arange(L, device=DEV)[None, None, :]
    seen = j <= p
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
    a = a.masked_fill_(~seen[:, None, None], float("-inf"))
    a = torch.exp_(a.sub_(a.amax(dim=-1, keepdim=True)))
    a = a.div_(a.sum(dim=-1, keepdim=True))
    o = (a.view(B, Hkv, -1, L) @ v).view(B, Hkv, H // Hkv, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    return o[seq, i].to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    rows, V = x.shape
    z, order = torch.sort(x, dim=1, descending=True, stable=True)  # rank: by value, then by index
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    z = (z - z[:, :1]) / torch.where(greedy, torch.ones_like(t), t)
    w = torch.exp(z)
    rank = torch.arange(V, device=DEV)[None, :]
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        keep = rank < s["top_k"].long()[:, None]
    if s["top_p"] is not None:
        upto = torch.cumsum(w * keep, dim=1)
        keep = keep & ((upto - w < s["top_p"].double()[:, None] * upto[:, -1:]) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    keep = torch.where(greedy, rank == 0, keep)
    w = w * keep
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    upto = torch.cumsum(by_index, dim=1)
    token = (upto <= s["uniforms"].double()[:, None] * upto[:, -1:]).sum(dim=1)
    picked = by_index.gather(1, token[:, None])[:, 0]
    return [token, torch.log(picked / upto[:, -1]).float()]


# ---------------------------------------------------------------------------------------------------------------------
# the operators' values in 64 bits, sequence by sequence and row by row
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    ctx, new = _lengths(case)
    if case["op"] == "append":
        return _exact_append(s, case, ctx, new)
    out, at = [], 0
    table = s["block_table"].cpu().tolist()
    G, D, W, S = case["heads"] // case["kv_heads"], case["dim"], case["window"], case["sinks"]
    for b, (c, n) in enumerate(zip(ctx, new)):
        L = c + n
        ids = torch.tensor(table[b][: -(-L // case["page"])], device=DEV)
        heads = []
        for h in range(case["kv_heads"]):
            k, v = s["k_pages"][ids, h].double(), s["v_pages"][ids, h].double()
            if s["k_scales"] is not None:
                k = k * s["k_scales"][ids, h].double()[:, None, None]
                v = v * s["v_scales"][ids, h].double()[:, None, None]
            k, v = k.reshape(-1, D)[:L], v.reshape(-1, D)[:L]
            q = s["q"][at: at + n, h * G: (h + 1) * G].double()
            a = torch.einsum("tgd,ld->gtl", q, k) * D ** -0.5
            far = torch.arange(c, L, device=DEV)[:, None] - torch.arange(L, device=DEV)[None, :]
            hidden = far < 0
            if W:
                hidden = hidden | ((far >= W) & (torch.arange(L, device=DEV)[None, :] >= S))
            a[:, hidden] = -math.inf
            heads.append(torch.einsum("gtl,ld->tgd", torch.softmax(a, dim=-1), v))
        out.append(torch.cat(heads, dim=1))
        at += n
    return torch.cat(out)


def _exact_append(s, case, ctx, new):
    half, ps = case["rotary"] // 2, case["page"]
    table = s["block_table"].cpu().tolist()

    def turned(x, pos):
        z = torch.view_as_complex(s["freqs"][pos].double())[:, None]
        x = x.double().clone()
        if case["interleaved"]:
            y = torch.view_as_complex(x[..., : 2 * half].reshape(*x.shape[:2], half, 2).contiguous()) * z
            x[..., : 2 * half] = torch.view_as_real(y).flatten(-2)
        else:
            y = torch.complex(x[..., :half], x[..., half: 2 * half]) * z
            x[..., :half], x[..., half: 2 * half] = y.real, y.imag
        return x

    pos = torch.tensor([c + i for c, n in zip(ctx, new) for i in range(n)], device=DEV)
    outs = [turned(s["q"], pos)]
    pools, scales = [], []
    for name, x in (("k", turned(s["k"], pos)), ("v", s["v"].double())):
        pool = s[name + "_pages"].double()
        scale = None if s[name + "_scales"] is None else s[name + "_scales"].double()
        at = 0
        for b, (c, n) in enumerate(zip(ctx, new)):
            for first in range(c // ps * ps, c + n, ps):
                lo, hi = max(first, c), min(first + ps, c + n)
                rows, p = x[at + lo - c: at + hi - c], table[b][first // ps]
                rows = rows.transpose(0, 1)
                if scale is not None:
                    top = rows.abs().amax(dim=(1, 2)).clamp(min=2.0 ** -100)
                    fit = torch.exp2(torch.ceil(torch.log2(top / 448.0)))
                    if lo > first:
                        fit = torch.maximum(fit, scale[p])
                        pool[p, :, : lo - first] *= (scale[p] / fit)[:, None, None]
                    scale[p] = fit
                    rows = rows / fit[:, None, None]
                pool[p, :, lo - first: hi - first] = rows
            at += n
        pools.append(pool)
        scales.append(scale)
    return outs + pools + scales


def _exact_sample(s):
    tokens, logs = [], []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        if t <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            logs.append(0.0)
            continue
        p = torch.softmax(x / t, dim=0)
        k = int(s["top_k"][r]) if s["top_k"] is not None else x.numel()
        # by value, ties by index: all above the k-th value, then the first ones at it
        val, idx = torch.sort(x, descending=True, stable=True)
        idx = idx[:k]
        q = p[idx] / p[idx].sum()
        if s["top_p"] is not None:
            before = torch.cumsum(q, 0) - q
            n = max(1, int((before < float(s["top_p"][r].double())).sum()))
            idx = idx[:n]
        if s["min_p"] is not None:
            idx = idx[p[idx] >= float(s["min_p"][r].double()) * p.max()]
        idx = torch.sort(idx).values
        q = torch.cumsum(p[idx], 0)
        at = int((q <= float(s["uniforms"][r].double()) * q[-1]).sum())
        tokens.append(int(idx[at]))
        logs.append(math.log(float(p[idx[at]] / q[-1])))
    return [torch.tensor(tokens, device=DEV), torch.tensor(logs, dtype=torch.float64, device=DEV)]
