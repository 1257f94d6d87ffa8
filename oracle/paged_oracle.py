"""64-bit restatement of the paged-cache operators and of token sampling, sequence by sequence and row by row, on the CPU
(test infrastructure)."""
import math

import torch


def rotary_table(positions, rotary_dim, theta=10000.0):
    """[positions, rotary_dim / 2, 2] fp32 (cos, sin)."""
    half = rotary_dim // 2
    inv = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], dim=-1).float()


def rotate(x, cs, interleaved):
    """x [..., D] with table row cs [rotary_dim / 2, 2] (or None), in fp64. Returns (rotated, sum of the magnitudes)."""
    x = x.double().clone()
    mag = x.abs()
    if cs is None:
        return x, mag
    half = cs.shape[0]
    c, s = cs[:, 0].double(), cs[:, 1].double()
    sl = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., sl[0]].clone(), x[..., sl[1]].clone()
    x[..., sl[0]], x[..., sl[1]] = a * c - b * s, b * c + a * s
    mag[..., sl[0]] = mag[..., sl[1]] = a.abs() + b.abs()
    return x, mag


def page_scale(amax):
    """Smallest power of two s >= 2^-100 with amax <= 448 s."""
    if amax == 0:
        return 2.0 ** -100
    m, e = math.frexp(amax / 448.0)
    return 2.0 ** max(-100, e - 1 if m == 0.5 else e)


def positions(ctx, new, position_ids=None):
    flat = [c + i for c, n in zip(ctx, new) for i in range(n)]
    return flat if position_ids is None else [int(p) for p in position_ids]


def append(k_pages, v_pages, k_scales, v_scales, table, ctx, new, k, v, freqs, interleaved, position_ids=None):
    """Expected cache: per pool (values fp64 [pages, heads, page, D], tolerance of the same shape, scales fp64 or None,
    written-or-rescaled mask [pages, heads, page]). Pages and scales are the state before the call."""
    ps = k_pages.shape[2]
    pos = positions(ctx, new, position_ids)
    out = []
    for which, pages, scales, x in (("k", k_pages, k_scales, k), ("v", v_pages, v_scales, v)):
        e4m3 = scales is not None
        step = 2.0 ** -4 if e4m3 else torch.finfo(pages.dtype).eps / 2
        val = pages.to(torch.float32).double()
        sc = scales.double().clone() if e4m3 else None
        if e4m3:
            val = val * sc[:, :, None, None]
        tol = torch.zeros_like(val)
        touched = torch.zeros(val.shape[:3], dtype=torch.bool)
        at = 0
        for b, (c, n) in enumerate(zip(ctx, new)):
            for first in range(c // ps * ps, c + n, ps):
                if n == 0:
                    continue
                lo, hi = max(first, c), min(first + ps, c + n)
                p = int(table[b][first // ps])
                rows = list(range(at + lo - c, at + hi - c))
                y = torch.stack([rotate(x[r], freqs[pos[r]] if freqs is not None and which == "k" else None, interleaved)[0]
                                 for r in rows], dim=1)  # [heads, rows, D]
                mag = torch.stack([rotate(x[r], freqs[pos[r]] if freqs is not None and which == "k" else None,
                                          interleaved)[1] for r in rows], dim=1)
                t = y.abs() * step + mag * 2.0 ** -22
                if e4m3:
                    for h in range(y.shape[0]):
                        finite = y[h][torch.isfinite(y[h])]
                        s = page_scale(float(finite.abs().max()) if finite.numel() else 0.0)
                        if lo > first:
                            old = float(sc[p, h])
                            s = max(s, old)
                            if s > old:
                                # rescaling rounds again only where the result is an e4m3 subnormal
                                tol[p, h, : lo - first] = s * 2.0 ** -10
                                touched[p, h, : lo - first] = True
                        sc[p, h] = s
                        t[h] += s * 2.0 ** -10
                        y[h] = y[h].clamp(-448 * s, 448 * s)
                else:
                    t += 2.0 ** -25  # half a step of fp16 subnormals
                val[p, :, lo - first: hi - first] = y
                tol[p, :, lo - first: hi - first] = t
                touched[p, :, lo - first: hi - first] = True
            at += n
        out.append((val, tol, sc, touched))
    return out


def visible(c, n, window, sinks):
    """[new, cached + new] bool."""
    p = torch.arange(c, c + n)[:, None]
    j = torch.arange(c + n)[None, :]
    see = j <= p
    if window:
        see = see & ((j > p - window) | (j < sinks))
    return see


def attention(q, k_pages, v_pages, k_scales, v_scales, table, ctx, new, window=0, sinks=0, scale=None, row_by_row=False):
    """(out fp64 [total, Hq, D], sum of p |v| of the same shape). Rows that nobody sees may hold anything. What a token does
    not see has weight 0, or, row_by_row, is left out of its sums, so that infinities there do not matter either."""
    total, Hq, D = q.shape
    Hkv, ps = k_pages.shape[1:3]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(total, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    at = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        L = c + n
        see = visible(c, n, window, sinks)
        rows = [j for j in range(L) if bool(see[:, j].any())]
        ids = torch.tensor([int(table[b][j // ps]) for j in rows])
        slots = torch.tensor([j % ps for j in rows])
        kk = k_pages[ids, :, slots].to(torch.float32).double()
        vv = v_pages[ids, :, slots].to(torch.float32).double()
        if k_scales is not None:
            kk = kk * k_scales[ids].double()[:, :, None]
            vv = vv * v_scales[ids].double()[:, :, None]
        for h in range(Hkv):
            a = torch.einsum("tgd,ld->gtl", q[at: at + n, h * G: (h + 1) * G].double(), kk[:, h]) * scale
            a = a.masked_fill(~see[:, rows][None], -math.inf)
            w = torch.softmax(a, dim=-1)
            if row_by_row:
                for t in range(n):
                    seen = see[t, rows]
                    for res, val in ((out, vv[:, h]), (mag, vv[:, h].abs())):
                        res[at + t, h * G: (h + 1) * G] = torch.einsum("gl,ld->gd", w[:, t, seen], val[seen])
                continue
            out[at: at + n, h * G: (h + 1) * G] = torch.einsum("gtl,ld->tgd", w, vv[:, h])
            mag[at: at + n, h * G: (h + 1) * G] = torch.einsum("gtl,ld->tgd", w, vv[:, h].abs())
        at += n
    return out, mag


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(token, log share of the kept weight, kept tokens) of one row (a 1-D tensor and numbers), in fp64."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.max()
    if top == -math.inf:
        return 0, -math.inf, [0]
    best = int((x == top).nonzero()[0])
    t = 1.0 if temperature is None else temperature
    if not t > 0:
        return best, 0.0, [best]
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / t))
    w = torch.where(x == -math.inf, torch.zeros_like(w), w)
    order = torch.sort(x, descending=True, stable=True).indices
    if top_k is not None and top_k > 0:
        order = order[:top_k]
    if top_p is not None and top_p < 1:
        before = torch.cumsum(w[order], 0) - w[order]
        order = order[: max(1, int((before < top_p * w[order].sum()).sum()))]
    if min_p is not None and min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    kept = torch.sort(order[w[order] > 0]).values
    run = torch.cumsum(w[kept], 0)
    at = int((run <= u * run[-1]).sum())
    return int(kept[at]), math.log(float(w[kept[at]] / run[-1])), kept.tolist()
