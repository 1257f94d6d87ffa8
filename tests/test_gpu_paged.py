"""Paged-cache append, attention over 16-bit and e4m3 pages (windows, sinks, prompts) and token sampling against the
64-bit oracle."""
import itertools
import math

import pytest
import torch

from muillm_b200 import capi, ops
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    """A pool of pages with a random block table, filled rows, and poison (NaN) in every row that no sequence holds."""

    def __init__(self, ctx, new, Hkv, D, page, dtype, e4m3, seed, spread=1.0, spare=2, poison=True):
        g = _gen(seed)
        need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
        self.num_pages = sum(need) + spare
        ids = torch.randperm(self.num_pages, generator=g).tolist()
        self.table = torch.full((len(ctx), max(need + [1]) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                self.table[b, i] = ids.pop()
        shape = (self.num_pages, Hkv, page, D)
        self.pools, self.scales = [], []
        for _ in range(2):
            x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(self.num_pages, Hkv, 1, 1, generator=g))
            held = torch.zeros(self.num_pages, page, dtype=torch.bool)
            for b, c in enumerate(ctx):
                for j in range(c):
                    held[int(self.table[b, j // page]), j % page] = True
            if e4m3:
                s = torch.tensor([[oracle.page_scale(float((x[p, h] * held[p][:, None]).abs().max())) for h in range(Hkv)]
                                  for p in range(self.num_pages)], dtype=torch.float32)
                y = (x / s[:, :, None, None]).clamp(-448, 448).to(E4M3)
                if poison:
                    y.view(torch.uint8).masked_fill_(~held[:, None, :, None], 0x7F)
                    empty = ~held.any(dim=1)
                    s[empty] = math.nan
                self.scales.append(s)
            else:
                y = x.to(dtype)
                if poison:
                    y.masked_fill_(~held[:, None, :, None], math.nan)
            self.pools.append(y)
        self.e4m3 = e4m3
        self.ctx, self.new = ctx, new
        self.cu = [0] + list(itertools.accumulate(new))

    def cuda(self):
        d = dict(k_pages=self.pools[0].cuda(), v_pages=self.pools[1].cuda(), block_table=self.table.cuda(),
                 context_lens=_i32(self.ctx))
        if self.e4m3:
            d.update(k_scales=self.scales[0].cuda(), v_scales=self.scales[1].cuda())
        if any(n != 1 for n in self.new):
            d["cu_tokens"] = _i32(self.cu)
        return d

    def oracle_args(self):
        s = self.scales if self.e4m3 else [None, None]
        return self.pools[0], self.pools[1], s[0], s[1]


def _within(got, want, tol):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err - tol).max())} over its bound"


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def _check_append(c, q, k, v, freqs, interleaved, position_ids=None, strided=None):
    d = c.cuda()
    want = oracle.append(*c.oracle_args(), c.table, c.ctx, c.new, k, v, freqs, interleaved, position_ids)
    gq, gk, gv = strided if strided is not None else (q.cuda(), k.cuda(), v.cuda())
    out = ops.paged_kv_append(d["k_pages"], d["v_pages"], d["block_table"], d["context_lens"], gq, gk, gv,
                              freqs=None if freqs is None else freqs.cuda(), cu_tokens=d.get("cu_tokens"),
                              interleaved=interleaved, k_scales=d.get("k_scales"), v_scales=d.get("v_scales"),
                              position_ids=None if position_ids is None else position_ids.cuda())
    if q is not None:
        pos = oracle.positions(c.ctx, c.new, position_ids)
        for t, p in enumerate(pos):
            y, mag = oracle.rotate(q[t], None if freqs is None else freqs[p], interleaved)
            _within(out[t], y, y.abs() * torch.finfo(q.dtype).eps / 2 + mag * 2.0 ** -22 + 2.0 ** -25)
    for name, (val, tol, sc, touched), before in zip("kv", want, c.pools):
        got = d[name + "_pages"].cpu()
        if c.e4m3:
            gs = d[name + "_scales"].cpu()
            assert torch.equal(gs.double().nan_to_num(-1.0), sc.nan_to_num(-1.0))
            raw, raw_before = got.view(torch.uint8), before.view(torch.uint8)
            got = got.float().double() * gs.double()[:, :, None, None]
        else:
            raw, raw_before = got.view(torch.int16), before.view(torch.int16)
        assert torch.equal(raw[~touched], raw_before[~touched]), "a row that the call does not own changed"
        _within(got[touched], val[touched], tol[touched])
    return d, out


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page,rotary,interleaved", [
    ([0], [1], 4, 2, 128, 16, 128, False),                          # the first token of all
    ([15, 16, 17, 300], [1, 1, 1, 1], 8, 8, 64, 16, 64, False),     # page borders, no grouping
    ([5, 0, 31], [1, 40, 3], 6, 2, 128, 32, 64, True),              # ragged, part of the head, interleaved
    ([0, 7, 64, 100], [64, 57, 1, 0], 5, 1, 128, 64, 32, False),    # exact pages; a sequence without new tokens
    ([130, 3], [129, 126], 4, 4, 64, 128, 20, False),               # odd quarter of the head: no 16-byte partners
    ([10, 200], [150, 1], 3, 1, 128, 128, 6, True),
    ([9, 1], [17, 2], 2, 2, 64, 16, 0, False),                      # no rotation at all
])
def test_append(dtype, e4m3, ctx, new, Hq, Hkv, D, page, rotary, interleaved):
    g = _gen(sum(ctx) + 3 * sum(new))
    c = Cache(ctx, new, Hkv, D, page, dtype, e4m3, seed=1)
    total = sum(new)
    q, k, v = (torch.randn(total, h, D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
    k, v = (x * torch.exp(torch.randn(total, 1, 1, generator=g)).to(dtype) for x in (k, v))
    freqs = oracle.rotary_table(max(a + b for a, b in zip(ctx, new)), rotary) if rotary else None
    _check_append(c, q, k, v, freqs, interleaved)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_append_strided_views(e4m3, offset):
    """q, k, v as slices of a packed projection; with an odd offset their rows are not 16-byte aligned."""
    ctx, new, Hq, Hkv, D = [3, 40], [20, 2], 4, 2, 64
    g = _gen(5)
    c = Cache(ctx, new, Hkv, D, 16, BF16, e4m3, seed=2)
    width = (Hq + 2 * Hkv) * D
    buf = torch.randn(sum(new), width + 3, generator=g).to(BF16)
    gb = buf.cuda()

    def views(t):
        t = t[:, offset: offset + width]
        return [x.unflatten(1, (-1, D)) for x in (t[:, : Hq * D], t[:, Hq * D: (Hq + Hkv) * D], t[:, (Hq + Hkv) * D:])]

    q, k, v = views(buf)
    _check_append(c, q, k, v, oracle.rotary_table(64, D), False, strided=views(gb))


@pytest.mark.parametrize("e4m3", [False, True])
def test_append_position_ids_and_no_q(e4m3):
    ctx, new = [4, 9], [2, 3]
    g = _gen(6)
    c = Cache(ctx, new, 2, 128, 16, F16, e4m3, seed=3)
    k, v = (torch.randn(5, 2, 128, generator=g).to(F16) for _ in range(2))
    pos = torch.tensor([0, 49, 7, 7, 1], dtype=torch.int64)
    _check_append(c, None, k, v, oracle.rotary_table(50, 128), False, position_ids=pos, strided=(None, k.cuda(), v.cuda()))


def test_append_padding_rows_are_left():
    """Rows behind the last sequence are neither read nor written."""
    ctx, new, pad = [4, 9], [2, 3], 6
    for e4m3 in (False, True):
        c = Cache(ctx, new, 2, 128, 16, F16, e4m3, seed=4)
        d = c.cuda()
        before = d["k_pages"].view(torch.uint8).clone()
        q, k, v = (torch.full((5 + pad, h, 128), math.nan, dtype=F16) for h in (4, 2, 2))
        for x in (q, k, v):
            x[:5] = torch.randn(x[:5].shape, generator=_gen(7))
        q_out = torch.full((5 + pad, 4, 128), 7.0, dtype=F16, device="cuda")
        ops.paged_kv_append(d["k_pages"], d["v_pages"], d["block_table"], d["context_lens"], q.cuda(), k.cuda(), v.cuda(),
                            cu_tokens=d["cu_tokens"], k_scales=d.get("k_scales"), v_scales=d.get("v_scales"), q_out=q_out)
        assert torch.equal(q_out[:5].cpu(), q[:5]) and (q_out[5:] == 7.0).all()
        changed = (d["k_pages"].view(torch.uint8) != before).flatten(2).any(dim=2).any(dim=1).sum()
        assert int(changed) <= 2  # the pages of the two sequences
        out = ops.paged_attention(torch.zeros_like(q_out), d["k_pages"], d["v_pages"], d["block_table"], d["context_lens"],
                                  cu_tokens=d["cu_tokens"], max_new_tokens=3, k_scales=d.get("k_scales"),
                                  v_scales=d.get("v_scales"), out=q_out)
        assert torch.isfinite(out[:5]).all() and (out[5:] == 7.0).all()


def test_append_scale_growth_and_reuse():
    """One page filled token by token: its scale never shrinks and its rows keep their values; a page that starts again
    at row 0 forgets the old scale. Infinities saturate and do not count; NaN stays."""
    D, page = 64, 16
    kp = torch.full((2, 1, page, D), 0x7F, dtype=torch.uint8, device="cuda").view(E4M3)
    vp = kp.clone()
    ks = torch.full((2, 1), math.nan, device="cuda")
    vs = ks.clone()
    table = _i32([[1]])
    g = _gen(8)
    rows = torch.randn(page, 1, D, generator=g) * torch.tensor([2.0 ** (i - 4) for i in range(page)])[:, None, None]
    rows = rows.to(BF16)
    for i in range(page):
        ops.paged_kv_append(kp, vp, table, _i32([i]), None, rows[i:i + 1].cuda(), rows[i:i + 1].cuda(), k_scales=ks,
                            v_scales=vs)
        s = oracle.page_scale(float(rows[: i + 1].abs().max()))
        assert float(ks[1, 0]) == s and float(vs[1, 0]) == s
        got = kp[1, 0, : i + 1].float().cpu().double() * s
        want = rows[: i + 1, 0].double()
        # each value: one rounding at its own scale, then up to i roundings into subnormals of ever larger steps (each
        # at most half a step, the steps double: twice the last half step together)
        _within(got, want, want.abs() * 2.0 ** -4 + 2 * s * 2.0 ** -10)
    assert float(ks[0, 0]) != float(ks[0, 0])  # the other page is as it was
    small = (rows[0] * 2.0 ** -6).reshape(1, 1, D).clone()
    small[0, 0, 3], small[0, 0, 4], small[0, 0, 5] = math.inf, -math.inf, math.nan
    ops.paged_kv_append(kp, vp, table, _i32([0]), None, small.cuda(), small.cuda(), k_scales=ks, v_scales=vs)
    finite = small[torch.isfinite(small)]
    s = oracle.page_scale(float(finite.abs().max()))
    assert float(ks[1, 0]) == s
    first = kp[1, 0, 0].float().cpu()
    assert first[3] == 448 and first[4] == -448 and first[5] != first[5]


def test_append_zero_rows():
    """A page of zeros has the smallest scale, and the first row that is not zero sets it."""
    kp = torch.zeros(1, 1, 16, 64, dtype=torch.uint8, device="cuda").view(E4M3)
    vp, ks = kp.clone(), torch.zeros(1, 1, device="cuda")
    vs = ks.clone()
    table = _i32([[0]])
    z = torch.zeros(1, 1, 64, dtype=F16, device="cuda")
    ops.paged_kv_append(kp, vp, table, _i32([0]), None, z, z, k_scales=ks, v_scales=vs)
    assert float(ks) == 2.0 ** -100 and (kp.float() == 0).all()
    x = torch.linspace(-3, 3, 64).to(F16).reshape(1, 1, 64).cuda()
    ops.paged_kv_append(kp, vp, table, _i32([1]), None, x, x, k_scales=ks, v_scales=vs)
    assert float(ks) == 2.0 ** -7
    assert (kp[0, 0, 0].float() == 0).all()
    _within(kp[0, 0, 1].float() * 2.0 ** -7, x[0, 0].double().cpu(), x[0, 0].double().cpu().abs() * 2.0 ** -4 + 2.0 ** -17)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def _attention_tolerance(dtype, e4m3, prompt, want, mag):
    """Half a step of the result's type; probabilities rounded to the tensor cores' type (fp16 for fp16 and e4m3 pages,
    bf16 for prompts over bf16 pages, bf16 value + bf16 rest else) times sum p |v|; scores in fp32, off by at most 128
    products * 2^-24 * sum |q k| scale (about 11 here), which moves a probability by as much."""
    p = 2.0 ** -11 if dtype == F16 or e4m3 else (2.0 ** -8 if prompt else 2.0 ** -16)
    return want.abs() * torch.finfo(dtype).eps / 2 + mag * (p + 2.0 ** -13) + 2.0 ** -24


def _check_attention(c, q, window=0, sinks=0, scale=None, max_context=None, max_new=None):
    d = c.cuda()
    want, mag = oracle.attention(q, *c.oracle_args(), c.table, c.ctx, c.new, window, sinks, scale)
    max_new = max_new or max(c.new)
    got = ops.paged_attention(q.cuda(), max_new_tokens=max_new, window=window, sinks=sinks, scale=scale,
                              max_context=max_context, **d)
    prompt = max_new * (q.shape[1] // c.pools[0].shape[1]) > 32
    _within(got, want, _attention_tolerance(q.dtype, c.e4m3, prompt, want, mag))
    return got


def _filled(ctx, new, Hkv, D, page, dtype, e4m3, seed, **kw):
    """A cache that holds the new rows already, described as before the append."""
    c = Cache([a + b for a, b in zip(ctx, new)], [0] * len(ctx), Hkv, D, page, dtype, e4m3, seed, **kw)
    c.ctx, c.new = ctx, new
    c.cu = [0] + list(itertools.accumulate(new))
    return c


SHAPES = [
    # ctx, new, Hq, Hkv, D, page
    ([0], [1], 8, 2, 128, 16),                                   # only itself
    ([0, 1, 15, 16, 31, 300], [1] * 6, 32, 8, 128, 16),          # ragged single tokens
    ([777, 5, 2500], [1] * 3, 8, 8, 64, 64),                     # no grouping; split over CTAs
    ([1000, 63], [1, 1], 10, 2, 128, 128),                       # five heads to a KV head
    ([640, 100], [1, 1], 12, 1, 64, 32),                         # twelve: two blocks of rows
    ([5000], [1], 32, 1, 128, 32),                               # thirty-two; many splits
    ([100, 0, 31], [3, 4, 1], 8, 2, 128, 16),                    # a few new tokens each (speculation)
    ([513, 40], [2, 0], 16, 1, 128, 16),                         # a sequence without new tokens
    ([0, 33], [40, 7], 8, 2, 64, 16),                            # prompts
    ([70, 0, 1], [65, 130, 1], 4, 4, 128, 64),                   # prompts and a single token together
    ([0], [257], 5, 1, 128, 128),
    ([190], [65], 32, 1, 64, 32),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page", SHAPES)
def test_attention(dtype, e4m3, ctx, new, Hq, Hkv, D, page):
    c = _filled(ctx, new, Hkv, D, page, dtype, e4m3, seed=11, spread=0.5)
    q = (1.5 * torch.randn(sum(new), Hq, D, generator=_gen(12))).to(dtype)
    _check_attention(c, q)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (16, 16), (100, 3), (33, 40), (10000, 4), (64, 0),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page", [
    ([0, 6, 50, 200, 1500], [1] * 5, 8, 2, 128, 16),
    ([600, 40], [4, 2], 8, 2, 64, 32),
    ([300, 0], [70, 90], 4, 2, 128, 64),
])
def test_attention_window_sinks(window, sinks, e4m3, ctx, new, Hq, Hkv, D, page):
    """Rows that the window hides hold NaN: nobody may look at them."""
    c = _filled(ctx, new, Hkv, D, page, BF16, e4m3, seed=13, spread=0.3)
    for b, (a, n) in enumerate(zip(ctx, new)):
        hidden = ~oracle.visible(a, n, window, sinks).any(dim=0)
        for j in hidden.nonzero()[:, 0].tolist():
            for pool in c.pools:
                if e4m3:
                    pool.view(torch.uint8)[int(c.table[b, j // page]), :, j % page] = 0x7F
                else:
                    pool[int(c.table[b, j // page]), :, j % page] = math.nan
    q = torch.randn(sum(new), Hq, D, generator=_gen(14)).to(BF16)
    _check_attention(c, q, window, sinks)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_scales_and_peaks(dtype, e4m3):
    """Page scales that differ by many powers of two, scores that peak on one row, and queries of any size."""
    ctx, new = [700, 333, 90], [1, 1, 1]
    c = _filled(ctx, new, 2, 128, 16, dtype, e4m3, seed=15, spread=2.0)
    q = torch.randn(3, 8, 128, generator=_gen(16))
    q[0] *= 8.0
    q[1] *= 2.0 ** -12
    _check_attention(c, q.to(dtype), scale=0.02)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page", [
    ([5000], [40], 8, 2, 128, 64),                      # a short prompt behind a long context: the span is split and joined
    ([3000, 4100], [33, 9], 4, 1, 64, 16),              # the same, two sequences
    ([300, 40, 900, 7], [1, 90, 2, 1], 8, 2, 128, 16),  # single tokens and prompts in one call: both kernels
    ([20, 0, 129], [300, 128, 1], 16, 1, 64, 128),
    ([1], [1023], 2, 1, 128, 32),                       # rows of two whole tiles but one
])
def test_attention_prompts_split_and_mixed(e4m3, ctx, new, Hq, Hkv, D, page):
    for dtype in (F16, BF16):
        c = _filled(ctx, new, Hkv, D, page, dtype, e4m3, seed=24, spread=0.5)
        q = torch.randn(sum(new), Hq, D, generator=_gen(25)).to(dtype)
        _check_attention(c, q)
        _check_attention(c, q, window=700, sinks=5)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("ctx,new,Hq,Hkv,D,page", [
    ([40, 0], [3, 8], 8, 2, 128, 16),                   # few new tokens
    ([1000], [5], 20, 4, 64, 64),
    ([2000], [30], 1, 1, 64, 16),                       # thirty-two rows; split over CTAs
    ([70, 0, 500], [90, 300, 40], 4, 2, 128, 16),       # prompts
    ([3000], [40], 8, 1, 64, 64),                       # a split prompt
    ([130], [270], 2, 2, 128, 128),
])
def test_attention_hidden_infinities(e4m3, ctx, new, Hq, Hkv, D, page):
    """Infinities and NaN in K and V of rows that only some of the new tokens see: the others are as without them, and what
    the formula makes infinite or NaN is so."""
    for dtype, (window, sinks) in itertools.product((F16, BF16), ((0, 0), (21, 2))):
        c = _filled(ctx, new, Hkv, D, page, dtype, e4m3, seed=41, spread=0.3, poison=False)
        for b, (a, n) in enumerate(zip(ctx, new)):
            # late rows, and one that a window drops half-way through the new tokens
            for i, j in enumerate({a + n - 1, a + n // 2, max(0, a + n // 2 - 21), max(0, a + 1 - 21)}):
                pg, slot = int(c.table[b, j // page]), j % page
                for pool, d in ((c.pools[1], 3 + 5 * i), (c.pools[1], D - 2 - i), (c.pools[0], 0)):
                    if pool is c.pools[0] and j != a + n - 1:
                        continue
                    value = (math.nan, math.inf, -math.inf, math.nan)[i]
                    if e4m3:
                        pool.view(torch.uint8)[pg, 0, slot, d] = 0xFF if i & 1 else 0x7F
                    else:
                        pool[pg, 0, slot, d] = value
        q = torch.randn(sum(new), Hq, D, generator=_gen(42)).to(dtype)
        d = c.cuda()
        want, mag = oracle.attention(q, *c.oracle_args(), c.table, c.ctx, c.new, window, sinks, row_by_row=True)
        got = ops.paged_attention(q.cuda(), max_new_tokens=max(new), window=window, sinks=sinks, **d).double().cpu()
        fine = torch.isfinite(want)
        assert 0.5 < fine.double().mean() < 1
        assert torch.equal(torch.isfinite(got), fine)
        prompt = max(new) * (Hq // Hkv) > 32
        tol = _attention_tolerance(dtype, e4m3, prompt, want, mag)
        _within(got.masked_fill(~fine, 0), want.masked_fill(~fine, 0), tol.masked_fill(~fine, 1))


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_attention_scales_of_any_sign(new, scale):
    """A scale of 0 (the mean over the visible rows), a negative one, and one that lets a single row win."""
    for e4m3 in (False, True):
        c = _filled([170, 3], [new, new], 2, 64, 16, F16, e4m3, seed=26, spread=0.2)
        q = torch.randn(2 * new, 4, 64, generator=_gen(27)).to(F16)
        _check_attention(c, q, scale=scale)
        _check_attention(c, torch.zeros_like(q), scale=scale, window=20, sinks=2)


@pytest.mark.parametrize("hint", [1, 64, 600, 100000])
def test_attention_context_hint_does_not_matter(hint):
    c = _filled([900, 10, 0], [1, 1, 1], 2, 128, 16, F16, False, seed=17)
    q = torch.randn(3, 8, 128, generator=_gen(18)).to(F16)
    _check_attention(c, q, max_context=hint)


def test_attention_rows_of_lowest_scores():
    """Scores of -infinity beside finite ones, and keys so far below that their weight is zero."""
    c = _filled([200], [1], 1, 64, 16, F16, False, seed=19)
    c.pools[0][int(c.table[0, 2]), 0, 3, :] = -60000.0  # score far below every other one
    c.pools[0][int(c.table[0, 5]), 0, 7, 0] = -math.inf
    q = torch.ones(1, 1, 64, dtype=F16)
    _check_attention(c, q)


@pytest.mark.parametrize("new", [1, 50])
def test_attention_bad_pages_are_skipped(new):
    """A page id outside the pool is recorded, and the rest is attended."""
    c = _filled([100], [new], 1, 64, 16, F16, False, seed=20)
    q = torch.randn(new, 2, 64, generator=_gen(21)).to(F16)
    d = c.cuda()
    for bad in (-1, c.num_pages, 2 ** 31 - 1):
        d["block_table"][0, 1] = bad
        got = ops.paged_attention(q.cuda(), max_new_tokens=new, **d)
        assert torch.isfinite(got).all()
        assert capi.device_status(clear=True) >> 24 == 6
        # appending there writes nothing
        before = d["k_pages"].clone()
        x = torch.ones(1, 1, 64, dtype=F16, device="cuda")
        ops.paged_kv_append(d["k_pages"], d["v_pages"], d["block_table"], _i32([20]), None, x, x)
        assert torch.equal(d["k_pages"].view(torch.int16), before.view(torch.int16))
        assert capi.device_status(clear=True) >> 24 == 6


def test_lengths_beyond_the_table_are_recorded():
    """Positions behind the block table's reach or the rotary table, and more new tokens than announced."""
    c = _filled([30], [2], 1, 64, 16, F16, False, seed=22)
    d = c.cuda()
    d["block_table"] = d["block_table"][:, :2].contiguous()
    x = torch.ones(2, 1, 64, dtype=F16, device="cuda")
    for e4m3 in (False, True):
        kp, vp, ks = d["k_pages"], d["v_pages"], None
        if e4m3:
            kp, vp = (t.float().nan_to_num(0).to(E4M3) for t in (kp, vp))
            ks = torch.ones(c.num_pages, 1, device="cuda")
        before = kp.view(torch.uint8).clone()
        for ctx in (32, 2 ** 31 - 5, -3):
            ops.paged_kv_append(kp, vp, d["block_table"], _i32([ctx]), None, x, x, cu_tokens=_i32([0, 2]), k_scales=ks,
                                v_scales=None if ks is None else ks.clone())
            assert capi.device_status(clear=True) >> 24 == 5
        assert torch.equal(kp.view(torch.uint8), before)
        # a rotary table of 31 rows: position 31 is not written
        ops.paged_kv_append(kp, vp, d["block_table"], _i32([30]), None, x, x, cu_tokens=_i32([0, 2]), k_scales=ks,
                            v_scales=None if ks is None else ks.clone(), freqs=torch.ones(31, 32, 2, device="cuda"))
        assert capi.device_status(clear=True) >> 24 == 5
    q = torch.ones(2, 1, 64, dtype=F16, device="cuda")
    out = torch.full_like(q, 5.0)
    d["cu_tokens"] = _i32([0, 2])
    ops.paged_attention(q, max_new_tokens=1, out=out, **d)
    assert capi.device_status(clear=True) >> 24 == 5 and (out == 5.0).all()


def test_attention_empty_batches():
    c = _filled([4], [1], 2, 64, 16, F16, False, seed=23)
    d = c.cuda()
    none = torch.empty(0, 4, 64, dtype=F16, device="cuda")
    got = ops.paged_attention(none, d["k_pages"], d["v_pages"], d["block_table"][:0], d["context_lens"][:0])
    assert got.shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 3.0, dtype=F16, device="cuda")
    got = ops.paged_attention(torch.ones_like(out), d["k_pages"], d["v_pages"], d["block_table"], d["context_lens"],
                              cu_tokens=_i32([0, 0]), max_new_tokens=1, out=out)
    assert (got == 3.0).all()
    assert ops.paged_kv_append(d["k_pages"], d["v_pages"], d["block_table"][:0], d["context_lens"][:0], none,
                               none[:, :2], none[:, :2]).shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------------------------------------------------
def _check_sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    dev = {n: None if x is None else x.cuda() for n, x in
           dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).items()}
    tokens, logprobs = ops.sample_tokens(logits.cuda(), u.cuda(), **dev)
    again, _ = ops.sample_tokens(logits.cuda(), u.cuda(), **dev)
    assert torch.equal(tokens, again)
    for r in range(logits.shape[0]):
        # parameters as the fp32 numbers that they are
        one = [None if x is None else x[r].item() for x in (temperature, top_k, top_p, min_p)]
        want, lp, _ = oracle.sample(logits[r], u[r].item(), *one)
        assert int(tokens[r]) == want, (r, int(tokens[r]), want, one)
        got = float(logprobs[r])
        assert got == lp or abs(got - lp) <= 1e-6 * max(1.0, abs(lp)), (r, got, lp)  # fp32 rounding of the logarithm
    return tokens


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 37), (4, 1000), (2, 4099), (3, 32000), (9, 128256),
                                        (160, 5003)])
@pytest.mark.parametrize("which", ["plain", "k", "p", "m", "kp", "kpm"])
def test_sample(dtype, rows, vocab, which):
    g = _gen(rows * vocab)
    logits = (2.5 * torch.randn(rows, vocab, generator=g)).to(dtype)
    u = torch.rand(rows, generator=g)
    kw = dict(temperature=0.3 + 1.5 * torch.rand(rows, generator=g))
    if "k" in which:
        kw["top_k"] = torch.randint(1, max(2, min(vocab, 600)), (rows,), generator=g).to(torch.int32)
    if which in ("p", "kp", "kpm"):
        kw["top_p"] = 0.2 + 0.79 * torch.rand(rows, generator=g)
    if "m" in which:
        kw["min_p"] = 0.3 * torch.rand(rows, generator=g)
    _check_sample(logits, u, **kw)


@pytest.mark.parametrize("dtype", [F16, torch.float32])
def test_sample_ties_and_constant_rows(dtype):
    """Whole rows of one value, and a threshold inside a run of equal logits: the lowest indices are kept."""
    g = _gen(31)
    flat = torch.zeros(4, 50000)
    steps = torch.randint(0, 3, (4, 50000), generator=g).float()
    signed = torch.where(torch.rand(4, 50000, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    for x in (flat, steps, signed):
        u = torch.tensor([0.0, 0.25, 0.5, 0.9999999])
        _check_sample(x.to(dtype), u)
        _check_sample(x.to(dtype), u, top_k=torch.tensor([1, 7, 20000, 49999], dtype=torch.int32))
        _check_sample(x.to(dtype), u, top_p=torch.tensor([0.1, 0.37, 0.9, 0.61]),
                      top_k=torch.tensor([0, 30000, 0, 12345], dtype=torch.int32))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows", [2, 40])
def test_sample_many_candidates(dtype, rows):
    """Flat rows: more kept tokens than are collected in one place, for each kind of cut and all together."""
    g = _gen(35 + rows)
    V = 60000
    logits = torch.randn(rows, V, generator=g).to(dtype)
    u = torch.rand(rows, generator=g)
    t = 1.0 + torch.rand(rows, generator=g)
    k = torch.randint(12200, 50000, (rows,), generator=g).to(torch.int32)
    p = 0.6 + 0.39 * torch.rand(rows, generator=g)
    m = 0.01 + 0.02 * torch.rand(rows, generator=g)
    _check_sample(logits, u, t)
    _check_sample(logits, u, t, top_k=k)
    _check_sample(logits, u, t, top_p=p)
    _check_sample(logits, u, t, min_p=m)
    _check_sample(logits, u, t, top_k=k, top_p=p)
    _check_sample(logits, u, t, top_p=p, min_p=m)
    _check_sample(logits, u, t, top_k=k, top_p=p, min_p=m)
    # so hot that one bin holds thousands
    _check_sample(logits, u, 60 * t, top_k=k, top_p=p)
    _check_sample(logits, u, 400 * t, top_p=p)


def test_sample_masked_logits():
    """Tokens that a grammar forbids carry the type's lowest value or -infinity."""
    g = _gen(36)
    x = 3 * torch.randn(6, 5000, generator=g)
    allowed = torch.rand(6, 5000, generator=g) < 0.01
    u = torch.rand(6, generator=g)
    for dtype in (F16, BF16, torch.float32):
        for low in (torch.finfo(dtype).min, -math.inf):
            y = torch.where(allowed, x, torch.tensor(low)).to(dtype)
            for kw in ({}, dict(top_k=torch.full((6,), 200, dtype=torch.int32)), dict(top_p=torch.full((6,), 0.99)),
                       dict(min_p=torch.full((6,), 1e-6))):
                tokens = _check_sample(y, u, **kw)
                assert allowed[torch.arange(6), tokens.cpu()].all()


def test_sample_special_values():
    inf, nan = math.inf, math.nan
    x = torch.tensor([
        [-inf, -inf, -inf, -inf, -inf],
        [nan, nan, nan, nan, nan],
        [-inf, 1.0, nan, 1.0, -inf],
        [inf, 3.0, inf, -inf, 0.0],
        [-3e38, -3e38, -3e38, 3e38, -3e38],
        [1e-45, 0.0, -0.0, 1e-45, -1e-45],
        [nan, -inf, -5.0, -inf, nan],
    ])
    for u in (0.0, 0.3, 0.75, 0.999):
        uu = torch.full((7,), u)
        _check_sample(x, uu)
        _check_sample(x, uu, top_k=torch.full((7,), 2, dtype=torch.int32), top_p=torch.full((7,), 0.8),
                      min_p=torch.full((7,), 0.01), temperature=torch.full((7,), 0.7))
        _check_sample(x, uu, temperature=torch.zeros(7))


def test_sample_parameters_that_are_off():
    g = _gen(33)
    x = torch.randn(6, 3001, generator=g)
    u = torch.rand(6, generator=g)
    base = _check_sample(x, u)
    same = _check_sample(x, u, temperature=torch.ones(6), top_k=torch.tensor([0, -5, 3001, 10 ** 6, 0, 2 ** 31 - 1],
                                                                             dtype=torch.int32),
                         top_p=torch.tensor([1.0, 1.5, math.inf, 1.0, 1.0, 1.0]),
                         min_p=torch.tensor([0.0, -1.0, 0.0, 0.0, 0.0, 0.0]))
    assert torch.equal(base, same)
    # a top-p that is not above 0 and a min-p above 1 leave the largest one
    _check_sample(x, u, top_p=torch.tensor([0.0, -1.0, 1e-30, 0.0, 0.0, 0.0]))
    _check_sample(x, u, min_p=torch.full((6,), 1.5))


def test_sample_strided_rows_and_extreme_temperatures():
    g = _gen(34)
    wide = torch.randn(5, 2 * 1999 + 3, generator=g).to(BF16)
    x = wide[:, 3: 3 + 1999]
    u = torch.rand(5, generator=g)
    t = torch.tensor([1e-6, 1e-3, 1.0, 1e3, 1e30])
    dev = wide.cuda()[:, 3: 3 + 1999]
    tokens, _ = ops.sample_tokens(dev, u.cuda(), temperature=t.cuda())
    for r in range(5):
        assert int(tokens[r]) == oracle.sample(x[r], u[r].item(), t[r].item())[0]


def test_sample_frequencies():
    """2^16 draws over a grid of uniform numbers give each token its share, to one draw."""
    n = 1 << 16
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5])
    u = (torch.arange(n).double() / n).float()
    tokens, _ = ops.sample_tokens(x.expand(n, 5).contiguous().cuda(), u.cuda())
    want = torch.softmax(x.double(), 0) * n
    got = torch.bincount(tokens.cpu(), minlength=5).double()
    assert (got - want).abs().max() <= 1.0


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
def _decode_setup(e4m3, seed=41):
    g = _gen(seed)
    V, Hq, Hkv, D, page, B, steps = 97, 4, 2, 64, 16, 3, 20
    embed = torch.randn(V, (Hq + 2 * Hkv) * D, generator=g).to(BF16)
    head = (0.2 * torch.randn(Hq * D, V, generator=g)).to(BF16)
    freqs = oracle.rotary_table(80, D)
    prompts = [torch.randint(0, V, (n,), generator=g) for n in (33, 5, 18)]
    u = torch.rand(steps, B, generator=g)
    pages = B * 5
    shape = (pages, Hkv, page, D)
    if e4m3:
        kp = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda").view(E4M3)
        extra = dict(k_scales=torch.full(shape[:2], math.nan, device="cuda"),
                     v_scales=torch.full(shape[:2], math.nan, device="cuda"))
    else:
        kp, extra = torch.full(shape, math.nan, dtype=BF16, device="cuda"), {}
    table = torch.randperm(pages, generator=g).reshape(B, 5).to(torch.int32).cuda()
    return dict(V=V, Hq=Hq, Hkv=Hkv, D=D, B=B, steps=steps, embed=embed.cuda(), head=head.cuda(), freqs=freqs.cuda(),
                prompts=prompts, u=u.cuda(), k=kp, v=kp.clone(), extra=extra, table=table)


def _layer(s, tokens, ctx, cu=None, max_new=1, window=24, sinks=2):
    """One attention layer and a head over the new tokens: append, attend, logits."""
    Hq, Hkv, D = s["Hq"], s["Hkv"], s["D"]
    qkv = s["embed"][tokens].unflatten(1, (-1, D))
    q = ops.paged_kv_append(s["k"], s["v"], s["table"], ctx, qkv[:, :Hq], qkv[:, Hq: Hq + Hkv], qkv[:, Hq + Hkv:],
                            freqs=s["freqs"], cu_tokens=cu, **s["extra"])
    o = ops.paged_attention(q, s["k"], s["v"], s["table"], ctx, cu_tokens=cu, max_new_tokens=max_new, max_context=80,
                            window=window, sinks=sinks, **s["extra"])
    return o


def _reference_layer(s, seqs, window=24, sinks=2):
    """The last token's attention output of each whole sequence, dense, from the rounded inputs, in fp64 with unrounded
    keys and values."""
    out = []
    Hq, Hkv, D = s["Hq"], s["Hkv"], s["D"]
    freqs = s["freqs"].cpu()
    for seq in seqs:
        qkv = s["embed"].cpu()[seq].unflatten(1, (-1, D))
        n = len(seq)
        q = oracle.rotate(qkv[-1, :Hq], freqs[n - 1], False)[0]
        k = torch.stack([oracle.rotate(qkv[j, Hq: Hq + Hkv], freqs[j], False)[0] for j in range(n)])
        v = qkv[:, Hq + Hkv:].double()
        see = oracle.visible(n - 1, 1, window, sinks)[0]
        heads = []
        for h in range(Hq):
            a = (k[:, h // 2] @ q[h]) * D ** -0.5
            heads.append(torch.softmax(a.masked_fill(~see, -math.inf), 0) @ v[:, h // 2])
        out.append(torch.stack(heads))
    return torch.stack(out)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_loop(e4m3, graph):
    """Prompts in one call, then single tokens: append, attention with window and sinks, logits, sampling; the decode step
    replayed as a CUDA graph gives the same tokens as eager calls."""
    s = _decode_setup(e4m3)
    B, steps = s["B"], s["steps"]
    lens = [len(p) for p in s["prompts"]]
    cu = _i32([0] + list(itertools.accumulate(lens)))
    ctx = _i32([0] * B)
    o = _layer(s, torch.cat(s["prompts"]).cuda(), ctx, cu, max(lens))
    last = (cu[1:] - 1).long()
    # one key and one value rounding (2^-8 or 2^-4 of a value, and e4m3's subnormals), random over 26 visible rows, move an
    # output by about 2^-4 of the values' size at most: sum p |v| * 2^-4 + scores off by 2^-4 * |q||k| / sqrt(rows)
    want = _reference_layer(s, s["prompts"])
    rel = (o[last].double().cpu() - want).norm() / want.norm()
    assert rel < (2.0 ** -2 if e4m3 else 2.0 ** -6), rel
    temperature = torch.full((B,), 0.8, device="cuda")
    top_p = torch.full((B,), 0.9, device="cuda")
    top_k = torch.full((B,), 40, dtype=torch.int32, device="cuda")

    ctx = _i32(lens)
    token, _ = ops.sample_tokens(o[last].reshape(B, -1) @ s["head"], s["u"][0], temperature, top_k, top_p)
    u_now = s["u"][0].clone()

    def step():
        o = _layer(s, token, ctx)
        t, _ = ops.sample_tokens(o.reshape(B, -1) @ s["head"], u_now, temperature, top_k, top_p)
        token.copy_(t)
        ctx.add_(1)
        return o

    seqs = [p.tolist() for p in s["prompts"]]
    if graph:
        saved = [x.clone() for x in (token, ctx, s["k"].view(torch.uint8), s["v"].view(torch.uint8))]
        saved_scales = {n: x.clone() for n, x in s["extra"].items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        for x, y in zip((token, ctx, s["k"].view(torch.uint8), s["v"].view(torch.uint8)), saved):
            x.copy_(y)
        for n, x in saved_scales.items():
            s["extra"][n].copy_(x)
    for i in range(1, steps):
        for b in range(B):
            seqs[b].append(int(token[b]))
        u_now.copy_(s["u"][i])
        if graph:
            gr.replay()
        else:
            out = step()
        want = _reference_layer(s, seqs)
        rel = (out.double().cpu() - want).norm() / want.norm()
        assert rel < (2.0 ** -2 if e4m3 else 2.0 ** -6), (i, rel)
    if not hasattr(test_serving_loop, "tokens"):
        test_serving_loop.tokens = {}
    prev = test_serving_loop.tokens.setdefault(e4m3, seqs)
    assert prev == seqs  # eager and replayed runs agree


def test_two_streams_at_once():
    """Calls on two streams share no scratch."""
    c = _filled([3000, 2500], [1, 1], 2, 128, 16, F16, False, seed=51)
    d = c.cuda()
    qs = [torch.randn(2, 8, 128, generator=_gen(52 + i)).to(F16).cuda() for i in range(2)]
    want = [ops.paged_attention(q, **d) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(qs[i], **d))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


@pytest.mark.parametrize("rows", [2, 200])
def test_sample_top_p_around_the_end_of_min_p(rows):
    """Top-p that ends before, at and behind the end of min-p's tokens: a few of them, some hundred, some thousand."""
    vocab = 20000
    g = _gen(51)
    logits, top_p, min_p = [], [], []
    for spread in (0.5, 1.0, 2.0, 4.0):
        x = spread * torch.randn(vocab, generator=g)
        w = torch.softmax(x.double(), 0)
        m = 0.05
        part = float(w[w >= m * w.max()].sum())
        for p in (0.2 * part, 0.99 * part, part * (1 - 1e-5), part * (1 + 1e-5), part * 1.0005, part * 1.002, 0.5 * (1 + part)):
            logits.append(x)
            top_p.append(min(p, 0.99999))
            min_p.append(m)
    n = len(logits)
    x = torch.stack(logits)
    pick = torch.arange(rows) % n
    u = torch.rand(rows, generator=g)
    p, m = torch.tensor(top_p)[pick], torch.tensor(min_p)[pick]
    if rows == 2:
        for first in range(0, n, 2):
            sub = slice(first, first + 2)
            _check_rows(x[sub], u, torch.tensor(top_p)[sub], torch.tensor(min_p)[sub])
    else:
        _check_rows(x[pick], u, p, m)


def _check_rows(x, u, top_p, min_p):
    tokens, logprobs = ops.sample_tokens(x.cuda(), u.cuda(), top_p=top_p.cuda(), min_p=min_p.cuda())
    for i in range(x.shape[0]):
        want, share, _ = oracle.sample(x[i], float(u[i]), top_p=float(top_p[i]), min_p=float(min_p[i]))
        assert int(tokens[i]) == want
        assert abs(float(logprobs[i]) - share) < 1e-5
