"""Calls of the paged-cache and sampling operators at the ends of what their documentation allows."""
import ctypes
import math

import pytest
import torch

from muillm_b200 import capi, ops
from oracle import paged_oracle as oracle
from test_gpu_paged import BF16, E4M3, F16, Cache, _attention_tolerance, _check_append, _filled, _gen, _i32, _within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------------------------------------------------
def _check_written(logits, u, **kw):
    """Tokens and log shares into buffers that hold something else before the call."""
    rows, vocab = logits.shape
    code = {F16: capi.MUI_F16, BF16: capi.MUI_BF16, torch.float32: capi.MUI_COMM_F32}[logits.dtype]
    x, dev = logits.cuda(), {n: t.cuda() for n, t in kw.items()}
    tokens = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
    logprobs = torch.full((rows,), 7.0, device="cuda")
    uu = u.cuda()

    def ptr(n):
        return dev[n].data_ptr() if n in dev else None

    capi.check(capi.lib().mui_sample_tokens(
        torch.cuda.current_stream().cuda_stream, code, rows, vocab, x.data_ptr(), x.stride(0), ptr("temperature"),
        ptr("top_k"), ptr("top_p"), ptr("min_p"), uu.data_ptr(), tokens.data_ptr(), logprobs.data_ptr(), 0))
    for r in range(rows):
        one = {n: t[r].item() for n, t in kw.items()}
        want, lp, _ = oracle.sample(logits[r], u[r].item(), **one)
        assert int(tokens[r]) == want, (r, int(tokens[r]), want, one)
        got = float(logprobs[r])
        assert got == lp or abs(got - lp) <= 1e-6 * max(1.0, abs(lp)), (r, got, lp)  # fp32 rounding of the logarithm


@pytest.mark.parametrize("rows", [2, 100])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_sample_min_p_and_top_p_within_thousands_of_alike_logits(dtype, rows):
    """Top-p ends among thousands of tokens of about the same logit, all of which min-p keeps."""
    g = _gen(61)
    vocab = 9000
    ties = torch.where(torch.rand(rows, vocab, generator=g) < 0.4, 0.0, -3.0)
    hot = torch.randn(rows, vocab, generator=g)
    u = torch.rand(rows, generator=g)
    top_p = 0.1 + 0.5 * torch.rand(rows, generator=g)
    _check_written(ties.to(dtype), u, top_p=top_p, min_p=torch.full((rows,), 0.5))
    _check_written(hot.to(dtype), u, top_p=top_p, min_p=torch.full((rows,), 0.5), temperature=torch.full((rows,), 40.0))


@pytest.mark.parametrize("which", ["none", "k", "p", "kp", "m", "pm", "kpm"])
def test_sample_smallest_temperatures_at_logits_of_zero(which):
    """Temperatures next to the smallest normal number in rows whose largest logit is 0 or +infinity: the steps between
    logits next to 0 are not smaller than those temperatures, so several tokens have weight."""
    g = _gen(62)
    near = -torch.rand(4, 3001, generator=g) * 4e-37
    far = -torch.rand(4, 3001, generator=g)
    far[:, 77] = 0.0
    near[:, 1234] = 0.0
    inf = far.clone()
    inf[:, [5, 900]] = math.inf
    u = torch.tensor([0.0, 0.3, 0.6, 0.95])
    kw = {}
    if "k" in which:
        kw["top_k"] = torch.tensor([1, 40, 700, 3000], dtype=torch.int32)
    if "p" in which:
        kw["top_p"] = torch.tensor([0.9, 0.5, 0.97, 0.3])
    if "m" in which:
        kw["min_p"] = torch.tensor([0.01, 0.2, 1e-4, 0.05])
    for t in (1.2e-38, 1e-37, 1.6e-37, 1e-36):
        for x in (near, far, inf):
            _check_written(x, u, temperature=torch.full((4,), t), **kw)
    for t in (1e-38, 1e-45):  # below the smallest normal number: as that one, which these rows cannot tell
        for x in (far, inf):
            _check_written(x, u, temperature=torch.full((4,), t), **kw)


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 3e38])
def test_sample_rows_of_lowest_values(dtype, temperature):
    """Rows whose tokens all carry the type's lowest value, or that and next to nothing more: what lies behind the row's end
    has no part in them, nor do -infinity and NaN."""
    g = _gen(65)
    low = torch.finfo(dtype).min
    for vocab in (3, 219, 9001):
        x = torch.full((6, vocab), low)
        x[1, 1:] = -math.inf
        x[2, ::2] = math.nan
        x[3, torch.rand(vocab, generator=g) < 0.3] = -math.inf
        x[4, ::3] = low * (1 - 3 * torch.finfo(dtype).eps)  # the next larger numbers
        x[5, 0] = -1.0
        u = torch.rand(6, generator=g)
        one = dict(temperature=torch.full((6,), temperature))
        for kw in ({}, dict(top_p=torch.full((6,), 0.5558)), dict(top_k=torch.full((6,), 50, dtype=torch.int32)),
                   dict(top_p=torch.full((6,), 0.9), min_p=torch.full((6,), 0.05)),
                   dict(top_p=torch.full((6,), 0.3), top_k=torch.full((6,), 100, dtype=torch.int32))):
            y = x.to(dtype)
            if temperature > 1e30:
                # counts as 10^29, which these rows can tell only where logits of that size differ
                y = y[[0, 1, 2, 3]]
                _check_written(y, u[:4], **{n: t[:4] for n, t in {**one, **kw}.items()})
            else:
                _check_written(y, u, **one, **kw)


def test_sample_clusters_beside_other_work():
    """Rows shared by a cluster of CTAs, launched while another stream fills the GPU: every launch gives the same tokens."""
    g = _gen(63)
    x = (2.5 * torch.randn(3, 40000, generator=g)).cuda()
    u = torch.rand(3, generator=g).cuda()
    p = torch.full((3,), 0.9, device="cuda")
    want = ops.sample_tokens(x, u, top_p=p)
    other = torch.cuda.Stream()
    a = torch.randn(2048, 2048, device="cuda")
    other.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(30):
        with torch.cuda.stream(other):
            a = a * 1.0001
        got.append(ops.sample_tokens(x, u, top_p=p))
    torch.cuda.synchronize()
    for tokens, logprobs in got:
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])


@pytest.mark.parametrize("kw", [{}, dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_p=0.9, min_p=0.02), dict(min_p=1e-4),
                                dict(top_k=3000)])
def test_sample_rows_do_not_depend_on_the_batch(kw):
    """A row draws the same token, with the same log share to the last bit, alone (by eight CTAs) and among many (by one)."""
    g = _gen(64)
    for spread in (0.2, 2.5):
        x = (spread * torch.randn(100, 40000, generator=g)).cuda()
        u = torch.rand(100, generator=g).cuda()
        one = {n: torch.full((100,), v, dtype=torch.int32 if n == "top_k" else torch.float32, device="cuda") for n, v in kw.items()}
        tokens, logprobs = ops.sample_tokens(x, u, **one)
        for r in range(0, 100, 9):
            t, lp = ops.sample_tokens(x[r:r + 1], u[r:r + 1], **{n: v[r:r + 1] for n, v in one.items()})
            assert int(t) == int(tokens[r]) and float(lp) == float(logprobs[r])


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cu", [[0, -40, 3], [-40, -20, 3], [3, 0, 3], [0, 90, 3]])
def test_append_new_token_counts_that_make_no_sense(cu):
    """cu_tokens that decrease or are negative: nothing outside the sequences' own pages is written."""
    ctx, ps = [40, 24], 16
    for e4m3 in (False, True):
        dt = E4M3 if e4m3 else F16
        kp = torch.ones(12, 1, ps, 64, dtype=F16, device="cuda").to(dt)
        vp = kp.clone()
        extra = {}
        if e4m3:
            extra = {n: torch.zeros(12, 1, device="cuda") for n in ("k_scales", "v_scales")}
        table = _i32([[4, 5, 6, 7], [8, 9, 10, 11]])
        x = torch.ones(3, 1, 64, dtype=F16, device="cuda")
        before = kp.view(torch.uint8).clone()
        ops.paged_kv_append(kp, vp, table, _i32(ctx), None, x, x, cu_tokens=_i32(cu), **extra)
        for pool in (kp, vp):
            assert torch.equal(pool.view(torch.uint8)[:4], before[:4])
            # the rows in front of the new ones, but for those in the page that the first new one falls into
            assert torch.equal(pool.view(torch.uint8)[[4, 5, 8]], before[[4, 5, 8]])
        capi.device_status(clear=True)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("batch,G,max_new", [(64, 4, 16), (40, 8, 4096), (1, 8, 64), (3, 32, 2)])
def test_attention_loose_bound_on_new_tokens(batch, G, max_new, e4m3):
    """One token per sequence, without cu_tokens, and a max_new_tokens that is not reached. Behind the lengths, in the same
    buffer, there are words that are no lengths."""
    ctx = [(37 * b) % 120 for b in range(batch)]
    c = _filled(ctx, [1] * batch, 1, 64, 16, F16, e4m3, seed=71, spread=0.3)
    q = torch.randn(batch, G, 64, generator=_gen(72)).to(F16)
    d = c.cuda()
    d["context_lens"] = _i32(ctx + [-9] * 400)[:batch]
    want, mag = oracle.attention(q, *c.oracle_args(), c.table, c.ctx, c.new)
    got = ops.paged_attention(q.cuda(), max_new_tokens=max_new, **d)
    _within(got, want, _attention_tolerance(F16, e4m3, False, want, mag))
    assert capi.device_status(clear=False) == 0
    assert torch.equal(got, ops.paged_attention(q.cuda(), **d))
    # the scratch that the C call asks for is the scratch that it is content with
    kv = capi.PagedKV(capi.MUI_KV_E4M3 if e4m3 else capi.MUI_KV_16BIT, c.num_pages, 16, 1, 64, batch, c.table.shape[1], batch,
                      d["k_pages"].data_ptr(), d["v_pages"].data_ptr(),
                      d["k_scales"].data_ptr() if e4m3 else None, d["v_scales"].data_ptr() if e4m3 else None,
                      d["block_table"].data_ptr(), d["context_lens"].data_ptr(), None)
    for max_context in (1, 3000, 2 ** 31 - 1):
        n = capi.lib().mui_paged_attention_workspace_bytes(batch, batch, G, 1, 64, max_new, max_context, 0, 0)
        ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
        qq, out = q.cuda(), torch.full_like(q, 7.0, device="cuda")
        capi.check(capi.lib().mui_paged_attention(
            torch.cuda.current_stream().cuda_stream, capi.MUI_F16, ctypes.byref(kv), G, max_new, max_context, 0, 0, 0.125,
            qq.data_ptr(), capi.Strides2(G * 64, 64), out.data_ptr(), ws.data_ptr() if n else None, n, 0))
        _within(out, want, _attention_tolerance(F16, e4m3, False, want, mag))


BEYOND = [
    # new tokens of the sequence that lies beyond its table, window, sinks
    (1, 10, 0), (3, 10, 0), (50, 10, 0), (1, 0, 0), (50, 0, 0), (1, 10, 5), (50, 10, 5),
]


@pytest.mark.parametrize("ctx", [32, 500, 2 ** 31 - 3])
@pytest.mark.parametrize("new,window,sinks", BEYOND)
@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_beyond_the_table(new, window, sinks, ctx, e4m3):
    """Positions behind the block table's reach are recorded; their tokens see what the table holds, 0 where that is
    nothing. The other sequences of the call are served."""
    c = _filled([20, 9], [12, 1], 2, 64, 16, F16, e4m3, seed=73, spread=0.3)
    d = c.cuda()
    d["block_table"] = d["block_table"][:, :2].contiguous()
    d["context_lens"] = _i32([ctx, 9])
    d["cu_tokens"] = _i32([0, new, new + 1])
    q = torch.randn(new + 1, 4, 64, generator=_gen(74)).to(F16)
    out = torch.full((new + 1, 4, 64), 7.0, dtype=F16, device="cuda")
    ops.paged_attention(q.cuda(), max_new_tokens=new, window=window, sinks=sinks, out=out, **d)
    assert capi.device_status(clear=True) >> 24 == 5
    # what a token at ctx + i sees of the 32 rows that there are
    far = [min(ctx, 10 ** 6) + i for i in range(new)]
    rows = torch.arange(32)
    see = torch.stack([(rows <= p) & ((rows > p - window) | (rows < sinks) if window else rows >= 0) for p in far])
    pk, pv, sk, sv = c.oracle_args()
    for h in range(4):
        k, v = (torch.cat([p[int(c.table[0, i]), h // 2].float().double() * (1.0 if s is None else float(s[int(c.table[0, i]), h // 2]))
                           for i in range(2)]) for p, s in ((pk, sk), (pv, sv)))
        a = (q[:new, h].double() @ k.T * 64 ** -0.5).masked_fill(~see, -math.inf)
        w = torch.softmax(a, 1).nan_to_num(0.0)
        want, mag = w @ v, w @ v.abs()
        _within(out[:new, h], want, _attention_tolerance(F16, e4m3, new * 2 > 32, want, mag))
    want, mag = oracle.attention(q[new:], pk, pv, sk, sv, c.table[1:], [9], [1], window, sinks)
    _within(out[new:], want, _attention_tolerance(F16, e4m3, False, want, mag))


@pytest.mark.parametrize("ctx", [33, 500, 2 ** 31 - 3])
@pytest.mark.parametrize("sinks", [40, 300, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 50])
def test_attention_sinks_beyond_the_table(new, sinks, ctx):
    """More sink tokens than the block table has rows for, and a position behind it: the table is not read further than it
    reaches."""
    c = _filled([32], [0], 1, 64, 16, F16, False, seed=75, spread=0.3)
    d = c.cuda()
    table = torch.full((4, 2), 2 ** 30, dtype=torch.int32)  # behind the sequence's own row there are no pages
    table[0] = c.table[0, :2]
    d["block_table"] = table.cuda()[:1]
    d["context_lens"] = _i32([ctx])
    d["cu_tokens"] = _i32([0, new])
    q = torch.randn(new, 2, 64, generator=_gen(76)).to(F16)
    got = ops.paged_attention(q.cuda(), max_new_tokens=new, window=4, sinks=sinks, **d)
    assert capi.device_status(clear=True) >> 24 == 5  # a length, not a bad page
    k, v = (torch.cat([p[int(i), 0].double() for i in c.table[0, :2]]) for p in c.pools)
    for h in range(2):
        w = torch.softmax(q[:, h].double() @ k.T * 64 ** -0.5, 1)
        _within(got[:, h], w @ v, _attention_tolerance(F16, False, new * 2 > 32, w @ v, w @ v.abs()))


def _low_rows(n, new, dtype, e4m3, low_scale, D=64, page=64):
    """One sequence of n rows and one KV head. Rows 0, 32, ... 224 win: their V is 1 in element 0, and 0 elsewhere. All other
    rows have 128.5 * 2^-24 of the winners' probability, half-way between two fp16 numbers, and V in the other elements;
    on e4m3 pages the V scale is low_scale for the pages behind row 256. Returns (arguments, q, want)."""
    g = _gen(81)
    pages = -(-n // page)
    k, v = torch.zeros(pages * page, D), 0.5 + torch.rand(pages * page, D, generator=g)
    v[:, 0] = 0.0
    win = torch.arange(0, 256, 32)
    k[win, 0] = 11.0
    v[win] = 0.0
    v[win, 0] = 1.0
    k, v = (x.reshape(pages, 1, page, D).to(E4M3 if e4m3 else dtype) for x in (k, v))
    scale = math.log(2.0 ** 24 / 128.5) / 11.0
    args = dict(k_pages=k.cuda(), v_pages=v.cuda(), block_table=torch.arange(pages, dtype=torch.int32)[None].cuda(),
                context_lens=_i32([n - new]), scale=scale, max_new_tokens=new, max_context=1)
    v = v.float().double()
    if e4m3:
        sv = torch.where(torch.arange(pages) * page < 256, 1.0, low_scale)[:, None].clone()
        args.update(k_scales=torch.ones(pages, 1, device="cuda"), v_scales=sv.cuda())
        v = v * sv.double()[:, :, None, None]
    if new > 1:
        args["cu_tokens"] = _i32([0, new])
    q = torch.zeros(new, 2, D)
    q[..., 0] = 1.0
    a = k.float().double().reshape(-1, D)[:, 0] * float(torch.tensor(scale, dtype=torch.float32))
    v = v.reshape(-1, D)
    return args, q.to(dtype), lambda t: torch.softmax(a[: n - new + 1 + t], 0) @ v[: n - new + 1 + t]


LOW_ROWS = pytest.mark.parametrize("dtype,e4m3,low_scale", [
    (F16, False, None), (BF16, False, None), (F16, True, 1.0), (BF16, True, 2.0 ** -9), (F16, True, 3.0 * 2.0 ** -8),
    (F16, True, 2.0 ** 9)])


def _check_low_rows(n, new, dtype, e4m3, low_scale, **kw):
    """The running sums are fp32: of the output, an addition for every 16 rows, which the tensor cores may cut off (2^-23 of the
    sum); of the weights, at most as many, rounded (2^-24). One CTA takes all rows: four warps a quarter each (up to 32
    rows of queries), or one accumulator."""
    args, q, want_of = _low_rows(n, new, dtype, e4m3, low_scale, **kw)
    got = ops.paged_attention(q.cuda(), **args)
    prompt = 2 * new > 32
    steps = n / 16 / (1 if prompt else 4)
    for t in {0, new - 1}:
        want = want_of(t)[None].expand(2, -1)
        _within(got[t], want, _attention_tolerance(dtype, e4m3, prompt, want, want) + want * steps * (2.0 ** -23 + 2.0 ** -24))


@LOW_ROWS
def test_attention_many_rows_of_little_weight(dtype, e4m3, low_scale):
    """Thousands of rows of 2^-17 of the largest probability each, which have elements of V to themselves."""
    _check_low_rows(400000, 1, dtype, e4m3, low_scale)
    _check_low_rows(200000, 16, dtype, e4m3, low_scale, D=128, page=32)
    _check_low_rows(20000, 1, dtype, e4m3, low_scale)
    _check_low_rows(20000, 16, dtype, e4m3, low_scale, D=128, page=32)


@LOW_ROWS
def test_attention_prompts_many_rows_of_little_weight(dtype, e4m3, low_scale):
    """The same for prompts."""
    _check_low_rows(20000, 40, dtype, e4m3, low_scale)
    _check_low_rows(9000, 70, dtype, e4m3, low_scale, D=128, page=128)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("batch", [1, 129, 1500])
def test_large_batches(batch, e4m3):
    """Append and attention for many sequences of few or no new tokens: each token finds its sequence, each result its row."""
    g = _gen(91)
    new = torch.randint(0, 4, (batch,), generator=g).tolist()
    new[-1] = 40
    for counts in (new, [1] * batch):
        ctx = torch.randint(0, 30, (batch,), generator=g).tolist()
        c = Cache(ctx, counts, 1, 64, 16, F16, e4m3, seed=92, spread=0.3)
        k, v = (torch.randn(sum(counts), 1, 64, generator=g).to(F16) for _ in range(2))
        q = torch.randn(sum(counts), 2, 64, generator=g).to(F16)
        d, _ = _check_append(c, q, k, v, oracle.rotary_table(80, 64), False)
        for max_new in {max(counts), 40 if max(counts) > 1 else 1}:
            got = ops.paged_attention(q.cuda(), max_new_tokens=max_new, **d)
            c.pools = [d[n].cpu() for n in ("k_pages", "v_pages")]
            if e4m3:
                c.scales = [d[n].cpu() for n in ("k_scales", "v_scales")]
            want, mag = oracle.attention(q, *c.oracle_args(), c.table, c.ctx, c.new)
            _within(got, want, _attention_tolerance(F16, e4m3, max_new > 16, want, mag))
