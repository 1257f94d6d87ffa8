"""Host-side argument checks of the paged-cache and sampling entry points (no GPU call is reached), and the oracle they
are tested with on the GPU."""
import math

import pytest
import torch

from muillm_b200 import capi, ops
from oracle import paged_oracle as oracle

P = 1 << 20  # stands for a device pointer; nothing dereferences it


def _cache(**kw):
    f = dict(format=capi.MUI_KV_16BIT, num_pages=4, page_size=16, kv_heads=2, head_dim=128, batch=2, table_stride=3,
             total_tokens=2, k_pages=P, v_pages=P, k_scales=None, v_scales=None, block_table=P, context_lens=P,
             cu_tokens=None)
    f.update(kw)
    return capi.PagedKV(*[f[n] for n, _ in capi.PagedKV._fields_])


def _append(cache, dtype=capi.MUI_F16, heads=4, freqs=P, max_pos=100, rotary=128, q=P, k=P, v=P, q_out=P):
    st = capi.Strides2(1024, 128)
    return capi.lib().mui_paged_kv_append(None, dtype, cache, heads, freqs, max_pos, rotary, 0, None, q, st, k, st, v, st,
                                          q_out, 0)


def _attend(cache, dtype=capi.MUI_F16, heads=4, max_new=1, max_context=100, window=0, sinks=0, q=P, out=P):
    st = capi.Strides2(1024, 128)
    return capi.lib().mui_paged_attention(None, dtype, cache, heads, max_new, max_context, window, sinks, 0.1, q, st, out,
                                          None, 0, 0)


BAD_CACHES = [
    (dict(format=7), capi.MUI_ERR_UNSUPPORTED),
    (dict(head_dim=96), capi.MUI_ERR_UNSUPPORTED),
    (dict(page_size=8), capi.MUI_ERR_UNSUPPORTED),
    (dict(page_size=48), capi.MUI_ERR_UNSUPPORTED),
    (dict(kv_heads=0), capi.MUI_ERR_INVALID_ARG),
    (dict(num_pages=0), capi.MUI_ERR_INVALID_ARG),
    (dict(batch=-1), capi.MUI_ERR_INVALID_ARG),
    (dict(table_stride=0), capi.MUI_ERR_INVALID_ARG),
    (dict(total_tokens=3), capi.MUI_ERR_INVALID_ARG),      # no cu_tokens: one per sequence
    (dict(batch=70000, total_tokens=70000), capi.MUI_ERR_UNSUPPORTED),
    (dict(k_pages=None), capi.MUI_ERR_INVALID_ARG),
    (dict(v_pages=P + 8), capi.MUI_ERR_INVALID_ARG),       # 16-byte alignment
    (dict(block_table=None), capi.MUI_ERR_INVALID_ARG),
    (dict(context_lens=None), capi.MUI_ERR_INVALID_ARG),
    (dict(format=capi.MUI_KV_E4M3), capi.MUI_ERR_INVALID_ARG),
    (dict(format=capi.MUI_KV_E4M3, k_scales=P), capi.MUI_ERR_INVALID_ARG),
]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches_are_refused(change, status):
    c = _cache(**change)
    assert _append(c) == status and len(capi.lib().mui_last_error()) > 0
    assert _attend(c) == status


def test_bad_arguments_are_refused():
    c = _cache()
    inv, uns = capi.MUI_ERR_INVALID_ARG, capi.MUI_ERR_UNSUPPORTED
    for kw in (dict(heads=-1), dict(rotary=0), dict(rotary=130), dict(rotary=5), dict(max_pos=0), dict(q=None),
               dict(k=None), dict(v=None), dict(q_out=None), dict(q_out=P + 2)):
        assert _append(c, **kw) == inv, kw
    assert _append(c, dtype=capi.MUI_COMM_F32) == uns
    for kw in (dict(heads=0), dict(heads=3), dict(max_new=0), dict(max_context=0), dict(window=-1), dict(sinks=-1),
               dict(q=None), dict(out=None), dict(out=P + 4)):
        assert _attend(c, **kw) == inv, kw
    assert _attend(c, heads=66) == uns  # 33 query heads to a KV head
    assert _attend(c, dtype=9) == uns


def test_empty_calls_do_nothing():
    assert _append(_cache(batch=0, total_tokens=0, k_pages=None, block_table=None)) == capi.MUI_OK
    assert _attend(_cache(batch=0, total_tokens=0, k_pages=None, block_table=None)) == capi.MUI_OK
    assert capi.lib().mui_paged_attention_workspace_bytes(0, 0, 8, 2, 128, 1, 100, 0, 0) == 0


def test_sample_arguments_are_refused():
    def call(dtype=capi.MUI_F16, rows=2, vocab=10, logits=P, stride=10, u=P, tokens=P):
        return capi.lib().mui_sample_tokens(None, dtype, rows, vocab, logits, stride, None, None, None, None, u, tokens,
                                            None, 0)

    inv = capi.MUI_ERR_INVALID_ARG
    assert call(dtype=5) == capi.MUI_ERR_UNSUPPORTED
    for kw in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(stride=-1), dict(logits=None), dict(u=None),
               dict(tokens=None)):
        assert call(**kw) == inv, kw
    assert call(rows=0, logits=None) == capi.MUI_OK


def test_tensor_entry_points_refuse_host_tensors():
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    pages = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    table, ctx = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_kv_append(pages, pages, table, ctx, x, x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(x, pages, pages, table, ctx)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sample_tokens(torch.zeros(1, 4), torch.zeros(1))


def test_oracle_page_scale():
    for amax, want in ((448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (1.75, 2.0 ** -8), (1.0, 2.0 ** -8),
                       (1.7500001, 2.0 ** -7), (0.0, 2.0 ** -100), (1e-40, 2.0 ** -100)):
        assert oracle.page_scale(amax) == want
    g = torch.Generator().manual_seed(0)
    for a in torch.exp(20 * torch.randn(200, generator=g)).tolist():
        s = oracle.page_scale(a)
        assert math.log2(s) == int(math.log2(s)) and a <= 448 * s and a > 224 * s


def test_oracle_sample():
    """Against a plain enumeration on small rows."""
    g = torch.Generator().manual_seed(1)
    for _ in range(50):
        x = torch.randint(-3, 4, (6,), generator=g).float()
        t, k, p, m = 0.7, 4, 0.8, 0.1
        w = torch.exp((x.double() - x.max()) / t).tolist()
        rank = sorted(range(6), key=lambda i: (-w[i], i))[:k]
        total, run, kept = sum(w[i] for i in rank), 0.0, []
        for i in rank:
            if kept and run >= p * total:
                break
            kept.append(i)
            run += w[i]
        kept = sorted(i for i in kept if w[i] >= m)
        u = float(torch.rand(1, generator=g))
        run, mass = 0.0, sum(w[i] for i in kept)
        for i in kept:
            run += w[i]
            if run > u * mass:
                break
        token, lp, got = oracle.sample(x, u, t, k, p, m)
        assert got == kept and token == i and abs(lp - math.log(w[i] / mass)) < 1e-12
