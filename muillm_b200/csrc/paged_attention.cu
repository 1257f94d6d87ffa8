// Attention over a paged cache (16-bit pages, or e4m3 pages with a power-of-two scale per page and head):
//   o = sum_j softmax_j(q . k_j * scale) v_j   over the rows j a token at position p sees: j <= p and, with a window,
//   j > p - window or j < sinks.
// K and V are read once per KV head; the query heads of the group (and the new tokens of a sequence) are the rows that
// share them. Softmax is taken in one pass with a running maximum and sum in fp32.
//
// Two kernels. Up to 32 rows per KV head (decode): paged_decode_kernel, bound by the bytes of K and V; the visible tokens are
// split over CTAs and joined by paged_merge_kernel. More rows (prompts): paged_prompt_kernel, bound by the tensor cores.
#include "paged_common.cuh"

#include <algorithm>
#include <type_traits>

MUI_STATUS_ACCESSOR(paged_attention)

namespace {

constexpr int PA_TILE = 16;        // tokens per tile: never crosses a page
constexpr int PA_THREADS = 128;
constexpr int PA_WARPS = PA_THREADS / 32;
constexpr int PA_MIN_TILES = 16;   // tiles per split at least (256 tokens)
constexpr int PA_MAX_SPLITS = 128;
constexpr int PA_MAX_DECODE_ROWS = 32;

struct PaArgs {
  PagedView kv;
  const void* q;
  mui_strides2_t qs;
  void* out;
  float* partials;  // [total * Hq, splits, D + 2]: maximum, sum, unnormalised output
  int Hq, G, splits, max_new, window, sinks;
  float scale_log2;
};

// The cache rows that a sequence's new tokens see: tiles [0, n_sink) and [first, first + n - n_sink)
struct Span {
  int kv_len, lo_min, n_sink, first, n;
};
__device__ __forceinline__ Span visible_span(const PaArgs& a, int ctx, int count) {
  Span s;
  const long long room = static_cast<long long>(a.kv.table_stride) << a.kv.page_shift;
  s.kv_len = static_cast<int>(min(room, static_cast<long long>(ctx) + count));
  s.lo_min = a.window > 0 ? max(0, ctx - a.window + 1) : 0;
  s.first = s.lo_min / PA_TILE;
  s.n_sink = min((min(a.sinks, s.lo_min) + PA_TILE - 1) / PA_TILE, s.first);
  s.n = s.n_sink + max(0, (s.kv_len + PA_TILE - 1) / PA_TILE - s.first);
  return s;
}
__device__ __forceinline__ int span_tile(const Span& s, int i) { return i < s.n_sink ? i : i - s.n_sink + s.first; }

// tiles per split and the splits that have any, for a sequence of n tiles
__device__ __forceinline__ int split_tiles(int n, int splits) {
  const int t = (n + splits - 1) / splits;
  return max(PA_MIN_TILES, (t + PA_WARPS - 1) / PA_WARPS * PA_WARPS);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 ld_kv16(const void* p) { return ld_stream16(p); }
__device__ __forceinline__ uint2 ld_kv8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// One tile of 16 cache rows in registers, as the tensor-core fragments want it. K as the A operand of S^T = K q^T: a lane
// holds rows g and g + 8 (g = lane / 4), of each block of 32 (16-bit) or 64 (e4m3) head-dim elements the 16 bytes number
// t = lane % 4; which head-dim element counts as which k index of an MMA is free as long as q agrees. V as the A operand
// of O^T = V^T P^T: a lane holds rows 2t, 2t + 1, 2t + 8, 2t + 9 and of each the 16 bytes number g of every block of 128
// bytes, so its elements e and e + 1 are rows g and g + 8 of an MMA's 16 output dims. Nothing passes through shared memory.
template <bool KV8, int D>
struct Tile {
  static constexpr int KB = KV8 ? D / 64 : D / 32;   // 16-byte pieces per K row and lane
  static constexpr int VW = KV8 ? D / 32 : D / 16;   // 32-bit words per V row and lane
  uint4 k[KB][2];
  uint32_t v[4][VW];
  float ks, vs;  // page scales (e4m3)
};

template <bool KV8, int D>
__device__ __forceinline__ void load_tile(const PaArgs& a, Tile<KV8, D>& t, int page, int kvh, int tb, int kv_len,
                                          int lo_min) {
  constexpr int ES = KV8 ? 1 : 2;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + kvh;
  const size_t row0 = (head << a.kv.page_shift) + (tb & ((1 << a.kv.page_shift) - 1));
  const bool there = page >= 0;
  const unsigned char* kp = reinterpret_cast<const unsigned char*>(a.kv.k_pages) + row0 * (D * ES) + q * 16;
  const unsigned char* vp = reinterpret_cast<const unsigned char*>(a.kv.v_pages) + row0 * (D * ES);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    // a row that nobody sees is not read: what it holds (another owner's bytes, NaN) must not matter
    const int j = tb + g + 8 * r;
    const bool ok = there && j < kv_len && (j >= lo_min || j < a.sinks);
#pragma unroll
    for (int c = 0; c < Tile<KV8, D>::KB; ++c)
      t.k[c][r] = ok ? ld_kv16(kp + (g + 8 * r) * (D * ES) + c * 64) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int slot = 2 * q + (r & 1) + (r >> 1) * 8;
    const int j = tb + slot;
    const bool ok = there && j < kv_len && (j >= lo_min || j < a.sinks);
    const unsigned char* p = vp + slot * (D * ES);
    if (KV8 && D == 64) {
      const uint2 w = ok ? ld_kv8(p + g * 8) : make_uint2(0, 0);
      t.v[r][0] = w.x;
      t.v[r][1] = w.y;
    } else {
#pragma unroll
      for (int c = 0; c < Tile<KV8, D>::VW / 4; ++c) {
        const uint4 w = ok ? ld_kv16(p + c * 128 + g * 16) : make_uint4(0, 0, 0, 0);
        t.v[r][4 * c] = w.x;
        t.v[r][4 * c + 1] = w.y;
        t.v[r][4 * c + 2] = w.z;
        t.v[r][4 * c + 3] = w.w;
      }
    }
  }
}

// grid (splits, KV heads, sequences); 4 warps that take the split's tiles in turn (U at a time) and are joined at the end.
// NT: blocks of eight rows (row = new token * G + head in the group).
template <typename T, bool KV8, int D, int NT, int U>
__global__ void __launch_bounds__(PA_THREADS) paged_decode_kernel(const PaArgs a) {
  // e4m3 goes through the tensor cores as fp16, which holds every e4m3 value; so do q, after a power-of-two scaling per
  // row that brings its largest element near 1, and the probabilities
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr bool SPLIT_P = std::is_same<M, __nv_bfloat16>::value;  // probabilities as bf16 value + bf16 rest
  constexpr int KB = Tile<KV8, D>::KB, KS = KV8 ? 4 : 2;           // k16 steps per 16-byte piece
  constexpr int MT = D / 16;                                       // 16-dim blocks of the output
  extern __shared__ float pa_smem[];                               // [PA_WARPS][NT * 8][D] then m, l
  float* sm_o = pa_smem;
  float* sm_m = pa_smem + PA_WARPS * NT * 8 * D;
  float* sm_l = sm_m + PA_WARPS * NT * 8;

  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  int first, count;
  paged_new_tokens(a.kv, b, first, count);
  const int ctx = __ldcg(a.kv.context_lens + b);
  if (count == 0 || ctx < 0) {
    if (ctx < 0 && threadIdx.x == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx));
    return;
  }
  const int R = count * a.G;
  if (count > a.max_new || R > NT * 8) {
    if (threadIdx.x == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(count));
    return;
  }
  const Span sp = visible_span(a, ctx, count);
  if (sp.kv_len < ctx + count && threadIdx.x == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx + count));
  const int per = split_tiles(sp.n, a.splits);
  const int active = max(1, (sp.n + per - 1) / per);
  if (split >= active) return;
  const int i_end = min(sp.n, (split + 1) * per);

  // q fragments (B operand: n = row g of the block, k in the order of K's pieces) and the rows' visible range
  uint32_t qf[NT][KB * KS][2];
  float qs[NT][2];        // e4m3: scale_log2 times the row's power of two, for the lane's two rows
  int hi[NT][2], lo[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    const T* qp = nullptr;
    if (r < R) qp = reinterpret_cast<const T*>(a.q) + (first + r / a.G) * a.qs.tok + (kvh * a.G + r % a.G) * a.qs.head;
    float amax = 0.f;
    float qv[KB][KS * 4];
#pragma unroll
    for (int c = 0; c < KB; ++c)
#pragma unroll
      for (int e = 0; e < KS * 4; ++e) {
        const int d = c * (KS * 16) + tq * (KS * 4) + e;
        qv[c][e] = qp ? ld_act_f32<T>(qp + d) : 0.f;
        amax = fmaxf(amax, fabsf(qv[c][e]));
      }
    float mul = 1.f, back = 1.f;
    if (KV8) {
      amax = fmaxf(amax, __shfl_xor_sync(MUI_FULL_MASK, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(MUI_FULL_MASK, amax, 2));
      const int e = min(100, max(-100, static_cast<int>(__float_as_uint(amax) >> 23) - 127));
      mul = exp2_int(-e);
      back = exp2_int(e);
    }
#pragma unroll
    for (int c = 0; c < KB; ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[n][c * KS + s][0] = Elt<M>::pack2(qv[c][4 * s] * mul, qv[c][4 * s + 1] * mul);
        qf[n][c * KS + s][1] = Elt<M>::pack2(qv[c][4 * s + 2] * mul, qv[c][4 * s + 3] * mul);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rr = n * 8 + 2 * tq + i;
      const int p = ctx + rr / a.G;
      hi[n][i] = rr < R ? p : -1;
      lo[n][i] = a.window > 0 ? p - a.window + 1 : 0;
      // the scale of row 2 tq + i sits in the lanes with g = 2 tq + i
      qs[n][i] = a.scale_log2 * (KV8 ? __shfl_sync(MUI_FULL_MASK, back, (2 * tq + i) * 4) : 1.f);
    }
  }
  const int lo_max = a.window > 0 ? ctx + count - a.window : 0;  // first row the last new token's window holds

  float m[NT][2], l[NT][2], o[MT][NT][4], vref = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.f;
  }

  // The warp's tiles in the order in which it takes them: U neighbours, then the next U that are its own. Pages and scales of 32
  // of them are looked up at a time, one per lane, so that K and V do not wait for the block table tile by tile.
  const int32_t* table = a.kv.block_table + static_cast<size_t>(b) * a.kv.table_stride;
  constexpr int STEP = PA_WARPS * U;
  const int i_begin = split * per + warp * U;
  int my_page = -1, my_tb = -1;
  float my_ks = 0.f, my_vs = 0.f;
  auto look_up = [&](int n0) {
    const int n = n0 + lane, i = i_begin + (n / U) * STEP + n % U;
    my_page = my_tb = -1;
    my_ks = my_vs = 0.f;
    if (i < i_end) {
      const int tile = span_tile(sp, i);
      const int page = __ldcg(table + (tile * PA_TILE >> a.kv.page_shift));
      if (page >= 0 && page < a.kv.num_pages) {
        my_page = page;
        my_tb = tile * PA_TILE;
        if (KV8) {
          const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + kvh;
          my_ks = __ldcg(a.kv.k_scales + head);
          my_vs = __ldcg(a.kv.v_scales + head);
        }
      } else {
        mui_dev_set_status(MUI_DEV_BAD_PAGE, static_cast<unsigned>(b));
      }
    }
  };
  // tiles n .. n + U - 1 of the warp; those beyond the end have page -1 (all of them masked). n rises from call to call.
  auto fetch = [&](int n, Tile<KV8, D>(&t)[U], int (&tb)[U]) {
    if ((n & 31) == 0) look_up(n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int from = (n + u) & 31;
      const int page = __shfl_sync(MUI_FULL_MASK, my_page, from);
      tb[u] = __shfl_sync(MUI_FULL_MASK, my_tb, from);
      if (KV8) {
        t[u].ks = __shfl_sync(MUI_FULL_MASK, my_ks, from);
        t[u].vs = __shfl_sync(MUI_FULL_MASK, my_vs, from);
      }
      load_tile<KV8, D>(a, t[u], page, kvh, max(tb[u], 0), sp.kv_len, sp.lo_min);
    }
  };

  auto consume = [&](Tile<KV8, D>(&t)[U], int (&tb)[U]) {
    float s[U][NT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KB; ++c) {
        const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&t[u].k[c][0]);
        const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&t[u].k[c][1]);
#pragma unroll
        for (int st = 0; st < KS; ++st) {
          uint32_t a0, a1, a2, a3;
          if (KV8) {
            a0 = e4m3_to_half2(static_cast<uint16_t>(r0[st]));
            a1 = e4m3_to_half2(static_cast<uint16_t>(r1[st]));
            a2 = e4m3_to_half2(static_cast<uint16_t>(r0[st] >> 16));
            a3 = e4m3_to_half2(static_cast<uint16_t>(r1[st] >> 16));
          } else {
            a0 = r0[2 * st];
            a1 = r1[2 * st];
            a2 = r0[2 * st + 1];
            a3 = r1[2 * st + 1];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<M>(s[u][n], a0, a1, a2, a3, qf[n][c * KS + st][0], qf[n][c * KS + st][1]);
        }
      }
      const float ks = KV8 ? t[u].ks : 1.f;
      const bool open = tb[u] >= 0 && tb[u] + PA_TILE - 1 <= ctx && (tb[u] >= lo_max || tb[u] + PA_TILE <= a.sinks);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][n][e] *= qs[n][e & 1] * ks;
          if (!open) {
            const int j = tb[u] + g + (e >> 1) * 8;
            const bool see = tb[u] >= 0 && j <= hi[n][e & 1] && (j >= lo[n][e & 1] || j < a.sinks);
            if (!see) s[u][n][e] = -INFINITY;
          }
        }
    }
    float turn = 1.f;  // e4m3: change of the reference scale of the output
    if (KV8) {
      float v = vref;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tb[u] >= 0) v = fmaxf(v, t[u].vs);
      if (v > vref) {
        turn = vref / v;
        vref = v;
      }
    }
    bool moved = turn != 1.f;
    float corr[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, fmaxf(s[u][n][i], s[u][n][2 + i]));
        mx = fmaxf(mx, __shfl_xor_sync(MUI_FULL_MASK, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(MUI_FULL_MASK, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(MUI_FULL_MASK, mx, 16));
        const float mn = fmaxf(m[n][i], mx);
        const float use = mn == -INFINITY ? 0.f : mn;
        corr[n][i] = ex2(m[n][i] - use);
        moved |= mn != m[n][i];
        m[n][i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[u][n][i] = ex2(s[u][n][i] - use);
          s[u][n][2 + i] = ex2(s[u][n][2 + i] - use);
          sum += s[u][n][i] + s[u][n][2 + i];
        }
        l[n][i] = l[n][i] * corr[n][i] + sum;
      }
    if (__any_sync(MUI_FULL_MASK, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float c0 = corr[n][0] * turn, c1 = corr[n][1] * turn;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          o[j][n][0] *= c0;
          o[j][n][1] *= c1;
          o[j][n][2] *= c0;
          o[j][n][3] *= c1;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = KV8 ? (tb[u] >= 0 && vref > 0.f ? t[u].vs / vref : 0.f) : 1.f;
      uint32_t pb[NT][2], pr[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = s[u][n][2 * h] * f, p1 = s[u][n][2 * h + 1] * f;
          const uint32_t x = Elt<M>::pack2(p0, p1);
          pb[n][h] = movmatrix(x);
          if (SPLIT_P) {
            const float2 back = Elt<M>::unpack2(x);
            pr[n][h] = movmatrix(Elt<M>::pack2(p0 - back.x, p1 - back.y));
          }
        }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        uint32_t a0, a1, a2, a3;
        if (KV8) {
          // word j / 2 of the four rows holds dims 4 (j / 2) .. + 3 of the lane's; bytes of two rows side by side
          const uint32_t lo01 = __byte_perm(t[u].v[0][j >> 1], t[u].v[1][j >> 1], (j & 1) ? 0x7362 : 0x5140);
          const uint32_t lo89 = __byte_perm(t[u].v[2][j >> 1], t[u].v[3][j >> 1], (j & 1) ? 0x7362 : 0x5140);
          a0 = e4m3_to_half2(static_cast<uint16_t>(lo01));
          a1 = e4m3_to_half2(static_cast<uint16_t>(lo01 >> 16));
          a2 = e4m3_to_half2(static_cast<uint16_t>(lo89));
          a3 = e4m3_to_half2(static_cast<uint16_t>(lo89 >> 16));
        } else {
          a0 = __byte_perm(t[u].v[0][j], t[u].v[1][j], 0x5410);
          a1 = __byte_perm(t[u].v[0][j], t[u].v[1][j], 0x7632);
          a2 = __byte_perm(t[u].v[2][j], t[u].v[3][j], 0x5410);
          a3 = __byte_perm(t[u].v[2][j], t[u].v[3][j], 0x7632);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<M>(o[j][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
          if (SPLIT_P) mma16816<M>(o[j][n], a0, a1, a2, a3, pr[n][0], pr[n][1]);
        }
      }
    }
  };

  {
    // two register sets: the loads of one are in flight while the other is multiplied
    Tile<KV8, D> t0[U], t1[U];
    int tb0[U], tb1[U];
    int n = 0;
    fetch(n, t0, tb0);
    for (int i = i_begin; i < i_end; i += 2 * STEP) {
      fetch(n + U, t1, tb1);
      consume(t0, tb0);
      if (i + STEP >= i_end) break;
      fetch(n + 2 * U, t0, tb0);
      consume(t1, tb1);
      n += 2 * U;
    }
  }

  // join the warps: sums over the lanes of a column first
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v = l[n][i];
      v += __shfl_xor_sync(MUI_FULL_MASK, v, 4);
      v += __shfl_xor_sync(MUI_FULL_MASK, v, 8);
      v += __shfl_xor_sync(MUI_FULL_MASK, v, 16);
      const int r = n * 8 + 2 * tq + i;
      if (g == 0) {
        sm_m[warp * NT * 8 + r] = m[n][i];
        sm_l[warp * NT * 8 + r] = v;
      }
      const float f = KV8 ? vref : 1.f;
      float* row = sm_o + (warp * NT * 8 + r) * D;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int d = KV8 ? g * (D / 8) + 2 * j : (j >> 2) * 64 + g * 8 + 2 * (j & 3);
        row[d] = o[j][n][i] * f;
        row[d + 1] = o[j][n][2 + i] * f;
      }
    }
  __syncthreads();
  T* out = reinterpret_cast<T*>(a.out);
  for (int idx = threadIdx.x; idx < R * D; idx += PA_THREADS) {
    const int r = idx / D, d = idx % D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) mm = fmaxf(mm, sm_m[w * NT * 8 + r]);
    const float use = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      const float f = ex2(sm_m[w * NT * 8 + r] - use);
      ll = fmaf(sm_l[w * NT * 8 + r], f, ll);
      oo = fmaf(sm_o[(w * NT * 8 + r) * D + d], f, oo);
    }
    const size_t row = static_cast<size_t>(first + r / a.G) * a.Hq + kvh * a.G + r % a.G;
    if (active == 1) {
      out[row * D + d] = Elt<T>::from_f32(ll != 0.f ? oo / ll : 0.f);
    } else {
      float* p = a.partials + (row * a.splits + split) * (D + 2);
      if (d == 0) {
        p[0] = mm;
        p[1] = ll;
      }
      p[2 + d] = oo;
    }
  }
}

// Joins the splits of a row in split order: a warp per (new token, query head).
template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS) paged_merge_kernel(const PaArgs a) {
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * PA_WARPS + (threadIdx.x >> 5);
  const int t = static_cast<int>(row / a.Hq);
  if (t >= a.kv.total) return;
  int b = t;
  if (a.kv.cu != nullptr) {
    const int32_t* cu = a.kv.cu;
    b = warp_count_le(a.kv.batch, t, [&](int k) { return __ldcg(cu + 1 + k); });
    if (b >= a.kv.batch) return;
  }
  int first, count;
  paged_new_tokens(a.kv, b, first, count);
  const int ctx = __ldcg(a.kv.context_lens + b);
  if (count == 0 || ctx < 0 || count > a.max_new) return;
  const Span sp = visible_span(a, ctx, count);
  const int per = split_tiles(sp.n, a.splits);
  const int active = (sp.n + per - 1) / per;
  if (active <= 1) return;
  const float* p = a.partials + static_cast<size_t>(row) * a.splits * (D + 2);
  float mm = -INFINITY;
  for (int s = lane; s < active; s += 32) mm = fmaxf(mm, __ldcg(p + static_cast<size_t>(s) * (D + 2)));
  mm = warp_max(mm);
  const float use = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, o[D / 32] = {};
#pragma unroll 4
  for (int s = 0; s < active; ++s) {
    const float* ps = p + static_cast<size_t>(s) * (D + 2);
    const float f = ex2(__ldcg(ps) - use);
    ll = fmaf(__ldcg(ps + 1), f, ll);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(ps + 2) + e * 32 + lane);
      o[2 * e] = fmaf(v.x, f, o[2 * e]);
      o[2 * e + 1] = fmaf(v.y, f, o[2 * e + 1]);
    }
  }
  const float inv = ll != 0.f ? 1.f / ll : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(a.out) + static_cast<size_t>(row) * (D / 2);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[e * 32 + lane] = Elt<T>::pack2(o[2 * e] * inv, o[2 * e + 1] * inv);
}

// ---------------------------------------------------------------------------------------------------------------------
// prompts: 64 rows per CTA (16 per warp), 64 cache rows at a time through shared memory
// ---------------------------------------------------------------------------------------------------------------------
constexpr int PP_ROWS = 64, PP_KEYS = 64;

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T, bool KV8, int D>
__global__ void __launch_bounds__(PA_THREADS) paged_prompt_kernel(const PaArgs a) {
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr int CH = D / 8;  // 16-byte chunks per row, stored at chunk ^ (row & 7)
  __shared__ __align__(16) uint4 sk[PP_KEYS * CH];
  __shared__ __align__(16) uint4 sv[PP_KEYS * CH];
  __shared__ float s_ks[PP_KEYS / PA_TILE], s_vs[PP_KEYS / PA_TILE];
  __shared__ int s_tb[PP_KEYS / PA_TILE];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int kvh = blockIdx.y;
  // row tiles are numbered through: sequence b's start at floor(cu[b] * G / 64) + b
  int b = 0, tile_in_seq = 0;
  const int x = gridDim.x - 1 - blockIdx.x;  // the longest spans first
  if (a.kv.cu != nullptr) {
    const int32_t* cu = a.kv.cu;
    auto start = [&](int k) {
      return static_cast<int>(static_cast<long long>(__ldcg(cu + k)) * a.G / PP_ROWS) + k;
    };
    b = warp_count_le(a.kv.batch, x, [&](int k) { return start(k + 1); });
    if (b >= a.kv.batch) return;
    tile_in_seq = x - start(b);
  } else {
    const int tiles = (a.G + PP_ROWS - 1) / PP_ROWS;
    b = x / tiles;
    tile_in_seq = x % tiles;
  }
  int first, count;
  paged_new_tokens(a.kv, b, first, count);
  const int ctx = __ldcg(a.kv.context_lens + b);
  const int R = count * a.G, r0 = tile_in_seq * PP_ROWS;
  if (count > a.max_new || ctx < 0) {
    if (threadIdx.x == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx < 0 ? ctx : count));
    return;
  }
  if (r0 >= R) return;
  const int tok_lo = r0 / a.G, tok_hi = (min(R, r0 + PP_ROWS) - 1) / a.G;  // new tokens of this tile
  const Span sp = visible_span(a, ctx + tok_lo, tok_hi - tok_lo + 1);
  if (sp.kv_len < ctx + tok_hi + 1 && threadIdx.x == 0)
    mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx + tok_hi + 1));

  // q fragments (A operand): rows g and g + 8 of the warp's sixteen
  uint32_t qf[D / 16][4];
  float qs[2];
  int hi[2], lo[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + warp * 16 + g + 8 * h;
    const T* qp = nullptr;
    if (r < R) qp = reinterpret_cast<const T*>(a.q) + (first + r / a.G) * a.qs.tok + (kvh * a.G + r % a.G) * a.qs.head;
    float v[D / 16][4], amax = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[c][e] = qp ? ld_act_f32<T>(qp + c * 16 + (e >> 1) * 8 + tq * 2 + (e & 1)) : 0.f;
        amax = fmaxf(amax, fabsf(v[c][e]));
      }
    float mul = 1.f, back = 1.f;
    if (KV8) {
      amax = fmaxf(amax, __shfl_xor_sync(MUI_FULL_MASK, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(MUI_FULL_MASK, amax, 2));
      const int e = min(100, max(-100, static_cast<int>(__float_as_uint(amax) >> 23) - 127));
      mul = exp2_int(-e);
      back = exp2_int(e);
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      qf[c][h] = Elt<M>::pack2(v[c][0] * mul, v[c][1] * mul);
      qf[c][2 + h] = Elt<M>::pack2(v[c][2] * mul, v[c][3] * mul);
    }
    qs[h] = a.scale_log2 * back;
    const int p = ctx + r / a.G;
    hi[h] = r < R ? p : -1;
    lo[h] = a.window > 0 ? p - a.window + 1 : 0;
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4], vref = 0.f;
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  const int32_t* table = a.kv.block_table + static_cast<size_t>(b) * a.kv.table_stride;
  constexpr int ES = KV8 ? 1 : 2;

  for (int i0 = 0; i0 < sp.n; i0 += PP_KEYS / PA_TILE) {
    __syncthreads();
    // each warp brings one tile of 16 rows
    {
      int tb = -1, page = -1;
      if (i0 + warp < sp.n) {
        const int tile = span_tile(sp, i0 + warp);
        page = __ldcg(table + (tile * PA_TILE >> a.kv.page_shift));
        if (page < 0 || page >= a.kv.num_pages) {
          if (lane == 0) mui_dev_set_status(MUI_DEV_BAD_PAGE, static_cast<unsigned>(b));
          page = -1;
        } else {
          tb = tile * PA_TILE;
        }
      }
      const size_t head = static_cast<size_t>(max(page, 0)) * a.kv.kv_heads + kvh;
      const size_t off = ((head << a.kv.page_shift) + (max(tb, 0) & ((1 << a.kv.page_shift) - 1))) * (D * ES);
      if (lane == 0) {
        s_tb[warp] = tb;
        if (KV8) {
          s_ks[warp] = tb >= 0 ? __ldcg(a.kv.k_scales + head) : 0.f;
          s_vs[warp] = tb >= 0 ? __ldcg(a.kv.v_scales + head) : 0.f;
        }
      }
      for (int c = lane; c < 16 * CH; c += 32) {
        const int row = c / CH, ch = c % CH, j = tb + row;
        const bool ok = tb >= 0 && j < sp.kv_len && (j >= sp.lo_min || j < a.sinks);
        uint4 k4 = make_uint4(0, 0, 0, 0), v4 = k4;
        if (ok) {
          const unsigned char* kp = reinterpret_cast<const unsigned char*>(a.kv.k_pages) + off + (row * D + ch * 8) * ES;
          const unsigned char* vp = reinterpret_cast<const unsigned char*>(a.kv.v_pages) + off + (row * D + ch * 8) * ES;
          if (KV8) {
            const uint2 k2 = ld_kv8(kp), v2 = ld_kv8(vp);
            k4 = make_uint4(e4m3_to_half2((uint16_t)k2.x), e4m3_to_half2((uint16_t)(k2.x >> 16)),
                            e4m3_to_half2((uint16_t)k2.y), e4m3_to_half2((uint16_t)(k2.y >> 16)));
            v4 = make_uint4(e4m3_to_half2((uint16_t)v2.x), e4m3_to_half2((uint16_t)(v2.x >> 16)),
                            e4m3_to_half2((uint16_t)v2.y), e4m3_to_half2((uint16_t)(v2.y >> 16)));
          } else {
            k4 = ld_kv16(kp);
            v4 = ld_kv16(vp);
          }
        }
        const int at = (warp * 16 + row) * CH + (ch ^ (row & 7));
        sk[at] = k4;
        sv[at] = v4;
      }
    }
    __syncthreads();
    float s[PP_KEYS / 8][4];
#pragma unroll
    for (int n = 0; n < PP_KEYS / 8; n += 2) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      s[n + 1][0] = s[n + 1][1] = s[n + 1][2] = s[n + 1][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        // matrices: rows n*8.. chunk 2c, same rows chunk 2c+1, rows n*8+8.. chunk 2c, chunk 2c+1
        const int row = n * 8 + (lane & 7) + ((lane >> 4) << 3), ch = 2 * c + ((lane >> 3) & 1);
        uint32_t r[4];
        ldmatrix_x4(r, smem_u32(&sk[row * CH + (ch ^ (row & 7))]));
        mma16816<M>(s[n], qf[c][0], qf[c][1], qf[c][2], qf[c][3], r[0], r[1]);
        mma16816<M>(s[n + 1], qf[c][0], qf[c][1], qf[c][2], qf[c][3], r[2], r[3]);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < PP_KEYS / 8; ++n) {
      const int tb = s_tb[n / 2];
      const float ks = KV8 ? s_ks[n / 2] : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e >> 1, j = tb + (n & 1) * 8 + 2 * tq + (e & 1);
        const bool see = tb >= 0 && j <= hi[h] && (j >= lo[h] || j < a.sinks);
        s[n][e] = see ? s[n][e] * (qs[h] * ks) : -INFINITY;
        mx[h] = fmaxf(mx[h], s[n][e]);
      }
    }
    float turn = 1.f;
    if (KV8) {
      float v = vref;
#pragma unroll
      for (int w = 0; w < PP_KEYS / PA_TILE; ++w) v = fmaxf(v, s_vs[w]);
      if (v > vref) {
        turn = vref / v;
        vref = v;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(MUI_FULL_MASK, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(MUI_FULL_MASK, mx[h], 2));
      const float mn = fmaxf(m[h], mx[h]);
      const float use = mn == -INFINITY ? 0.f : mn;
      const float corr = ex2(m[h] - use);
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < PP_KEYS / 8; ++n) {
        s[n][2 * h] = ex2(s[n][2 * h] - use);
        s[n][2 * h + 1] = ex2(s[n][2 * h + 1] - use);
        sum += s[n][2 * h] + s[n][2 * h + 1];
      }
      l[h] = l[h] * corr + sum;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][2 * h] *= corr * turn;
        o[j][2 * h + 1] *= corr * turn;
      }
    }
#pragma unroll
    for (int kk = 0; kk < PP_KEYS / 16; ++kk) {
      // probabilities rounded once to the type of the cache's values (half a step, 2^-9 for bf16 and 2^-11 for fp16)
      const float f = KV8 ? (vref > 0.f ? s_vs[kk] / vref : 0.f) : 1.f;
      const uint32_t a0 = Elt<M>::pack2(s[2 * kk][0] * f, s[2 * kk][1] * f);
      const uint32_t a1 = Elt<M>::pack2(s[2 * kk][2] * f, s[2 * kk][3] * f);
      const uint32_t a2 = Elt<M>::pack2(s[2 * kk + 1][0] * f, s[2 * kk + 1][1] * f);
      const uint32_t a3 = Elt<M>::pack2(s[2 * kk + 1][2] * f, s[2 * kk + 1][3] * f);
#pragma unroll
      for (int j = 0; j < D / 8; j += 2) {
        const int row = kk * 16 + (lane & 15), ch = j + (lane >> 4);
        uint32_t r[4];
        ldmatrix_x4_trans(r, smem_u32(&sv[row * CH + (ch ^ (row & 7))]));
        mma16816<M>(o[j], a0, a1, a2, a3, r[0], r[1]);
        mma16816<M>(o[j + 1], a0, a1, a2, a3, r[2], r[3]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(MUI_FULL_MASK, l[h], 1);
    l[h] += __shfl_xor_sync(MUI_FULL_MASK, l[h], 2);
    const int r = r0 + warp * 16 + g + 8 * h;
    if (r >= R) continue;
    const float inv = (l[h] != 0.f ? 1.f / l[h] : 0.f) * (KV8 ? vref : 1.f);
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out) +
                    (static_cast<size_t>(first + r / a.G) * a.Hq + kvh * a.G + r % a.G) * (D / 2);
#pragma unroll
    for (int j = 0; j < D / 8; ++j) out[j * 4 + tq] = Elt<T>::pack2(o[j][2 * h] * inv, o[j][2 * h + 1] * inv);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
// Splits per sequence: enough CTAs to fill the GPU, each with PA_MIN_TILES tiles at least for the longest span.
int pa_splits(int sm_count, int batch, int kv_heads, int max_new, int max_context, int window, int sinks) {
  long long span = max_context;
  if (window > 0) span = std::min<long long>(span, static_cast<long long>(window) + max_new + sinks);
  const long long tiles = (span + PA_TILE - 1) / PA_TILE + 1;
  const long long most = std::max<long long>(1, (tiles + PA_MIN_TILES - 1) / PA_MIN_TILES);
  const long long base = std::max(1, batch * kv_heads);
  const long long want = (static_cast<long long>(sm_count) * 4 + base - 1) / base;
  return static_cast<int>(std::max<long long>(1, std::min<long long>({want, most, PA_MAX_SPLITS})));
}

bool pa_decode(int G, int max_new) { return static_cast<long long>(G) * max_new <= PA_MAX_DECODE_ROWS; }

template <typename T, bool KV8, int D, int NT, int U>
mui_status_t launch_decode(cudaStream_t stream, const PaArgs& a, int pdl) {
  const size_t smem = sizeof(float) * PA_WARPS * NT * 8 * (D + 2);
  if (smem > 48 * 1024)
    MUI_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<T, KV8, D, NT, U>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(smem)));
  MUI_CUDA_CHECK(mui_launch(paged_decode_kernel<T, KV8, D, NT, U>, dim3(a.splits, a.kv.kv_heads, a.kv.batch),
                            dim3(PA_THREADS), smem, stream, pdl, a));
  if (a.splits > 1) {
    const long long rows = static_cast<long long>(a.kv.total) * a.Hq;
    MUI_CUDA_CHECK(mui_launch(paged_merge_kernel<T, D>, dim3(static_cast<unsigned>((rows + PA_WARPS - 1) / PA_WARPS)),
                              dim3(PA_THREADS), 0, stream, 1, a));
  }
  return MUI_OK;
}

template <typename T, bool KV8, int D>
mui_status_t launch_attention(cudaStream_t stream, const PaArgs& a, int pdl) {
  constexpr int U = KV8 ? 2 : 1;
  if (pa_decode(a.G, a.max_new)) {
    const int rows = a.G * a.max_new;
    if (rows <= 8) return launch_decode<T, KV8, D, 1, U>(stream, a, pdl);
    if (rows <= 16) return launch_decode<T, KV8, D, 2, U>(stream, a, pdl);
    return launch_decode<T, KV8, D, 4, U>(stream, a, pdl);
  }
  const long long tiles = a.kv.cu ? static_cast<long long>(a.kv.total) * a.G / PP_ROWS + a.kv.batch
                                  : static_cast<long long>(a.kv.batch) * ((a.G + PP_ROWS - 1) / PP_ROWS);
  MUI_REQUIRE(tiles <= 0x7fffffff, MUI_ERR_UNSUPPORTED, "too many rows");
  MUI_CUDA_CHECK(mui_launch(paged_prompt_kernel<T, KV8, D>, dim3(static_cast<unsigned>(tiles), a.kv.kv_heads),
                            dim3(PA_THREADS), 0, stream, pdl, a));
  return MUI_OK;
}

}  // namespace

extern "C" {

size_t mui_paged_attention_workspace_bytes(int total_tokens, int batch, int num_q_heads, int kv_heads, int head_dim,
                                           int max_new_tokens, int max_context, int window, int sinks) {
  if (total_tokens <= 0 || batch <= 0 || num_q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_new_tokens <= 0 ||
      max_context <= 0)
    return 0;
  if (!pa_decode(num_q_heads / kv_heads, max_new_tokens)) return 0;
  const MuiDeviceInfo* di = mui_current_device_info();
  if (!di) return 0;
  const int splits = pa_splits(di->sm_count, batch, kv_heads, max_new_tokens, max_context, window, sinks);
  if (splits == 1) return 0;
  return static_cast<size_t>(total_tokens) * num_q_heads * splits * (head_dim + 2) * sizeof(float);
}

mui_status_t mui_paged_attention(void* stream, mui_dtype_t dtype, const mui_paged_kv_t* cache, int num_q_heads,
                                 int max_new_tokens, int max_context, int window, int sinks, float scale, const void* q,
                                 mui_strides2_t q_strides, void* out, void* workspace, size_t workspace_bytes,
                                 unsigned flags) {
  if (mui_status_t s = paged_check(dtype, cache)) return s;
  MUI_REQUIRE(num_q_heads >= 1 && num_q_heads % cache->kv_heads == 0, MUI_ERR_INVALID_ARG,
              "num_q_heads=%d not a multiple of kv_heads=%d", num_q_heads, cache->kv_heads);
  const int G = num_q_heads / cache->kv_heads;
  MUI_REQUIRE(G <= PA_MAX_DECODE_ROWS, MUI_ERR_UNSUPPORTED, "%d query heads per KV head (at most %d)", G,
              PA_MAX_DECODE_ROWS);
  MUI_REQUIRE(max_new_tokens >= 1 && max_context >= 1 && window >= 0 && sinks >= 0, MUI_ERR_INVALID_ARG,
              "bad max_new_tokens=%d max_context=%d window=%d sinks=%d", max_new_tokens, max_context, window, sinks);
  if (cache->batch == 0 || cache->total_tokens == 0) return MUI_OK;
  MUI_REQUIRE(q && out, MUI_ERR_INVALID_ARG, "q and out must be non-null");
  MUI_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15) == 0, MUI_ERR_INVALID_ARG, "out must be 16-byte aligned");
  const MuiDeviceInfo* di = mui_current_device_info();
  if (!di) return MUI_ERR_CUDA;
  PaArgs a = {};
  a.kv = paged_view(*cache);
  a.q = q;
  a.qs = q_strides;
  a.out = out;
  a.Hq = num_q_heads;
  a.G = G;
  a.max_new = max_new_tokens;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.44269504088896341f;
  a.splits = 1;
  if (pa_decode(G, max_new_tokens)) {
    a.splits = pa_splits(di->sm_count, cache->batch, cache->kv_heads, max_new_tokens, max_context, window, sinks);
    const size_t need = a.splits == 1 ? 0
                                      : static_cast<size_t>(cache->total_tokens) * num_q_heads * a.splits *
                                            (cache->head_dim + 2) * sizeof(float);
    MUI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                              (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                MUI_ERR_INVALID_ARG, "workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
                workspace ? workspace_bytes : static_cast<size_t>(0));
    a.partials = reinterpret_cast<float*>(workspace);
  }
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define PA_GO(T, D)                                                            \
  (cache->format == MUI_KV_E4M3 ? launch_attention<T, true, D>(st, a, pdl) \
                                : launch_attention<T, false, D>(st, a, pdl))
  if (dtype == MUI_F16) return cache->head_dim == 128 ? PA_GO(__half, 128) : PA_GO(__half, 64);
  return cache->head_dim == 128 ? PA_GO(__nv_bfloat16, 128) : PA_GO(__nv_bfloat16, 64);
#undef PA_GO
}

}  // extern "C"
