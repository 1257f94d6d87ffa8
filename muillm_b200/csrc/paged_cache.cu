// Append of the new tokens' keys and values to a paged cache, the rotary position embedding of q and k applied on the
// way:  (y_a, y_b) = (x_a cos - x_b sin, x_b cos + x_a sin)  for the pairs (a, b) of the first rotary_dim elements of a
// head, evaluated in fp32 and rounded once.
//
// Traffic: (Hq + 2 Hkv) * D * 2 bytes in per token, Hq * D * 2 bytes (q) and 2 * Hkv * D * (2 or 1) bytes out, one
// (cos, sin) row per position: bound by memory for prompts, by the launch and two dependent round trips (lengths, then
// block table and rows) for single tokens.
//
//  * 16-bit pages: every (token, head) row is independent.
//  * e4m3 pages: all new rows of one (page, head) share a scale, so they are one unit of work: its rows are rotated in
//    registers, their largest magnitude gives the scale 2^e, rows that were in the page before are rescaled when it grew,
//    the new rows are rounded. No atomics, and K and V are units of their own. The q rows of an e4m3 call are rows as above, in
//    further CTAs of the same launch.
// Measured (device time; 32 q and 8 KV heads of 128, copy bandwidth 6560 GB/s): one token 2.6 us and 64 tokens into e4m3 pages
// 3.0 us, both the launch and the round trips; 9 prompts of 700 to 2500 tokens, 16-bit pages, 82 us = 4.6 TB/s: loads, rotation and
// stores of a warp alternate, at 24 warps an SM neither memory (47 %) nor the issue slots (60 %) are full (more rows in flight and packed
// arithmetic did not help); 3 prompts of 1021 to 2801 tokens, e4m3 pages of 32, 40 q heads, 42 us = 3.9 TB/s, the same: three
// quarters of the bytes are q rows, which are handled as with 16-bit pages.
// Eight consecutive elements of a row sit in one lane (16 bytes). In the half layout the partner of an element is
// rotary_dim / 2 elements away: in another lane, fetched with a shuffle, when that distance is a multiple of eight.
#include "paged_common.cuh"

MUI_STATUS_ACCESSOR(paged_cache)

namespace {

constexpr int PC_THREADS = 256;
constexpr int PC_WARPS = PC_THREADS / 32;

struct AppendArgs {
  PagedView kv;
  const void *q, *k, *v;
  mui_strides2_t qs, ks, vs;
  void* q_out;
  const float* freqs;
  const int64_t* position_ids;
  int Hq, max_positions, rotary, interleaved;
  int freqs_vec;    // the table can be read 16 bytes at a time: aligned, and a lane's eight elements all rotated or none
  int head_blocks;  // row part: blocks of heads per token, each `steps` turns of a warp
  int steps;
  int unit_blocks;  // CTAs of the e4m3 unit part
  int unit_heads;   // KV heads per CTA of it
};

// (cos, sin) of the eight elements from d0 on of a head; identity outside the rotated part. The sine of the first element of a
// pair is negated.
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ void load_turn(const AppendArgs& a, long long pos, int d0, Turn& t) {
  const int half = a.rotary >> 1;
  if (a.freqs == nullptr || d0 >= a.rotary) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t.c[i] = 1.f;
      t.s[i] = 0.f;
    }
    return;
  }
  const float* row = a.freqs + pos * a.rotary;
  if (a.freqs_vec) {
    // the eight elements are four pairs (interleaved) or one element of eight pairs (half), side by side in the table
    const float4* p = reinterpret_cast<const float4*>(row + (a.interleaved ? d0 : 2 * (d0 < half ? d0 : d0 - half)));
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = __ldg(p + i);
        t.c[4 * i] = t.c[4 * i + 1] = v.x;
        t.s[4 * i] = -v.y;
        t.s[4 * i + 1] = v.y;
        t.c[4 * i + 2] = t.c[4 * i + 3] = v.z;
        t.s[4 * i + 2] = -v.w;
        t.s[4 * i + 3] = v.w;
      }
    } else {
      const float sign = d0 < half ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = __ldg(p + i);
        t.c[2 * i] = v.x;
        t.s[2 * i] = sign * v.y;
        t.c[2 * i + 1] = v.z;
        t.s[2 * i + 1] = sign * v.w;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i;
    t.c[i] = 1.f;
    t.s[i] = 0.f;
    if (d < a.rotary) {
      const int pair = a.interleaved ? d >> 1 : (d < half ? d : d - half);
      t.c[i] = row[2 * pair];
      t.s[i] = row[2 * pair + 1];
      if (a.interleaved ? !(d & 1) : d < half) t.s[i] = -t.s[i];
    }
  }
}

// The lane's eight elements of a row as they are in memory, and, when rows are not ALIGNED, their partners in the rotation.
// ALIGNED: rows are 16-byte aligned and, in the half layout, rotary / 2 is a multiple of eight: the partners are another lane's
// eight elements (half) or neighbours (interleaved).
struct RawRow {
  uint4 x, p;
};
template <typename T, bool ALIGNED>
__device__ __forceinline__ RawRow load_row(const AppendArgs& a, const T* row, int d0) {  // row == nullptr: zeros
  RawRow r;
  r.x = r.p = make_uint4(0, 0, 0, 0);
  if (row == nullptr) return r;
  if (ALIGNED) {
    r.x = ld_act16(row + d0);
    return r;
  }
  const unsigned short* e16 = reinterpret_cast<const unsigned short*>(row);
  const int half = a.rotary >> 1;
  uint32_t x[8], p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i;
    int o = d;
    if (d < a.rotary) o = a.interleaved ? (d ^ 1) : (d < half ? d + half : d - half);
    x[i] = __ldcg(e16 + d);
    p[i] = __ldcg(e16 + o);
  }
  r.x = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
  r.p = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
  return r;
}
// The eight elements in fp32, rotated when `turn` (the same for the whole warp, which exchanges elements).
template <typename T, bool ALIGNED>
__device__ __forceinline__ void turn_row(const AppendArgs& a, const RawRow& r, int d0, bool turn, const Turn& t, float (&y)[8]) {
  float x[8], p[8];
  unpack8<T>(r.x, x);
  if (!turn) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
    return;
  }
  if (!ALIGNED) {
    unpack8<T>(r.p, p);
  } else if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i ^ 1];
  } else {
    const int step = a.rotary >> 4, l = d0 >> 3, lane = threadIdx.x & 31;  // lanes from an element to its partner
    const int src = l < step ? lane + step : (l < 2 * step ? lane - step : lane);
    uint4 q;
    q.x = __shfl_sync(MUI_FULL_MASK, r.x.x, src);
    q.y = __shfl_sync(MUI_FULL_MASK, r.x.y, src);
    q.z = __shfl_sync(MUI_FULL_MASK, r.x.z, src);
    q.w = __shfl_sync(MUI_FULL_MASK, r.x.w, src);
    unpack8<T>(q, p);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fmaf(x[i], t.c[i], p[i] * t.s[i]);
  if (d0 + 8 > a.rotary) {  // elements that pass through, infinities and all
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i >= a.rotary) y[i] = x[i];
  }
}

// sequence, place and rotary position of new token t; false for a token behind the last sequence. Whole warp.
__device__ __forceinline__ bool find_token(const AppendArgs& a, int t, int& b, int& ctx, int& i) {
  const int32_t* cu = a.kv.cu;
  if (cu == nullptr) {
    b = t;
    i = 0;
  } else {
    b = warp_count_le(a.kv.batch, t, [&](int k) { return __ldcg(cu + 1 + k); });
    if (b >= a.kv.batch) return false;
    i = t - __ldcg(cu + b);
  }
  ctx = __ldcg(a.kv.context_lens + b);
  if (ctx < 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx));
  return i >= 0 && ctx >= 0;
}

// rotary position of a token; false (and recorded) when the table does not hold it
__device__ __forceinline__ bool find_position(const AppendArgs& a, int t, int ctx, int i, long long& pos) {
  pos = a.position_ids ? __ldcg(a.position_ids + t) : static_cast<long long>(ctx) + i;
  if (a.freqs == nullptr) return true;
  if (pos >= 0 && pos < a.max_positions) return true;
  mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(pos));
  return false;
}

// page of cache position p of sequence b; -1 (and recorded) when there is none
__device__ __forceinline__ int find_page(const PagedView& kv, int b, long long p) {
  const long long idx = p >> kv.page_shift;
  if (p < 0 || idx >= kv.table_stride) {
    mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(p));
    return -1;
  }
  const int page = __ldcg(kv.block_table + static_cast<size_t>(b) * kv.table_stride + idx);
  if (page < 0 || page >= kv.num_pages) {
    mui_dev_set_status(MUI_DEV_BAD_PAGE, static_cast<unsigned>(b));
    return -1;
  }
  return page;
}

// Rows of token t and a block of the heads of the concatenation q | k | v (q only with QONLY): a warp looks the token up and
// loads its (cos, sin) row once for all of them. The rows come TURNS turns at a time, requested before the token is looked up
// and then before the turns in front of them are stored (the compiler must keep loads and stores in order).
template <typename T, int D, bool ALIGNED, bool QONLY, int TURNS>
__device__ __forceinline__ void append_rows(const AppendArgs& a, long long unit) {
  constexpr int LPR = D / 8, RPS = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int t = static_cast<int>(unit / a.head_blocks);
  const int h_begin = static_cast<int>(unit % a.head_blocks) * (a.steps * RPS);
  const int h_end = min(QONLY ? a.Hq : a.Hq + 2 * a.kv.kv_heads, h_begin + a.steps * RPS);
  const int d0 = (lane % LPR) * 8;
  if (t >= a.kv.total) return;
  RawRow raw[TURNS];
  auto request = [&](int h0) {
#pragma unroll
    for (int st = 0; st < TURNS; ++st) {
      const int h = h0 + st * RPS + lane / LPR, hk = h - a.Hq, hv = hk - a.kv.kv_heads;
      const T* in = nullptr;
      if (h < h_end) {
        if (QONLY || hk < 0) in = reinterpret_cast<const T*>(a.q) + t * a.qs.tok + h * a.qs.head;
        else if (hv < 0) in = reinterpret_cast<const T*>(a.k) + t * a.ks.tok + hk * a.ks.head;
        else in = reinterpret_cast<const T*>(a.v) + t * a.vs.tok + hv * a.vs.head;
      }
      raw[st] = load_row<T, ALIGNED>(a, in, d0);
    }
  };
  request(h_begin);
  int b, ctx, i;
  if (!find_token(a, t, b, ctx, i)) return;
  long long pos;
  if (!find_position(a, t, ctx, i, pos)) return;
  T* krow = nullptr;
  T* vrow = nullptr;
  if (!QONLY) {
    const long long p = static_cast<long long>(ctx) + i;
    const int page = find_page(a.kv, b, p);
    if (page >= 0) {
      const size_t off = ((static_cast<size_t>(page) * a.kv.kv_heads << a.kv.page_shift) +
                          static_cast<size_t>(p & ((1 << a.kv.page_shift) - 1))) * D + d0;
      krow = reinterpret_cast<T*>(a.kv.k_pages) + off;
      vrow = reinterpret_cast<T*>(a.kv.v_pages) + off;
    }
  }
  T* qrow = reinterpret_cast<T*>(a.q_out) + static_cast<size_t>(t) * a.Hq * D + d0;
  Turn turn;
  load_turn(a, pos, d0, turn);
#pragma unroll 1
  for (int h0 = h_begin; h0 < h_end; h0 += TURNS * RPS) {
    uint4 w[TURNS];
#pragma unroll
    for (int st = 0; st < TURNS; ++st) {
      const int h = h0 + st * RPS + lane / LPR;
      const bool rot = a.freqs != nullptr && (QONLY || h < a.Hq + a.kv.kv_heads);
      w[st] = raw[st].x;
      if (__any_sync(MUI_FULL_MASK, rot)) {
        float y[8];
        turn_row<T, ALIGNED>(a, raw[st], d0, true, turn, y);
        if (rot) w[st] = pack8<T>(y);
      }
    }
    if (h0 + TURNS * RPS < h_end) request(h0 + TURNS * RPS);
#pragma unroll
    for (int st = 0; st < TURNS; ++st) {
      const int h = h0 + st * RPS + lane / LPR, hk = h - a.Hq, hv = hk - a.kv.kv_heads;
      if (h >= h_end) continue;
      T* out = qrow + h * D;
      if (!QONLY && hk >= 0) {
        out = hv < 0 ? krow : vrow;
        if (out == nullptr) continue;
        out += (static_cast<size_t>(hv < 0 ? hk : hv) << a.kv.page_shift) * D;
      }
      *reinterpret_cast<uint4*>(out) = w[st];
    }
  }
}

template <typename T, int D, bool ALIGNED, int TURNS>
__global__ void __launch_bounds__(PC_THREADS, TURNS == 1 ? 4 : 3) append_rows_kernel(const AppendArgs a) {
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  append_rows<T, D, ALIGNED, false, TURNS>(a, static_cast<long long>(blockIdx.x) * PC_WARPS + (threadIdx.x >> 5));
}

// Units: the new rows of K (which == 0) or V of the heads [head, head_end) in one page, by `GROUPS` groups of D / 8 lanes, at
// most ROWS rows per group. BLOCK: the groups span the CTA (s_max: two sets of one float per warp, used in turn), else one warp.
template <typename T, int D, bool ALIGNED, int ROWS, bool BLOCK>
__device__ __forceinline__ void append_units(const AppendArgs& a, int page, int first_row, int count, int ctx, int page_idx,
                                             int head, int head_end, int which, float (*s_max)[PC_WARPS]) {
  constexpr int LPR = D / 8;
  constexpr int GROUPS = (BLOCK ? PC_THREADS : 32) / LPR;
  const int tid = BLOCK ? threadIdx.x : (threadIdx.x & 31);
  const int group = tid / LPR, d0 = (tid % LPR) * 8;
  const int ps = 1 << a.kv.page_shift;
  const long long p0 = static_cast<long long>(page_idx) << a.kv.page_shift;  // first position of the page
  const int lo = p0 < ctx ? static_cast<int>(ctx - p0) : 0;                   // slots [lo, hi) are new
  const int hi = static_cast<int>(min(static_cast<long long>(ps), static_cast<long long>(ctx) + count - p0));
  const mui_strides2_t st = which == 0 ? a.ks : a.vs;
  const T* in = reinterpret_cast<const T*>(which == 0 ? a.k : a.v);
  const bool rot = which == 0 && a.freqs != nullptr;

  bool have[ROWS];
  long long pos[ROWS];
  const T* src[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int slot = lo + r * GROUPS + group;
    const int i = static_cast<int>(p0 - ctx) + slot;  // place among the sequence's new tokens
    have[r] = slot < hi;
    pos[r] = 0;
    if (have[r]) have[r] = find_position(a, first_row + i, ctx, i, pos[r]);
    if (!have[r]) pos[r] = 0;
    src[r] = in + (first_row + i) * st.tok;
  }
  RawRow raw[ROWS];
  float old_scale = 0.f;
  auto request = [&](int h) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) raw[r] = load_row<T, ALIGNED>(a, have[r] ? src[r] + h * st.head : nullptr, d0);
    float* p = (which == 0 ? a.kv.k_scales : a.kv.v_scales) + static_cast<size_t>(page) * a.kv.kv_heads + h;
    old_scale = lo > 0 ? __ldcg(p) : 0.f;
  };
  request(head);
#pragma unroll 1
  for (; head < head_end; ++head) {
    float* scale_p = (which == 0 ? a.kv.k_scales : a.kv.v_scales) + static_cast<size_t>(page) * a.kv.kv_heads + head;
    uint8_t* out = reinterpret_cast<uint8_t*>(which == 0 ? a.kv.k_pages : a.kv.v_pages) +
                   ((static_cast<size_t>(page) * a.kv.kv_heads + head) << a.kv.page_shift) * D + d0;
    const float was = old_scale;
    float y[ROWS][8];
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      Turn turn;
      if (rot) load_turn(a, pos[r], d0, turn);
      turn_row<T, ALIGNED>(a, raw[r], d0, rot, turn, y[r]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(y[r][e]);
        if (m <= 3.402823466e38f) amax = fmaxf(amax, m);  // false for infinities and NaN
      }
    }
    if (head + 1 < head_end) request(head + 1);  // in flight while this head is stored
    amax = warp_max(amax);
    if (BLOCK) {
      float* m = s_max[head & 1];
      if ((threadIdx.x & 31) == 0) m[threadIdx.x >> 5] = amax;
      __syncthreads();  // also: every thread has the old scale
#pragma unroll
      for (int w = 0; w < PC_WARPS; ++w) amax = fmaxf(amax, m[w]);
    }
    float scale = exp2_int(e4m3_scale_exp(amax));
    float inv = exp2_int(-e4m3_scale_exp(amax));
    if (lo > 0 && !(was < scale)) {
      scale = was;
      inv = 1.f / was;
    } else if (lo > 0) {
      // the page's earlier rows move to the larger scale
      const float ratio = was * inv;
      for (int slot = group; slot < lo; slot += GROUPS) {
        uint2* p = reinterpret_cast<uint2*>(out + static_cast<size_t>(slot) * D);
        const uint2 w = __ldcg(p);
        uint32_t n[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u = h == 0 ? w.x : w.y;
          const float2 f0 = Elt<__half>::unpack2(e4m3_to_half2(static_cast<uint16_t>(u)));
          const float2 f1 = Elt<__half>::unpack2(e4m3_to_half2(static_cast<uint16_t>(u >> 16)));
          n[h] = e4m3_pack2(f0.x * ratio, f0.y * ratio) | (e4m3_pack2(f1.x * ratio, f1.y * ratio) << 16);
        }
        *p = make_uint2(n[0], n[1]);
      }
    }
    if (!BLOCK) __syncwarp();
    if (tid == 0) *scale_p = scale;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (!have[r]) continue;
      const int slot = lo + r * GROUPS + group;
      uint2 w;
      w.x = e4m3_pack2(y[r][0] * inv, y[r][1] * inv) | (e4m3_pack2(y[r][2] * inv, y[r][3] * inv) << 16);
      w.y = e4m3_pack2(y[r][4] * inv, y[r][5] * inv) | (e4m3_pack2(y[r][6] * inv, y[r][7] * inv) << 16);
      *reinterpret_cast<uint2*>(out + static_cast<size_t>(slot) * D) = w;
    }
  }
}

// e4m3 pages, one new token per sequence: a warp per (sequence, head, K or V), then the q rows.
template <typename T, int D, bool ALIGNED>
__global__ void __launch_bounds__(PC_THREADS) append_e4m3_token_kernel(const AppendArgs a) {
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) >= a.unit_blocks) {
    append_rows<T, D, ALIGNED, true, 1>(a, static_cast<long long>(blockIdx.x - a.unit_blocks) * PC_WARPS + warp);
    return;
  }
  const long long u = static_cast<long long>(blockIdx.x) * PC_WARPS + warp;
  const int per_seq = 2 * a.kv.kv_heads;
  const int b = static_cast<int>(u / per_seq), r = static_cast<int>(u % per_seq);
  if (b >= a.kv.batch) return;
  const int ctx = __ldcg(a.kv.context_lens + b);
  if (ctx < 0) {
    mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx));
    return;
  }
  const int page = find_page(a.kv, b, ctx);
  if (page >= 0) 
    append_units<T, D, ALIGNED, 1, false>(a, page, b, 1, ctx, ctx >> a.kv.page_shift, r >> 1, (r >> 1) + 1, r & 1, nullptr);
}

// e4m3 pages, any number of new tokens: a CTA per (sequence, page, block of heads, K or V), then the q rows. Pages are numbered
// through: sequence b's start at cu[b] / page_size + 2 b, which leaves room for every page that its tokens can touch.
template <typename T, int D, bool ALIGNED, int ROWS>
__global__ void __launch_bounds__(PC_THREADS, ROWS <= 2 ? 3 : 2) append_e4m3_kernel(const AppendArgs a) {
  __shared__ float s_max[2][PC_WARPS];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= a.unit_blocks) {
    append_rows<T, D, ALIGNED, true, 4>(
        a, static_cast<long long>(blockIdx.x - a.unit_blocks) * PC_WARPS + (threadIdx.x >> 5));
    return;
  }
  const int per_page = 2 * ((a.kv.kv_heads + a.unit_heads - 1) / a.unit_heads);
  const int u = blockIdx.x / per_page, r = blockIdx.x % per_page;
  const int32_t* cu = a.kv.cu;
  const int sh = a.kv.page_shift;
  const int b = warp_count_le(a.kv.batch, u, [&](int k) { return (__ldcg(cu + 1 + k) >> sh) + 2 * (k + 1); });
  if (b >= a.kv.batch) return;
  int first, count;
  paged_new_tokens(a.kv, b, first, count);
  const int ctx = __ldcg(a.kv.context_lens + b);
  if (ctx < 0) {
    if (threadIdx.x == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx));
    return;
  }
  const int page_idx = (ctx >> sh) + u - ((first >> sh) + 2 * b);
  // never in front of the first new row's page, which cu_tokens that decrease would otherwise bring about
  if (count == 0 || page_idx < (ctx >> sh) || (static_cast<long long>(page_idx) << sh) >= static_cast<long long>(ctx) + count) return;
  const int page = find_page(a.kv, b, static_cast<long long>(page_idx) << sh);
  if (page < 0) return;
  const int head = (r >> 1) * a.unit_heads;
  append_units<T, D, ALIGNED, ROWS, true>(a, page, first, count, ctx, page_idx, head, min(a.kv.kv_heads, head + a.unit_heads), r & 1,
                                          s_max);
}

template <typename T, int D, bool ALIGNED>
mui_status_t launch_append(cudaStream_t stream, AppendArgs a, bool e4m3, int page_size, int sms, unsigned flags) {
  constexpr int RPS = 32 / (D / 8);
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  const dim3 block(PC_THREADS);
  const long long limit = 0x7fffffff;
  auto blocks = [](long long units) { return (units + PC_WARPS - 1) / PC_WARPS; };
  // Turns of heads per warp: one while that leaves the GPU unfilled (64 warps for each SM), up to all heads of a token
  // where it does not: what a warp looks up then serves 12 KiB of a 32 + 8-head token instead of 512 bytes.
  auto choose_steps = [&](int heads) {
    const int turns = (heads + RPS - 1) / RPS;
    a.steps = 1;
    while (a.steps < turns && static_cast<long long>(a.kv.total) * ((turns + a.steps - 1) / a.steps) > sms * 64ll) a.steps *= 2;
    a.head_blocks = (turns + a.steps - 1) / a.steps;
  };
  if (!e4m3) {
    choose_steps(a.Hq + 2 * a.kv.kv_heads);
    const long long n = blocks(static_cast<long long>(a.kv.total) * a.head_blocks);
    MUI_REQUIRE(n <= limit, MUI_ERR_UNSUPPORTED, "too many rows");
    if (a.steps == 1)
      MUI_CUDA_CHECK(mui_launch(append_rows_kernel<T, D, ALIGNED, 1>, dim3((unsigned)n), block, 0, stream, pdl, a));
    else
      MUI_CUDA_CHECK(mui_launch(append_rows_kernel<T, D, ALIGNED, 4>, dim3((unsigned)n), block, 0, stream, pdl, a));
    return MUI_OK;
  }
  choose_steps(a.Hq);
  if (a.Hq == 0) a.head_blocks = 1;
  const long long q_blocks = a.Hq == 0 ? 0 : blocks(static_cast<long long>(a.kv.total) * a.head_blocks);
  if (a.kv.cu == nullptr) {
    a.unit_blocks = static_cast<int>(blocks(static_cast<long long>(a.kv.batch) * 2 * a.kv.kv_heads));
    const long long n = a.unit_blocks + q_blocks;
    MUI_REQUIRE(n <= limit, MUI_ERR_UNSUPPORTED, "too many rows");
    MUI_CUDA_CHECK(mui_launch(append_e4m3_token_kernel<T, D, ALIGNED>, dim3((unsigned)n), block, 0, stream, pdl, a));
    return MUI_OK;
  }
  const long long pages = a.kv.total / page_size + 2ll * a.kv.batch;
  a.unit_heads = 1;  // as for the rows: eight CTAs for each SM
  while (a.unit_heads < a.kv.kv_heads && pages * 2 * (a.kv.kv_heads / a.unit_heads) > sms * 8ll) a.unit_heads *= 2;
  const long long units = pages * 2 * ((a.kv.kv_heads + a.unit_heads - 1) / a.unit_heads);
  const long long n = units + q_blocks;
  MUI_REQUIRE(n <= limit, MUI_ERR_UNSUPPORTED, "too many rows");
  a.unit_blocks = static_cast<int>(units);
  constexpr int GROUPS = PC_THREADS / (D / 8);  // 16 rows at a time for head dim 128, 32 for 64
  const int rows = (page_size + GROUPS - 1) / GROUPS;
  if (rows <= 1)
    MUI_CUDA_CHECK(mui_launch(append_e4m3_kernel<T, D, ALIGNED, 1>, dim3((unsigned)n), block, 0, stream, pdl, a));
  else if (rows <= 2)
    MUI_CUDA_CHECK(mui_launch(append_e4m3_kernel<T, D, ALIGNED, 2>, dim3((unsigned)n), block, 0, stream, pdl, a));
  else if (rows <= 4)
    MUI_CUDA_CHECK(mui_launch(append_e4m3_kernel<T, D, ALIGNED, 4>, dim3((unsigned)n), block, 0, stream, pdl, a));
  else
    MUI_CUDA_CHECK(mui_launch(append_e4m3_kernel<T, D, ALIGNED, 8>, dim3((unsigned)n), block, 0, stream, pdl, a));
  return MUI_OK;
}

bool row_aligned(const void* p, const mui_strides2_t& s) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (s.tok & 7) == 0 && (s.head & 7) == 0;
}

}  // namespace

extern "C" mui_status_t mui_paged_kv_append(void* stream, mui_dtype_t dtype, const mui_paged_kv_t* cache,
                                            int num_q_heads, const float* freqs, int max_positions, int rotary_dim,
                                            int interleaved, const int64_t* position_ids, const void* q,
                                            mui_strides2_t q_strides, const void* k, mui_strides2_t k_strides,
                                            const void* v, mui_strides2_t v_strides, void* q_out, unsigned flags) {
  if (mui_status_t s = paged_check(dtype, cache)) return s;
  MUI_REQUIRE(num_q_heads >= 0, MUI_ERR_INVALID_ARG, "num_q_heads=%d", num_q_heads);
  MUI_REQUIRE(freqs == nullptr || (max_positions >= 1 && rotary_dim >= 2 && rotary_dim <= cache->head_dim &&
                                   (rotary_dim & 1) == 0),
              MUI_ERR_INVALID_ARG, "rotary_dim=%d (even, 2..head_dim) or max_positions=%d (>= 1) out of range",
              rotary_dim, max_positions);
  if (cache->batch == 0 || cache->total_tokens == 0) return MUI_OK;
  MUI_REQUIRE(k && v && (num_q_heads == 0 || (q && q_out)), MUI_ERR_INVALID_ARG, "q, k, v and q_out must be non-null");
  MUI_REQUIRE((reinterpret_cast<uintptr_t>(q_out) & 15) == 0, MUI_ERR_INVALID_ARG, "q_out must be 16-byte aligned");
  const MuiDeviceInfo* di = mui_current_device_info();
  if (!di) return MUI_ERR_CUDA;
  AppendArgs a = {};
  a.kv = paged_view(*cache);
  a.q = q;
  a.k = k;
  a.v = v;
  a.qs = q_strides;
  a.ks = k_strides;
  a.vs = v_strides;
  a.q_out = q_out;
  a.freqs = freqs;
  a.position_ids = position_ids;
  a.Hq = num_q_heads;
  a.max_positions = max_positions;
  a.rotary = freqs ? rotary_dim : 0;
  a.interleaved = interleaved != 0;
  const bool aligned = (num_q_heads == 0 || row_aligned(q, q_strides)) && row_aligned(k, k_strides) &&
                       row_aligned(v, v_strides) && (a.interleaved || (a.rotary & 15) == 0);
  const int whole = a.interleaved ? 8 : 16;  // rotary_dim of which a lane's eight elements are all rotated or none, and paired alike
  a.freqs_vec = freqs != nullptr && (reinterpret_cast<uintptr_t>(freqs) & 15) == 0 && a.rotary % whole == 0;
  const bool e4m3 = cache->format == MUI_KV_E4M3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int ps = cache->page_size, sms = di->sm_count;
#define PC_GO(T, D) \
  (aligned ? launch_append<T, D, true>(st, a, e4m3, ps, sms, flags) : launch_append<T, D, false>(st, a, e4m3, ps, sms, flags))
  if (dtype == MUI_F16) return cache->head_dim == 128 ? PC_GO(__half, 128) : PC_GO(__half, 64);
  return cache->head_dim == 128 ? PC_GO(__nv_bfloat16, 128) : PC_GO(__nv_bfloat16, 64);
#undef PC_GO
}
