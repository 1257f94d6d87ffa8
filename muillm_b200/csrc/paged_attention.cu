// Attention over a paged cache (16-bit pages, or e4m3 pages with a power-of-two scale per page and head):
//   o = sum_j softmax_j(q . k_j * scale) v_j   over the rows j a token at position p sees: j <= p and, with a window,
//   j > p - window or j < sinks.
// K and V are read once per KV head; the query heads of the group (and the new tokens of a sequence) are the rows that
// share them. Softmax is taken in one pass with a running maximum and sum in fp32.
//
// Two kernels. Up to 32 rows per KV head (decode): paged_decode_kernel, bound by the bytes of K and V; the visible rows of all
// sequences are dealt out to the CTAs evenly, and what several CTAs share is joined by paged_merge_kernel. More rows (prompts): paged_prompt_kernel, bound by the tensor cores.
#include "paged_common.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

MUI_STATUS_ACCESSOR(paged_attention)

namespace {

constexpr int PA_TILE = 16;        // tokens per tile: never crosses a page
constexpr int PA_THREADS = 128;
constexpr int PA_WARPS = PA_THREADS / 32;
constexpr int PA_MIN_TILES = 16;   // tiles per CTA at least (256 tokens)
// What beginning and joining a triple costs a CTA, in the time of 4 KiB of K or V: the runs are cut by this measure
constexpr int PA_TRIPLE_COST = 24;
constexpr int PA_MAX_DECODE_ROWS = 32;

struct PaArgs {
  PagedView kv;
  const void* q;
  mui_strides2_t qs;
  void* out;
  float* partials;  // [ctas, 2, rows per block, D + 2]: maximum, sum, unnormalised output
  int Hq, G, ctas, row_blocks, lead, max_new, window, sinks, q_vec;
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
__device__ __forceinline__ uint2 ld_kv8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// ---------------------------------------------------------------------------------------------------------------------
// decode: few rows per KV head
// ---------------------------------------------------------------------------------------------------------------------
// The tiles of all (sequence, KV head, block of rows) triples are laid end to end and dealt out in equal runs, so that every
// CTA streams the same number of bytes whatever the lengths are. A run that covers a triple whole writes its output; the
// others leave partial results, at most two per CTA (the triple that the run starts in and the one it ends in), which
// paged_merge_kernel joins in order.
struct Run {
  int seq, first, count, ctx;  // sequence at the run's first place
  long long begin;             // place at which that sequence begins
};

// Length of a sequence's triples in places: `lead` places for their beginning, then one for each tile; 0: nothing to do
__device__ __forceinline__ int seq_places(const PaArgs& a, int b, Run& r) {
  paged_new_tokens(a.kv, b, r.first, r.count);
  r.ctx = __ldcg(a.kv.context_lens + b);
  r.seq = b;
  if (r.count == 0 || r.ctx < 0 || r.count > a.max_new) return 0;
  const int n = visible_span(a, r.ctx, r.count).n;
  return n ? a.lead + n : 0;
}
__device__ __forceinline__ int seq_places(const PaArgs& a, int b) {
  Run r;
  return seq_places(a, b, r);
}

// Places of all triples, and the place at which the sequences of this thread (blocks of `per_thread`) begin. CTA-wide.
__device__ __forceinline__ long long scan_sequences(const PaArgs& a, int per_thread, long long& mine_begin,
                                                    long long* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b0 = threadIdx.x * per_thread;
  long long sum = 0;
  for (int i = 0; i < per_thread; ++i)
    if (b0 + i < a.kv.batch) sum += seq_places(a, b0 + i);
  sum *= static_cast<long long>(a.kv.kv_heads) * a.row_blocks;
  long long run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(MUI_FULL_MASK, run, o);
    if (lane >= o) run += y;
  }
  if (lane == 31) s_warp[warp] = run;
  __syncthreads();
  long long all = 0;
  run -= sum;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w < warp) run += s_warp[w];
    all += s_warp[w];
  }
  mine_begin = run;
  return all;
}
__device__ __forceinline__ long long run_length(long long total, int ctas) {
  return max(static_cast<long long>(PA_MIN_TILES), (total + ctas - 1) / ctas);  // more than `lead`
}

// K and V pass through shared memory in items of 4 KiB, a ring of four per warp (K, V, K, V), copied asynchronously: three
// items are in flight while one is multiplied, 12 KiB per warp and 144 KiB per SM with three CTAs.
//
// Fragments: K is the A operand of S^T = K q^T; a lane holds rows g and g + 8 (g = lane / 4) of a tile, of each block of 64
// bytes the 16 bytes number t = lane % 4. Which head-dim element counts as which k index of an MMA is free as long as q
// agrees. V is the A operand of O^T = V^T P^T; a lane reads rows 2t, 2t + 1, 2t + 8, 2t + 9, of each block of 128 bytes the 16
// bytes number g, and pairs the rows' elements with byte permutes, its elements e and e + 1 being rows g and g + 8 of an MMA's 16
// output dims. Both reads are free of bank conflicts when row r's 16-byte chunks are stored at chunk ^ swizzle(r).
template <bool KV8, int D>
struct Item {
  static constexpr int ES = KV8 ? 1 : 2;
  static constexpr int RB = D * ES;            // bytes of a row
  static constexpr int CPR = RB / 16;          // chunks of a row
  static constexpr int TOKENS = 4096 / RB;     // 16, 32 or 64
  static constexpr int U = TOKENS / PA_TILE;   // tiles
  static constexpr int KB = RB / 64;           // 16-byte pieces of a K row per lane
  static constexpr int KS = KV8 ? 4 : 2;       // k16 steps of such a piece
  static constexpr int VW = KV8 ? D / 32 : D / 16;  // 32-bit words of a V row per lane
  static __device__ __forceinline__ int swizzle(int row) {
    if (CPR == 4) return (row >> 1) & 3;
    return (row & 2) | (((row >> 2) ^ row) & 1) << 2;
  }
};
constexpr int PA_ITEM = 4096, PA_RING = 4;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// eight consecutive elements of a q row (zeros for a row that does not exist); vec: rows are 16-byte aligned
template <typename T>
__device__ __forceinline__ uint4 load_q8(const T* p, int vec) {
  if (p == nullptr) return make_uint4(0, 0, 0, 0);
  if (vec) return ld_act16(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __ldcg(reinterpret_cast<const unsigned short*>(p) + 2 * i) |
           static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(p) + 2 * i + 1)) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct TileMeta {
  int tb;        // first cache row, -1: nothing to see
  float ks, vs;  // page scales (e4m3)
};

// 4 warps; row = new token * G + head in the group; NT blocks of eight rows per CTA
template <typename T, bool KV8, int D, int NT>
__global__ void __launch_bounds__(PA_THREADS, NT == 1 ? 3 : 2) paged_decode_kernel(const PaArgs a) {
  using I = Item<KV8, D>;
  // e4m3 goes through the tensor cores as fp16, which holds every e4m3 value; so do q, after a power-of-two scaling per
  // row that brings its largest element near 1, and the probabilities
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr bool SPLIT_P = std::is_same<M, __nv_bfloat16>::value;  // probabilities as bf16 value + bf16 rest
  constexpr int U = I::U, KB = I::KB, KS = I::KS, MT = D / 16;
  extern __shared__ __align__(128) unsigned char pa_smem[];        // [warp][PA_RING][PA_ITEM]; the join reuses it
  __shared__ float sm_m[PA_WARPS][NT * 8], sm_l[PA_WARPS][NT * 8];
  __shared__ TileMeta sm_meta[PA_WARPS][2][U];
  __shared__ long long s_warp[PA_WARPS];
  __shared__ Run s_run;

  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;

  // this CTA's run
  const int pairs = a.kv.kv_heads * a.row_blocks;
  const int per_thread = (a.kv.batch + PA_THREADS - 1) / PA_THREADS;
  long long begin;
  const long long total = scan_sequences(a, per_thread, begin, s_warp);
  const long long len = run_length(total, gridDim.x);
  long long place = len * blockIdx.x;
  const long long place_end = min(total, place + len);
  if (place >= place_end && blockIdx.x != 0) return;
  for (int i = 0; i < per_thread; ++i) {
    const int s = threadIdx.x * per_thread + i;
    if (s >= a.kv.batch) break;
    Run r;
    const long long n = static_cast<long long>(seq_places(a, s, r)) * pairs;
    // sequences that cannot be served have no places: say so
    if (blockIdx.x == 0 && n == 0 && r.count > 0 && (r.ctx < 0 || r.count > a.max_new))
      mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(r.ctx < 0 ? r.ctx : r.count));
    if (place >= begin && place < begin + n) {
      r.begin = begin;
      s_run = r;
    }
    begin += n;
  }
  if (place >= place_end) return;
  __syncthreads();
  Run run = s_run;

  const uint32_t ring = smem_u32(pa_smem) + warp * (PA_RING * PA_ITEM);
  while (true) {
    const int b = run.seq, first = run.first, count = run.count, ctx = run.ctx;
    const Span sp = visible_span(a, ctx, count);
    if (sp.kv_len < ctx + count && threadIdx.x == 0)
      mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(ctx + count));
    const int places = a.lead + sp.n;
    const int pair = static_cast<int>((place - run.begin) / places);
    const int kvh = pair / a.row_blocks, rblock = (pair % a.row_blocks) * (NT * 8);
    const int at = static_cast<int>(place - run.begin - static_cast<long long>(pair) * places);
    const int at_end = static_cast<int>(min(static_cast<long long>(places), at + (place_end - place)));
    const int i_begin = max(0, at - a.lead), i_end = max(0, at_end - a.lead);
    const int R = count * a.G - rblock;  // rows from this block on; none left: the tiles are walked past

    if (R > 0 && i_end > i_begin) {
    // The warp's groups of U tiles: every fourth. Pages and scales of 32 tiles are looked up at a time, one per lane, so that
    // K and V do not wait for the block table tile by tile.
    const int32_t* table = a.kv.block_table + static_cast<size_t>(b) * a.kv.table_stride;
    const int groups = (i_end - i_begin + U - 1) / U;           // of all warps
    const int my_groups = groups > warp ? (groups - warp + PA_WARPS - 1) / PA_WARPS : 0;
    // The next 32 are begun half a batch ahead: pages first, their scales once the pages are there.
    int my_page = -1, my_tb = -1, next_page = -1, next_tb = -1;
    float my_ks = 0.f, my_vs = 0.f, next_ks = 0.f, next_vs = 0.f;
    auto ask_pages = [&](int grp) {
      const int i = i_begin + ((grp + lane / U) * PA_WARPS + warp) * U + lane % U;
      next_page = next_tb = -1;
      if (i < i_end) {
        next_tb = span_tile(sp, i) * PA_TILE;
        next_page = __ldcg(table + (next_tb >> a.kv.page_shift));
      }
    };
    auto ask_scales = [&]() {
      if (next_tb >= 0 && (next_page < 0 || next_page >= a.kv.num_pages)) {
        mui_dev_set_status(MUI_DEV_BAD_PAGE, static_cast<unsigned>(b));
        next_page = next_tb = -1;
      }
      next_ks = next_vs = 0.f;
      if (KV8 && next_tb >= 0) {
        const size_t head = static_cast<size_t>(next_page) * a.kv.kv_heads + kvh;
        next_ks = __ldcg(a.kv.k_scales + head);
        next_vs = __ldcg(a.kv.v_scales + head);
      }
    };
    // starts the copy of group grp's K (which == 0) or V; always closes one copy group
    auto issue = [&](int grp, int which) {
      if (grp < my_groups) {
        if (which == 0) {
          const int phase = grp * U & 31;
          if (phase == 0) {
            if (grp == 0) {
              ask_pages(0);
              ask_scales();
            }
            my_page = next_page;
            my_tb = next_tb;
            my_ks = next_ks;
            my_vs = next_vs;
          }
          if (phase == 16) ask_pages(grp + 16 / U);
          if (phase == 24) ask_scales();
          if ((grp * U & 31) / U == lane / U) {
            TileMeta& t = sm_meta[warp][grp & 1][lane % U];
            t.tb = my_tb;
            t.ks = my_ks;
            t.vs = my_vs;
          }
        }
        const unsigned char* base = reinterpret_cast<const unsigned char*>(which == 0 ? a.kv.k_pages : a.kv.v_pages);
        const uint32_t slot = ring + ((grp & 1) * 2 + which) * PA_ITEM;
        constexpr int RPI = 32 / I::CPR;  // rows per copy instruction
        const int ch = lane % I::CPR;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int page = __shfl_sync(MUI_FULL_MASK, my_page, (grp * U + u) & 31);
          const int tb = __shfl_sync(MUI_FULL_MASK, my_tb, (grp * U + u) & 31);
          const size_t row0 = ((static_cast<size_t>(max(page, 0)) * a.kv.kv_heads + kvh) << a.kv.page_shift) +
                              (max(tb, 0) & ((1 << a.kv.page_shift) - 1));
          const unsigned char* src = base + row0 * I::RB + (lane / I::CPR) * I::RB + ch * 16;
          // a row that nobody sees is not read (zeros stand for it): what it holds, another owner's bytes or NaN, must not matter
          const bool whole = tb >= 0 && tb + PA_TILE <= sp.kv_len && (tb >= sp.lo_min || tb + PA_TILE <= a.sinks);
#pragma unroll
          for (int i = 0; i < PA_TILE / RPI; ++i) {
            const int row = u * PA_TILE + i * RPI + lane / I::CPR;
            const uint32_t dst = slot + row * I::RB + ((ch ^ I::swizzle(row)) << 4);
            int bytes = 16;
            if (!whole) {
              const int j = tb + (row & (PA_TILE - 1));
              bytes = tb >= 0 && j < sp.kv_len && (j >= sp.lo_min || j < a.sinks) ? 16 : 0;
            }
            copy16(dst, src + i * RPI * I::RB, bytes);
          }
        }
      }
      copy_commit();
    };

    // q is requested before the first copies, which would delay it by microseconds, and converted after them
    uint4 q_raw[NT][KB][KS / 2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = rblock + n * 8 + g;
      const T* qp = nullptr;
      if (r < count * a.G)
        qp = reinterpret_cast<const T*>(a.q) + (first + r / a.G) * a.qs.tok + (kvh * a.G + r % a.G) * a.qs.head;
#pragma unroll
      for (int c = 0; c < KB; ++c)
#pragma unroll
        for (int e = 0; e < KS / 2; ++e)
          q_raw[n][c][e] = load_q8<T>(qp ? qp + c * (KS * 16) + tq * (KS * 4) + e * 8 : nullptr, a.q_vec);
    }
    issue(0, 0);
    issue(0, 1);
    issue(1, 0);
    issue(1, 1);

    // q fragments (B operand: n = row g of the block, k in the order of K's pieces) and the rows' visible range
    uint32_t qf[NT][KB * KS][2];
    float qs[NT][2];  // scale_log2 (e4m3: times the row's power of two) for the lane's two rows
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float amax = 0.f;
      float qv[KB][KS * 4];
#pragma unroll
      for (int c = 0; c < KB; ++c)
#pragma unroll
        for (int e = 0; e < KS / 2; ++e) {
          float x[8];
          unpack8<T>(q_raw[n][c][e], x);
#pragma unroll
          for (int h = 0; h < 8; ++h) {
            qv[c][8 * e + h] = x[h];
            amax = fmaxf(amax, fabsf(x[h]));
          }
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
        const int p = ctx + (rblock + rr) / a.G;
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

    for (int grp = 0; grp < my_groups; ++grp) {
      const uint32_t kslot = ring + (grp & 1) * 2 * PA_ITEM, vslot = kslot + PA_ITEM;
      copy_wait<3>();
      __syncwarp();
      float s[U][NT][4];
      TileMeta meta[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        meta[u] = sm_meta[warp][grp & 1][u];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KB; ++c) {
          const uint32_t at = kslot + (u * PA_TILE + g) * I::RB + (((c * 4 + tq) ^ I::swizzle(g)) << 4);
          const uint4 k0 = lds16(at), k1 = lds16(at + 8 * I::RB);
          const uint32_t r0[4] = {k0.x, k0.y, k0.z, k0.w}, r1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int st = 0; st < KS; ++st) {
            uint32_t a0, a1, a2, a3;
            if (KV8) {
              a0 = e4m3_to_half2(static_cast<uint16_t>(r0[st]));
              a1 = e4m3_to_half2(static_cast<uint16_t>(r1[st]));
              a2 = e4m3_to_half2(static_cast<uint16_t>(r0[st] >> 16));
              a3 = e4m3_to_half2(static_cast<uint16_t>(r1[st] >> 16));
            } else {
              a0 = r0[2 * st & 3];
              a1 = r1[2 * st & 3];
              a2 = r0[(2 * st + 1) & 3];
              a3 = r1[(2 * st + 1) & 3];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<M>(s[u][n], a0, a1, a2, a3, qf[n][c * KS + st][0], qf[n][c * KS + st][1]);
          }
        }
      }
      __syncwarp();
      issue(grp + 2, 0);

#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tb = meta[u].tb;
        const float ks = KV8 ? meta[u].ks : 1.f;
        const bool open = tb >= 0 && tb + PA_TILE - 1 <= ctx && (tb >= lo_max || tb + PA_TILE <= a.sinks);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][n][e] *= KV8 ? qs[n][e & 1] * ks : qs[n][e & 1];
            if (!open) {
              const int j = tb + g + (e >> 1) * 8;
              const bool see = tb >= 0 && j <= hi[n][e & 1] && (j >= lo[n][e & 1] || j < a.sinks);
              if (!see) s[u][n][e] = -INFINITY;
            }
          }
      }
      float turn = 1.f;  // e4m3: change of the reference scale of the output
      if (KV8) {
        float v = vref;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (meta[u].tb >= 0) v = fmaxf(v, meta[u].vs);
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
      uint32_t pb[U][NT][2], pr[U][NT][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = KV8 ? (meta[u].tb >= 0 && vref > 0.f ? meta[u].vs / vref : 0.f) : 1.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = KV8 ? s[u][n][2 * h] * f : s[u][n][2 * h], p1 = KV8 ? s[u][n][2 * h + 1] * f : s[u][n][2 * h + 1];
            const uint32_t x = Elt<M>::pack2(p0, p1);
            pb[u][n][h] = movmatrix(x);
            if (SPLIT_P) {
              const float2 back = Elt<M>::unpack2(x);
              pr[u][n][h] = movmatrix(Elt<M>::pack2(p0 - back.x, p1 - back.y));
            }
          }
      }

      copy_wait<3>();
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t v[4][I::VW];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int slot = 2 * tq + (r & 1) + (r >> 1) * 8;
          const uint32_t at = vslot + (u * PA_TILE + slot) * I::RB;
          if (I::CPR == 4) {
            lds_v2(at + (((g >> 1) ^ I::swizzle(slot)) << 4) + (g & 1) * 8, v[r][0], v[r][1]);
          } else {
#pragma unroll
            for (int c = 0; c < I::VW / 4; ++c) {
              const uint4 w = lds16(at + (((c * 8 + g) ^ I::swizzle(slot)) << 4));
              v[r][4 * c] = w.x;
              v[r][4 * c + 1] = w.y;
              v[r][4 * c + 2] = w.z;
              v[r][4 * c + 3] = w.w;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          uint32_t a0, a1, a2, a3;
          if (KV8) {
            // word j / 2 of the four rows holds dims 4 (j / 2) .. + 3 of the lane's; bytes of two rows side by side
            const uint32_t p01 = __byte_perm(v[0][j >> 1], v[1][j >> 1], (j & 1) ? 0x7362 : 0x5140);
            const uint32_t p89 = __byte_perm(v[2][j >> 1], v[3][j >> 1], (j & 1) ? 0x7362 : 0x5140);
            a0 = e4m3_to_half2(static_cast<uint16_t>(p01));
            a1 = e4m3_to_half2(static_cast<uint16_t>(p01 >> 16));
            a2 = e4m3_to_half2(static_cast<uint16_t>(p89));
            a3 = e4m3_to_half2(static_cast<uint16_t>(p89 >> 16));
          } else {
            a0 = __byte_perm(v[0][j], v[1][j], 0x5410);
            a1 = __byte_perm(v[0][j], v[1][j], 0x7632);
            a2 = __byte_perm(v[2][j], v[3][j], 0x5410);
            a3 = __byte_perm(v[2][j], v[3][j], 0x7632);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816<M>(o[j][n], a0, a1, a2, a3, pb[u][n][0], pb[u][n][1]);
            if (SPLIT_P) mma16816<M>(o[j][n], a0, a1, a2, a3, pr[u][n][0], pr[u][n][1]);
          }
        }
      }
      __syncwarp();
      issue(grp + 2, 1);
    }

    // join the warps in shared memory (the ring is idle: what was issued last are empty copy groups)
    copy_wait<0>();
    __syncthreads();
    float* sm_o = reinterpret_cast<float*>(pa_smem);  // [warp][NT * 8][D]
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
          sm_m[warp][r] = m[n][i];
          sm_l[warp][r] = v;
        }
        const float f = KV8 ? vref : 1.f;
        float* row = sm_o + (warp * NT * 8 + r) * D;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int d = KV8 ? g * (D / 8) + 2 * j : (j >> 2) * 64 + g * 8 + 2 * (j & 3);
          *reinterpret_cast<float2*>(row + d) = make_float2(o[j][n][i] * f, o[j][n][2 + i] * f);
        }
      }
    __syncthreads();
    const bool whole = i_begin == 0 && i_end == sp.n;
    // partial results: slot 0 of a CTA for a triple that began before its run, slot 1 for one that goes on after it
    float* part = a.partials + (static_cast<size_t>(blockIdx.x) * 2 + (i_begin == 0 ? 1 : 0)) * (NT * 8 * (D + 2));
    T* out = reinterpret_cast<T*>(a.out);
    for (int idx = threadIdx.x; idx < min(R, NT * 8) * D; idx += PA_THREADS) {
      const int r = idx / D, d = idx % D;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) mm = fmaxf(mm, sm_m[w][r]);
      const float use = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float f = ex2(sm_m[w][r] - use);
        ll = fmaf(sm_l[w][r], f, ll);
        oo = fmaf(sm_o[(w * NT * 8 + r) * D + d], f, oo);
      }
      if (whole) {
        const int rr = rblock + r;
        out[(static_cast<size_t>(first + rr / a.G) * a.Hq + kvh * a.G + rr % a.G) * D + d] =
            Elt<T>::from_f32(ll != 0.f ? oo / ll : 0.f);
      } else {
        float* p = part + r * (D + 2);
        if (d == 0) {
          p[0] = mm;
          p[1] = ll;
        }
        p[2 + d] = oo;
      }
    }
    __syncthreads();
    }

    place += at_end - at;
    if (place >= place_end) break;
    if (place - run.begin >= static_cast<long long>(places) * pairs) {  // next sequence that has tiles
      const long long next = run.begin + static_cast<long long>(places) * pairs;
      int s = b + 1;
      while (s < a.kv.batch && seq_places(a, s, run) == 0) ++s;
      run.begin = next;
    }
  }
}

// Joins the partial results of the triples that several CTAs shared. A CTA per (triple, row): its warps take the partial
// results in turn and are joined in shared memory, always in the same order.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(PA_THREADS) paged_merge_kernel(const PaArgs a) {
  __shared__ long long s_warp[PA_WARPS];
  __shared__ long long s_begin;
  __shared__ float sm_m[PA_WARPS], sm_l[PA_WARPS], sm_o[PA_WARPS][D];
  // Lengths were there before the attention kernel began (it waits for its predecessors before it lets this one start), so
  // they are read while it still runs; its partial results only after the wait. Every CTA waits, also one without work: this
  // grid must not be done before the attention kernel is.
  pdl_launch_dependents();
  const int pairs = a.kv.kv_heads * a.row_blocks;
  const int r = blockIdx.x % (NT * 8), triple = blockIdx.x / (NT * 8);
  const int b = triple / pairs, pair = triple % pairs;
  const int kvh = pair / a.row_blocks, rblock = (pair % a.row_blocks) * (NT * 8);
  int first, count;
  paged_new_tokens(a.kv, b, first, count);
  if (rblock + r >= count * a.G) {
    pdl_wait_prior_grid();
    return;
  }
  const int per_thread = (a.kv.batch + PA_THREADS - 1) / PA_THREADS;
  long long begin;
  const long long total = scan_sequences(a, per_thread, begin, s_warp);
  if (b / per_thread == static_cast<int>(threadIdx.x)) {
    for (int i = threadIdx.x * per_thread; i < b; ++i) begin += static_cast<long long>(seq_places(a, i)) * pairs;
    s_begin = begin;
  }
  __syncthreads();
  const int places = seq_places(a, b);
  const long long len = run_length(total, a.ctas);
  const long long at = s_begin + static_cast<long long>(pair) * places;
  // the runs of the first and of the last tile; the first one left slot 1 (the triple begins in it), the others slot 0
  const int c0 = static_cast<int>((at + a.lead) / len), c1 = static_cast<int>((at + places - 1) / len);
  pdl_wait_prior_grid();
  if (places == 0 || c0 >= c1) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float mm = -INFINITY, ll = 0.f, o[D / 32] = {};
  for (int c = c0 + warp; c <= c1; c += 4 * PA_WARPS) {
    float pm[4], pl[4];
    float2 v[4][D / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // four partial results of loads in flight
      const int cc = c + i * PA_WARPS;
      pm[i] = -INFINITY;
      pl[i] = 0.f;
      if (cc <= c1) {
        const float* p = a.partials + ((static_cast<size_t>(cc) * 2 + (cc == c0 ? 1 : 0)) * (NT * 8) + r) * (D + 2);
        pm[i] = __ldcg(p);
        pl[i] = __ldcg(p + 1);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) v[i][e] = __ldcg(reinterpret_cast<const float2*>(p + 2) + e * 32 + lane);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (pm[i] == -INFINITY) continue;
      const float mn = fmaxf(mm, pm[i]), f0 = ex2(mm - mn), f1 = ex2(pm[i] - mn);
      mm = mn;
      ll = ll * f0 + pl[i] * f1;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        o[2 * e] = o[2 * e] * f0 + v[i][e].x * f1;
        o[2 * e + 1] = o[2 * e + 1] * f0 + v[i][e].y * f1;
      }
    }
  }
  if (lane == 0) {
    sm_m[warp] = mm;
    sm_l[warp] = ll;
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    *reinterpret_cast<float2*>(&sm_o[warp][(e * 32 + lane) * 2]) = make_float2(o[2 * e], o[2 * e + 1]);
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += PA_THREADS) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) m = fmaxf(m, sm_m[w]);
    const float use = m == -INFINITY ? 0.f : m;
    float l = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      const float f = ex2(sm_m[w] - use);
      l = fmaf(sm_l[w], f, l);
      x = fmaf(sm_o[w][d], f, x);
    }
    const int rr = rblock + r;
    reinterpret_cast<T*>(a.out)[(static_cast<size_t>(first + rr / a.G) * a.Hq + kvh * a.G + rr % a.G) * D + d] =
        Elt<T>::from_f32(l != 0.f ? x / l : 0.f);
  }
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
            k4 = ld_stream16(kp);
            v4 = ld_stream16(vp);
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
// rows per block of the decode kernel: one block of eight, else blocks of sixteen
int pa_block_rows(int G, int max_new) { return G * max_new <= 8 ? 8 : 16; }
// CTAs of the decode kernel: as many as fit the GPU at once, fewer when the longest sequence expected leaves them without
// PA_MIN_TILES tiles each
int pa_ctas(int sm_count, int batch, int kv_heads, int G, int max_new, int max_context, int window, int sinks) {
  long long span = max_context;
  if (window > 0) span = std::min<long long>(span, static_cast<long long>(window) + max_new + sinks);
  const int block = pa_block_rows(G, max_new);
  const long long tiles = ((span + PA_TILE - 1) / PA_TILE + 2) * batch * kv_heads * ((G * max_new + block - 1) / block);
  const long long most = static_cast<long long>(sm_count) * (block == 8 ? 3 : 2);
  return static_cast<int>(std::max<long long>(1, std::min(most, (tiles + PA_MIN_TILES - 1) / PA_MIN_TILES)));
}
size_t pa_workspace(int ctas, int block, int D) {
  return ctas == 1 ? 0 : static_cast<size_t>(ctas) * 2 * block * (D + 2) * sizeof(float);
}

bool pa_decode(int G, int max_new) { return static_cast<long long>(G) * max_new <= PA_MAX_DECODE_ROWS; }

template <typename T, bool KV8, int D, int NT>
mui_status_t launch_decode(cudaStream_t stream, const PaArgs& a, int pdl, int device) {
  constexpr size_t smem = PA_WARPS * PA_RING * PA_ITEM;
  static std::atomic<unsigned long long> configured{0};  // one bit per device
  const unsigned long long bit = 1ull << (device & 63);
  if (!(configured.load() & bit)) {
    MUI_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<T, KV8, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(smem)));
    configured.fetch_or(bit);
  }
  MUI_CUDA_CHECK(mui_launch(paged_decode_kernel<T, KV8, D, NT>, dim3(a.ctas), dim3(PA_THREADS), smem, stream, pdl, a));
  if (a.ctas > 1)
    MUI_CUDA_CHECK(mui_launch(paged_merge_kernel<T, D, NT>, dim3(static_cast<unsigned>(a.kv.batch) * a.kv.kv_heads * a.row_blocks * NT * 8),
                              dim3(PA_THREADS), 0, stream, 1, a));
  return MUI_OK;
}

template <typename T, bool KV8, int D>
mui_status_t launch_attention(cudaStream_t stream, const PaArgs& a, int pdl, int device) {
  if (pa_decode(a.G, a.max_new))
    return pa_block_rows(a.G, a.max_new) == 8 ? launch_decode<T, KV8, D, 1>(stream, a, pdl, device)
                                              : launch_decode<T, KV8, D, 2>(stream, a, pdl, device);
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
  const int G = num_q_heads / kv_heads;
  return pa_workspace(pa_ctas(di->sm_count, batch, kv_heads, G, max_new_tokens, max_context, window, sinks),
                      pa_block_rows(G, max_new_tokens), head_dim);
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
  a.q_vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && (q_strides.tok & 7) == 0 && (q_strides.head & 7) == 0;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.44269504088896341f;
  a.ctas = a.row_blocks = 1;
  // a tile is 16 rows of K and of V
  a.lead = PA_TRIPLE_COST * 4096 / (2 * PA_TILE * cache->head_dim * (cache->format == MUI_KV_E4M3 ? 1 : 2));
  if (pa_decode(G, max_new_tokens)) {
    const int block = pa_block_rows(G, max_new_tokens);
    a.row_blocks = (G * max_new_tokens + block - 1) / block;
    a.ctas = pa_ctas(di->sm_count, cache->batch, cache->kv_heads, G, max_new_tokens, max_context, window, sinks);
    const size_t need = pa_workspace(a.ctas, block, cache->head_dim);
    MUI_REQUIRE(static_cast<long long>(cache->batch) * cache->kv_heads * a.row_blocks * block <= 0x7fffffff, MUI_ERR_UNSUPPORTED,
                "batch=%d times kv_heads=%d is too large", cache->batch, cache->kv_heads);
    MUI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                              (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                MUI_ERR_INVALID_ARG, "workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
                workspace ? workspace_bytes : static_cast<size_t>(0));
    a.partials = reinterpret_cast<float*>(workspace);
  }
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define PA_GO(T, D)                                                            \
  (cache->format == MUI_KV_E4M3 ? launch_attention<T, true, D>(st, a, pdl, di->device) \
                                : launch_attention<T, false, D>(st, a, pdl, di->device))
  if (dtype == MUI_F16) return cache->head_dim == 128 ? PA_GO(__half, 128) : PA_GO(__half, 64);
  return cache->head_dim == 128 ? PA_GO(__nv_bfloat16, 128) : PA_GO(__nv_bfloat16, 64);
#undef PA_GO
}

}  // extern "C"
