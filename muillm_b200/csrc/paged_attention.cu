// Attention over a paged cache (16-bit pages, or e4m3 pages with a power-of-two scale per page and head):
//   o = sum_j softmax_j(q . k_j * scale) v_j   over the rows j a token at position p sees: j <= p and, with a window,
//   j > p - window or j < sinks.
// K and V are read once per KV head; the query heads of the group (and the new tokens of a sequence) are the rows that
// share them. Softmax is taken in one pass with a running maximum and sum in fp32.
//
// Two kernels. Up to 32 rows per KV head (decode): paged_decode_kernel, bound by the bytes of K and V; the visible rows of all
// sequences are dealt out to the CTAs evenly, and what several CTAs share is joined by paged_merge_kernel. More rows (prompts): paged_prompt_kernel, bound by the tensor cores.
#include "paged_common.cuh"
#include "tensor_map.cuh"

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
  long long* begins;  // [batch + 1] first place of each sequence and their number; nullptr: the merge works them out
  int Hq, G, ctas, row_blocks, splits, mixed, lead, max_new, window, sinks, q_vec;
  uint32_t q_flip;  // sign bits turned over in q
  float scale_log2;
};

// Length before the new tokens; 32-bit positions end at 2^31 - 1, so that no sum of a position passes 32 bits.
__device__ __forceinline__ int context_of(const PaArgs& a, int b, int count) {
  return min(__ldcg(a.kv.context_lens + b), 0x7fffffff - count);
}

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
  // kv_len: a position behind the block table may have more sinks than the table has rows
  s.n_sink = min((min(min(a.sinks, s.lo_min), s.kv_len) + PA_TILE - 1) / PA_TILE, s.first);
  s.n = s.n_sink + max(0, (s.kv_len + PA_TILE - 1) / PA_TILE - s.first);
  return s;
}
__device__ __forceinline__ int span_tile(const Span& s, int i) { return i < s.n_sink ? i : i - s.n_sink + s.first; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
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

// ---------------------------------------------------------------------------------------------------------------------
// decode: few rows per KV head
// ---------------------------------------------------------------------------------------------------------------------
// The tiles of all (sequence, KV head, block of rows) triples are laid end to end and dealt out in equal runs, so that every
// CTA streams the same number of bytes whatever the lengths are. A run that covers a triple whole writes its output; the
// others leave partial results, at most two per CTA (the triple that the run starts in and the one it ends in), which
// paged_merge_kernel joins in order.
// Measured (device time with the merge; 32 q and 8 KV heads of 128, copy bandwidth 6560 GB/s): 24 sequences of 150 to 6500
// tokens, bf16, 62 us = 5.1 TB/s; 32 sequences of 413 to 8111, e4m3, 62 us = 4.6 TB/s; one sequence of 131000, 64 q heads,
// e4m3, 57 us = 4.7 TB/s; 16 long ones with a window of 4096 and 4 sinks, 40 q heads, 53 us = 5.0 TB/s; one sequence of 300 tokens
// 13.2 us; 200 of 300 to 2500, e4m3, 135 us. About 8 us of a launch go to the chain before the first and after the last item (lengths, block table, q, merge);
// in between e4m3 is bound by its instructions: a conversion for each pair of elements, and byte permutes for V.
struct Run {
  int seq, first, count, ctx;  // sequence at the run's first place
  long long begin;             // place at which that sequence begins
};

// Length of a sequence's triples in places: `lead` places for their beginning, then one for each tile; 0: nothing to do
__device__ __forceinline__ int seq_places(const PaArgs& a, int b, Run& r) {
  paged_new_tokens(a.kv, b, r.first, r.count);
  r.ctx = context_of(a, b, r.count);
  r.seq = b;
  if (r.count == 0 || r.ctx < 0 || r.count > a.max_new) return 0;
  if (a.mixed && r.count * a.G > PA_MAX_DECODE_ROWS) return 0;  // the prompt kernel's
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
  // may be less than `lead`: a run that lies within one then has nothing to do, and the triple's first tile belongs to a later run
  return max(static_cast<long long>(PA_MIN_TILES), (total + ctas - 1) / ctas);
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

// Which elements of a word are infinite or NaN, all bits of each set. A V row that only some rows of a tile see must not reach
// the others as 0 * NaN: such elements are taken out of V and added, as they are, to the rows that see them.
template <typename T, bool KV8>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  if (KV8) return __vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu);  // e4m3 has NaN only
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  return __vcmpeq2(x & E, E);
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
  float ks, lv;  // e4m3: K scale of the page, logarithm of its V scale
};

// 4 warps; row = new token * G + head in the group; NT blocks of eight rows per CTA
template <typename T, bool KV8, int D, int NT>
__global__ void __launch_bounds__(PA_THREADS, NT == 1 ? 3 : 2) paged_decode_kernel(const PaArgs a) {
  using I = Item<KV8, D>;
  // e4m3 goes through the tensor cores as fp16, which holds every e4m3 value; so do q, after a power-of-two scaling per
  // row that brings its largest element near 1, and the probabilities
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr bool SPLIT_P = std::is_same<M, __nv_bfloat16>::value;  // probabilities as bf16 value + bf16 rest
  // Probabilities in fp16 are taken times 2^LIFT, the largest one next to the end of fp16's range, so that they have all eleven
  // bits down to 2^-29 of it (at 2^-14, without, half a million rows of little weight lose theirs together). Over e4m3 pages what is
  // rounded is the probability times V's scale, against the row's own largest such product. The references m (of the sum) and mo (of
  // the output, e4m3) stand LIFT below those maxima.
  constexpr float LIFT = std::is_same<M, __half>::value ? 15.f : 0.f;
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
    if (blockIdx.x == 0 && n == 0 && r.count > 0) {
      if (r.ctx < 0 || r.count > a.max_new) {
        mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(r.ctx < 0 ? r.ctx : r.count));
      } else if (!a.mixed || r.count * a.G <= PA_MAX_DECODE_ROWS) {
        // a window behind the block table's reach: nothing to see
        mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(r.ctx));
        uint4* row = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + static_cast<size_t>(r.first) * a.Hq * D);
        for (int e = 0; e < r.count * a.Hq * (D / 8); ++e) row[e] = make_uint4(0, 0, 0, 0);
      }
    }
    if (place >= begin && place < begin + n) {
      r.begin = begin;
      s_run = r;
    }
    if (blockIdx.x == 0 && a.begins != nullptr) {
      a.begins[s] = begin;
      if (s == a.kv.batch - 1) a.begins[s + 1] = total;
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
    float my_ks = 0.f, my_lv = 0.f, next_ks = 0.f, next_vs = 0.f;
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
            if (KV8) my_lv = log2f(next_vs);
          }
          if (phase == 16) ask_pages(grp + 16 / U);
          if (phase == 24) ask_scales();
          if ((grp * U & 31) / U == lane / U) {
            TileMeta& t = sm_meta[warp][grp & 1][lane % U];
            t.tb = my_tb;
            t.ks = my_ks;
            t.lv = my_lv;
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
          uint4 w = q_raw[n][c][e];
          w.x ^= a.q_flip;
          w.y ^= a.q_flip;
          w.z ^= a.q_flip;
          w.w ^= a.q_flip;
          unpack8<T>(w, x);
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

    float m[NT][2], mo[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = mo[n][0] = mo[n][1] = -INFINITY;
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

      unsigned shut = 0;  // tiles that some new tokens see and others do not
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tb = meta[u].tb;
        const float ks = KV8 ? meta[u].ks : 1.f;
        const bool open = tb >= 0 && tb + PA_TILE - 1 <= ctx && (tb >= lo_max || tb + PA_TILE <= a.sinks);
        if (!open && tb >= 0 && count > 1) shut |= 1u << u;
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
      bool moved = false;
      float corr[NT][2];  // of the output
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY, mv = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float t = fmaxf(s[u][n][i], s[u][n][2 + i]);
            mx = fmaxf(mx, t);
            if (KV8) mv = fmaxf(mv, t + meta[u].lv);
          }
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(MUI_FULL_MASK, mx, x));
            if (KV8) mv = fmaxf(mv, __shfl_xor_sync(MUI_FULL_MASK, mv, x));
          }
          const float mn = fmaxf(m[n][i], mx - LIFT);
          const float use = mn == -INFINITY ? 0.f : mn;
          corr[n][i] = ex2(m[n][i] - use);
          l[n][i] *= corr[n][i];
          float f[U];
          if (KV8) {
            const float vn = fmaxf(mo[n][i], mv - LIFT);
            const float use_v = vn == -INFINITY ? 0.f : vn;
            corr[n][i] = ex2(mo[n][i] - use_v);
            moved |= vn != mo[n][i];
            mo[n][i] = vn;
#pragma unroll
            for (int u = 0; u < U; ++u) f[u] = ex2(fminf(use - use_v + meta[u].lv, 120.f));  // finite: 0 stays 0
          } else {
            moved |= mn != m[n][i];
          }
          m[n][i] = mn;
          float sum = 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            s[u][n][i] = ex2(s[u][n][i] - use);
            s[u][n][2 + i] = ex2(s[u][n][2 + i] - use);
            sum += s[u][n][i] + s[u][n][2 + i];
            if (KV8) {
              s[u][n][i] *= f[u];
              s[u][n][2 + i] *= f[u];
            }
          }
          l[n][i] += sum;
        }
      if (__any_sync(MUI_FULL_MASK, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[j][n][0] *= corr[n][0];
            o[j][n][1] *= corr[n][1];
            o[j][n][2] *= corr[n][0];
            o[j][n][3] *= corr[n][1];
          }
      }
      uint32_t pb[U][NT][2], pr[U][NT][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = s[u][n][2 * h], p1 = s[u][n][2 * h + 1];
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
      // this lane's words of a V row
      auto v_words = [&](int u, int row, uint32_t(&x)[I::VW]) {
        const uint32_t at = vslot + (u * PA_TILE + row) * I::RB;
        if (I::CPR == 4) {
          lds_v2(at + (((g >> 1) ^ I::swizzle(row)) << 4) + (g & 1) * 8, x[0], x[1]);
        } else {
#pragma unroll
          for (int c = 0; c < I::VW / 4; ++c) {
            const uint4 w = lds16(at + (((c * 8 + g) ^ I::swizzle(row)) << 4));
            x[4 * c] = w.x;
            x[4 * c + 1] = w.y;
            x[4 * c + 2] = w.z;
            x[4 * c + 3] = w.w;
          }
        }
      };
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t v[4][I::VW];
#pragma unroll
        for (int r = 0; r < 4; ++r) v_words(u, 2 * tq + (r & 1) + (r >> 1) * 8, v[r]);
        if (shut >> u & 1) {
          uint32_t any = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < I::VW; ++w) any |= not_finite<M, KV8>(v[r][w]);
          if (__any_sync(MUI_FULL_MASK, any != 0)) {  // rare
#pragma unroll 1
            for (int row = 0; row < PA_TILE; ++row) {
              const int j = meta[u].tb + row;
              uint32_t x[I::VW];
              v_words(u, row, x);
#pragma unroll
              for (int w = 0; w < I::VW; ++w) {
                x[w] &= not_finite<M, KV8>(x[w]);
                constexpr int PAIRS = KV8 ? 2 : 1;
#pragma unroll
                for (int h = 0; h < PAIRS; ++h) {
                  float2 add;
                  if (KV8) {
                    add.x = x[w] >> (16 * h) & 0xffu ? __int_as_float(0x7fffffff) : 0.f;
                    add.y = x[w] >> (16 * h + 8) & 0xffu ? __int_as_float(0x7fffffff) : 0.f;
                  } else {
                    add = Elt<M>::unpack2(x[w]);
                  }
#pragma unroll
                  for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                      if (j <= hi[n][i] && (j >= lo[n][i] || j < a.sinks)) {
                        o[w * PAIRS + h][n][i] += add.x;
                        o[w * PAIRS + h][n][2 + i] += add.y;
                      }
                }
              }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int w = 0; w < I::VW; ++w) v[r][w] &= ~not_finite<M, KV8>(v[r][w]);
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
          sm_m[warp][r] = m[n][i] + LIFT;
          sm_l[warp][r] = v * exp2_int(-static_cast<int>(LIFT));
        }
        // o relative to the row's maximum, like the sum
        const float f = !KV8 ? exp2_int(-static_cast<int>(LIFT)) : mo[n][i] == -INFINITY ? 0.f : ex2(mo[n][i] - m[n][i] - LIFT);
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
// results in turn and are joined in shared memory, always in the same order. Where a sequence's places begin it works out from the
// lengths when they are one per thread, which is done while the attention kernel still runs; of larger batches (each CTA would read
// all of it) the attention kernel's first CTA leaves a table.
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
  const int places = seq_places(a, b);
  long long begin, total;
  if (a.begins == nullptr) {
    total = scan_sequences(a, 1, begin, s_warp);
    if (b == static_cast<int>(threadIdx.x)) s_begin = begin;
    __syncthreads();
    begin = s_begin;
  } else {
    pdl_wait_prior_grid();
    total = __ldcg(a.begins + a.kv.batch);
    begin = __ldcg(a.begins + b);
  }
  const long long len = run_length(total, a.ctas);
  const long long at = begin + static_cast<long long>(pair) * places;
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
// prompts: many rows per KV head, on the tcgen05 tensor cores
// ---------------------------------------------------------------------------------------------------------------------
// A CTA owns 256 rows (two groups of 128, row = new token * G + head in the group) of one sequence and KV head and walks the
// cache rows that they see, 128 at a time:
//   S_g = Q_g K^T    (128 x 128, K = D)   both operands in shared memory, K-major with the 128-byte swizzle
//   P_g = exp2(S_g * scale - reference)   one thread per row, tensor memory to tensor memory, P over S
//   O_g += P_g V     (128 x D, K = 128)   P from tensor memory, V as it lies in the cache (its head dims contiguous: MN-major)
// All of tensor memory is taken: S 2 x 128 columns, O 2 x D columns. One thread issues the MMAs, two warpgroups (one per group
// of rows) take the softmax, three warps bring K and V (16-bit pages: asynchronous copies; e4m3 pages: converted to fp16, exact, on
// the way) into a ring of four 128-row tiles. While one group's softmax runs, the tensor cores work for the other.
//
// The reference of a row's exponents is its running maximum, but moves only when the maximum is more than 8 (a factor 256)
// above it: then O is rescaled in tensor memory, which is rare after the first tiles; P stays below 2^8 and the sums are right in
// any case. P is rounded once to the type of the tensor-core operands (half a step is 2^-9 of it for bf16, 2^-12 for fp16: there P is
// taken times 2^7, so that it has all its bits down to 2^-21 of the reference).
// Bound: exp2 (16 a cycle and SM) and the MMAs need about 2050 cycles a step each.
// Measured (32 q and 8 KV heads of 128, device time; tensor cores 1651 TFLOP/s): one prompt of 8192 tokens, bf16 pages, 600 us =
// 920 TFLOP/s; three chunks of 1023 to 2049 tokens behind up to 2100, 222 us = 778 TFLOP/s (the steps alone are
// 147 us; the last round of CTAs is not full, and each of four CTAs in a row on an SM begins and ends with nothing beside it); e4m3
// pages 356 us (the three warps that convert K and V). A step takes 2.0 us, 1.6 of it MMA time: a group's softmax ends
// a little late for the other group's products. A part of the exponentials as polynomials on the fp32 pipes was slower (a
// quarter of them 231, half of them 239 us): their instructions come out of the same issue slots. So were tiles ordered by
// length over all sequences (269 us: the search costs each CTA more than it saves).
constexpr int PT_ROWS = 256, PT_GROUP = 128, PT_KEYS = 128;
constexpr int PT_SUB = PT_KEYS / PA_TILE;          // 16-row tiles of a step
constexpr int PT_SLOTS = 4;                        // ring of K and V tiles
constexpr int PT_MMA_WARP = 8, PT_LOAD_WARP = 9, PT_LOAD_WARPS = 3;
constexpr int PT_LOADERS = PT_LOAD_WARPS * 32;
constexpr int PT_THREADS = (PT_LOAD_WARP + PT_LOAD_WARPS) * 32;  // 384: 168 registers a thread
constexpr int PT_MAX_SPLITS = 16;
constexpr float PT_SLACK = 8.f;

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit_to(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of a converged warp. Unlike `lane == 0` it leaves the code around it warp-uniform, so that descriptors stay in
// uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[smem] B[smem]^T
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 consecutive 32-bit columns of this thread's tensor-memory lane; there after tmem_load_wait
__device__ __forceinline__ void tmem_ask32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
// the registers are named so that nothing that uses them moves above the wait
__device__ __forceinline__ void tmem_load_wait(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
        "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
        "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
        "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ask32(addr, r);
  tmem_load_wait(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart. K-major: a row
// is 64 elements along K; the leading offset is not used. MN-major: a row is 64 elements along N, the rows run along K, and
// `lead` is the distance from one block of 64 to the next along N.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// kind::f16 with fp32 accumulators: M = 128; b_mn: B is MN-major
__device__ __forceinline__ uint32_t f16_idesc(int is_bf16, int n, int b_mn) {
  return 1u << 4 | static_cast<uint32_t>(is_bf16) << 7 | static_cast<uint32_t>(is_bf16) << 10 |
         static_cast<uint32_t>(b_mn) << 16 | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(128 >> 4) << 24;
}

// Which rows a CTA owns and what they see. false: nothing to do. The prompt kernel runs with cu_tokens only: without them a
// sequence has one new token, at most 32 rows.
struct PromptTile {
  int b, first, count, ctx, r0, R;
  Span sp;
  int steps, per, active;  // steps of 128 cache rows; steps per split; splits that have any
};
__device__ __forceinline__ bool prompt_tile(const PaArgs& a, int x, PromptTile& t) {
  // tiles are numbered through: sequence b's start at floor(cu[b] * G / 256) + b
  const int32_t* cu = a.kv.cu;
  auto start = [&](int k) { return static_cast<int>(static_cast<long long>(__ldcg(cu + k)) * a.G / PT_ROWS) + k; };
  t.b = warp_count_le(a.kv.batch, x, [&](int k) { return start(k + 1); });
  if (t.b >= a.kv.batch) return false;
  const int tile = x - start(t.b);
  paged_new_tokens(a.kv, t.b, t.first, t.count);
  t.ctx = context_of(a, t.b, t.count);
  t.r0 = tile * PT_ROWS;
  t.R = t.count * a.G;
  if (tile < 0 || t.r0 >= t.R) return false;
  if (t.ctx < 0 || t.count > a.max_new) {
    if ((threadIdx.x & 31) == 0) mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(t.ctx < 0 ? t.ctx : t.count));
    return false;
  }
  if (a.mixed && t.R <= PA_MAX_DECODE_ROWS) return false;  // the decode kernel's
  const int lo = t.r0 / a.G, hi = (min(t.R, t.r0 + PT_ROWS) - 1) / a.G;  // new tokens of this tile
  t.sp = visible_span(a, t.ctx + lo, hi - lo + 1);
  t.steps = (t.sp.n + PT_SUB - 1) / PT_SUB;
  t.per = max(2, (t.steps + a.splits - 1) / a.splits);
  t.active = max(1, (t.steps + t.per - 1) / t.per);
  return true;
}

// The rows of a CTA again, a thread per row on the fp32 pipes, where one of them came out infinite or NaN: the tensor cores
// multiply V rows that a row does not see by 0, and 0 * NaN must not reach it. Here only what a row sees is added. About twenty
// times slower. q is still in shared memory; the ring is idle. (Inlined: as a function of its own it made every call 4 % slower.)
template <typename T, bool KV8, int D>
__device__ __forceinline__ void prompt_again(const PaArgs& a, uint32_t q_tiles, const float* q_back) {
  using M = typename std::conditional<KV8, __half, T>::type;
  const int kvh = blockIdx.x % a.kv.kv_heads, split = blockIdx.y, row = threadIdx.x;
  PromptTile t;
  if (!prompt_tile(a, static_cast<int>((gridDim.x - 1 - blockIdx.x) / a.kv.kv_heads), t)) return;
  const int rr = t.r0 + row;
  const bool mine = rr < t.R;
  const int pos = mine ? t.ctx + rr / a.G : -1, lo = a.window > 0 ? pos - a.window + 1 : 0;
  const uint32_t ring = q_tiles + PT_ROWS * D * 2;  // K, then V: 16 rows of fp32 each
  const uint32_t q_row = q_tiles + row / PT_GROUP * (PT_GROUP * D * 2) + row % PT_GROUP * 128;
  const float sc = KV8 ? a.scale_log2 * q_back[row] : fmaxf(a.scale_log2, 1e-37f);
  auto ldf4 = [](uint32_t at) {
    const uint4 w = lds16(at);
    return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  };
  float m = -INFINITY, l = 0.f, o[D];
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = 0.f;
  const int i_begin = split * t.per * PT_SUB, i_end = min(t.sp.n, i_begin + t.per * PT_SUB);
#pragma unroll 1
  for (int i = i_begin; i < i_end; ++i) {
    const int b0 = span_tile(t.sp, i) * PA_TILE;
    const int page = __ldcg(a.kv.block_table + static_cast<size_t>(t.b) * a.kv.table_stride + (b0 >> a.kv.page_shift));
    if (page < 0 || page >= a.kv.num_pages) continue;  // recorded before
    const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + kvh;
    const size_t first = ((head << a.kv.page_shift) + (b0 & ((1 << a.kv.page_shift) - 1))) * D;
    const float ks = KV8 ? __ldcg(a.kv.k_scales + head) : 1.f, vs = KV8 ? __ldcg(a.kv.v_scales + head) : 1.f;
    asm volatile("bar.sync 1, %0;" ::"n"(PT_ROWS) : "memory");
    for (int e = row; e < 2 * PA_TILE * D; e += PT_ROWS) {
      const size_t at = first + e % (PA_TILE * D);
      const void* pages = e < PA_TILE * D ? a.kv.k_pages : a.kv.v_pages;
      float x;
      if (KV8)
        x = Elt<__half>::unpack2(e4m3_to_half2(reinterpret_cast<const unsigned char*>(pages)[at])).x;
      else
        x = Elt<T>::to_f32(reinterpret_cast<const T*>(pages)[at]);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + e * 4), "f"(x) : "memory");
    }
    asm volatile("bar.sync 1, %0;" ::"n"(PT_ROWS) : "memory");
#pragma unroll 1
    for (int r = 0; r < PA_TILE; ++r) {
      const int j = b0 + r;
      if (j > pos || j >= t.sp.kv_len || (j < lo && j >= a.sinks)) continue;
      float s = 0.f;
#pragma unroll 1
      for (int ch = 0; ch < D / 8; ++ch) {
        const uint4 w = lds16(q_row + (ch >> 3) * (PT_GROUP * 128) + (((ch & 7) ^ (row & 7)) << 4));
        float q[8];
        unpack8<M>(w, q);
        const float4 k0 = ldf4(ring + (r * D + ch * 8) * 4), k1 = ldf4(ring + (r * D + ch * 8) * 4 + 16);
        s = fmaf(q[0], k0.x, fmaf(q[1], k0.y, fmaf(q[2], k0.z, fmaf(q[3], k0.w, s))));
        s = fmaf(q[4], k1.x, fmaf(q[5], k1.y, fmaf(q[6], k1.z, fmaf(q[7], k1.w, s))));
      }
      s *= KV8 ? fmaxf(sc * ks, 1e-37f) : sc;
      if (s > m) {
        const float f = m == -INFINITY ? 0.f : ex2(m - s);
        m = s;
        l *= f;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] *= f;
      }
      const float p = ex2(s - (m == -INFINITY ? 0.f : m));
      l += p;
#pragma unroll
      for (int d = 0; d < D; d += 4) {
        const float4 v = ldf4(ring + ((PA_TILE + r) * D + d) * 4);
        o[d] = fmaf(p * vs, v.x, o[d]);
        o[d + 1] = fmaf(p * vs, v.y, o[d + 1]);
        o[d + 2] = fmaf(p * vs, v.z, o[d + 2]);
        o[d + 3] = fmaf(p * vs, v.w, o[d + 3]);
      }
    }
  }
  if (!mine) return;
  const size_t out_row = static_cast<size_t>(t.first + rr / a.G) * a.Hq + kvh * a.G + rr % a.G;
  if (t.active == 1) {
    const float norm = l != 0.f ? 1.f / l : 0.f;
    T* out = reinterpret_cast<T*>(a.out) + out_row * D;
#pragma unroll
    for (int d = 0; d < D; ++d) out[d] = Elt<T>::from_f32(o[d] * norm);
  } else {
    float* part = a.partials + (out_row * a.splits + split) * (D + 2);
    part[0] = m;
    part[1] = l;
#pragma unroll
    for (int d = 0; d < D; ++d) part[2 + d] = o[d];
  }
}

template <typename T, bool KV8, int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PaArgs a) {
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr int QT = PT_GROUP * D * 2;                 // bytes of a group's Q
  constexpr int KT = PT_KEYS * D * 2;                  // bytes of a K or V tile
  constexpr int BLOCK = PT_KEYS * 128;                 // bytes of one 64-element block of a tile (Q, K or V)
  constexpr uint32_t TM_S = 0, TM_O = 2 * PT_KEYS;     // tensor-memory columns
  constexpr float PT_LIFT = std::is_same<M, __half>::value ? 7.f : 0.f;  // with the slack 2^15 at most, of fp16's 2^16
  extern __shared__ unsigned char pt_raw[];
  __shared__ uint64_t kv_full[PT_SLOTS], kv_empty[PT_SLOTS], s_full[2], p_half[2], p_full[2], pv_done[2];
  __shared__ float q_back[PT_ROWS];
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s, redo_s;
  const uint32_t tiles = (smem_u32(pt_raw) + 1023u) & ~1023u;  // Q0, Q1, then the ring
  const uint32_t ring = tiles + 2 * QT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // KV heads fastest, the longest spans first
  const int kvh = blockIdx.x % a.kv.kv_heads, split = blockIdx.y;
  volatile int* abort_flag = &abort_s;

  pdl_wait_prior_grid();
  pdl_launch_dependents();
  PromptTile t;
  if (!prompt_tile(a, static_cast<int>((gridDim.x - 1 - blockIdx.x) / a.kv.kv_heads), t)) return;
  if (split >= t.active) return;
  const int i_begin = split * t.per * PT_SUB, i_end = min(t.sp.n, i_begin + t.per * PT_SUB);  // 16-row tiles of this split
  const int n = (i_end - i_begin + PT_SUB - 1) / PT_SUB;
  const bool two = t.R - t.r0 > PT_GROUP;  // the second group has rows
  if (t.sp.kv_len < t.ctx + (min(t.R, t.r0 + PT_ROWS) - 1) / a.G + 1 && tid == 0)
    mui_dev_set_status(MUI_DEV_BAD_LENGTH, static_cast<unsigned>(t.sp.kv_len));

  if (tid == 0) {
    for (int i = 0; i < PT_SLOTS; ++i) {
      mbar_init(&kv_full[i], KV8 ? PT_LOADERS : 33);
      mbar_init(&kv_empty[i], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_half[g], PT_GROUP);
      mbar_init(&p_full[g], PT_GROUP);
      mbar_init(&pv_done[g], 1);
    }
    abort_s = redo_s = 0;
    mbar_fence_init();
  }
  if (warp == PT_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Q into shared memory: eight lanes (D = 64) or sixteen per row. e4m3 pages: as fp16, brought near 1 by a power of two per row.
  {
    constexpr int LPR = D / 8;
    for (int i = tid; i < PT_ROWS * LPR; i += PT_THREADS) {  // a row's lanes are neighbours in one warp, and whole warps take part
      const int r = i / LPR, ch = i % LPR, rr = t.r0 + r;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (rr < t.R)
        w = load_q8<T>(reinterpret_cast<const T*>(a.q) + (t.first + rr / a.G) * a.qs.tok + (kvh * a.G + rr % a.G) * a.qs.head + ch * 8,
                       a.q_vec);
      w.x ^= a.q_flip;
      w.y ^= a.q_flip;
      w.z ^= a.q_flip;
      w.w ^= a.q_flip;
      if (KV8) {
        float x[8], amax = 0.f;
        unpack8<T>(w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
        const unsigned mask = LPR == 16 ? 0xffffu << (lane & 16) : 0xffu << (lane & 24);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
        const int e2 = min(100, max(-100, static_cast<int>(__float_as_uint(amax) >> 23) - 127));
        const float mul = exp2_int(-e2);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= mul;
        w = pack8<__half>(x);
        if (ch == 0) q_back[r] = exp2_int(e2);
      }
      const int c = ch & 7;
      const uint32_t dst = tiles + (r / PT_GROUP) * QT + (ch >> 3) * BLOCK + (r % PT_GROUP) * 128 + ((c ^ (r & 7)) << 4);
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_s;
  // a wait that runs out records itself once and makes every other one give up
  auto wait = [&](uint64_t* bar, int phase, unsigned what) {
    if (mbar_wait_bounded(bar, phase & 1, abort_flag)) return true;
    if (!*abort_flag) mui_dev_set_status(MUI_DEV_TIMEOUT_FULL, 0x800000u | what);
    *abort_flag = 1;
    return false;
  };
  const int32_t* table = a.kv.block_table + static_cast<size_t>(t.b) * a.kv.table_stride;
  // lanes 0-7: page (-1: none) and first row (-1) of the 16-row tiles of step j
  auto find_tile = [&](int j, int& page, int& tb, bool record) {
    const int i = i_begin + j * PT_SUB + lane;
    page = tb = -1;
    if (lane < PT_SUB && i < i_end) {
      const int row = span_tile(t.sp, i) * PA_TILE;
      const int p = __ldcg(table + (row >> a.kv.page_shift));
      if (p >= 0 && p < a.kv.num_pages) {
        page = p;
        tb = row;
      } else if (record) {
        mui_dev_set_status(MUI_DEV_BAD_PAGE, static_cast<unsigned>(t.b));
      }
    }
  };

  if (KV8 && warp >= PT_LOAD_WARP) {
    // ------------------------------ K and V, e4m3: converted by three warps ------------------------------
    const int lw = warp - PT_LOAD_WARP;
    constexpr int RB = D, CPR = RB / 16;                         // bytes and 16-byte chunks of a cache row
    constexpr int RPI = 32 / CPR;                                // rows a warp copies at a time
    // A step is 16 units of eight rows; a warp takes every third one, so that addresses are worked out once per unit.
    constexpr int UNITS = 2 * PT_SUB, TURNS = (UNITS + PT_LOAD_WARPS - 1) / PT_LOAD_WARPS, CPU = 8 / RPI;
    const int ch = lane % CPR, row0 = lane / CPR;
    // where this lane's chunks of a unit go: 16-bit chunk c of row r sits at block c / 8, row r, chunk (c % 8) ^ (r % 8)
    auto place = [&](int r, int c) { return static_cast<uint32_t>((c >> 3) * BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };
    uint32_t at[CPU][2];
#pragma unroll
    for (int i = 0; i < CPU; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) at[i][h] = place(i * RPI + row0, 2 * ch + h);
    int page, tb, next_page, next_tb;
    find_tile(0, page, tb, true);
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      next_page = next_tb = -1;
      if (j + 1 < n) find_tile(j + 1, next_page, next_tb, true);
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const int it = 2 * j + which, slot = it % PT_SLOTS;
        const unsigned char* pages = reinterpret_cast<const unsigned char*>(which == 0 ? a.kv.k_pages : a.kv.v_pages);
        const uint32_t dst = ring + slot * KT;
        // calls f(turn, unit, lane's source, whole, first cache row) for the warp's units
        auto units = [&](auto f) {
#pragma unroll
          for (int k = 0; k < TURNS; ++k) {
            const int u = k * PT_LOAD_WARPS + lw;
            if (u >= UNITS) break;
            const int pg = __shfl_sync(MUI_FULL_MASK, page, u >> 1), b0 = __shfl_sync(MUI_FULL_MASK, tb, u >> 1);
            const int first = b0 < 0 ? -PA_TILE : b0 + (u & 1) * 8;
            const size_t row = ((static_cast<size_t>(max(pg, 0)) * a.kv.kv_heads + kvh) << a.kv.page_shift) +
                               (max(first, 0) & ((1 << a.kv.page_shift) - 1));
            const bool whole = first >= 0 && first + 8 <= t.sp.kv_len && (first >= t.sp.lo_min || first + 8 <= a.sinks);
            f(k, u, pages + (row + row0) * RB + ch * 16, whole, first);
          }
        };
        // whether anybody of this tile sees a cache row; zeros stand for the others: what they hold must not matter
        auto seen = [&](int first, int r) {
          const int jr = first + r;
          return first >= 0 && jr < t.sp.kv_len && (jr >= t.sp.lo_min || jr < a.sinks);
        };
        auto slot_free = [&]() {
          if (it >= PT_SLOTS) ok = __all_sync(MUI_FULL_MASK, wait(&kv_empty[slot], it / PT_SLOTS - 1, 0x100 + slot));
          return ok;
        };
        {
          uint4 hold[TURNS][CPU];  // requested before the slot is free
          units([&](int k, int, const unsigned char* src, bool whole, int first) {
#pragma unroll
            for (int i = 0; i < CPU; ++i)
              hold[k][i] = whole || seen(first, i * RPI + row0) ? ld_stream16(src + i * RPI * RB) : make_uint4(0, 0, 0, 0);
          });
          if (!slot_free()) break;
#pragma unroll
          for (int k = 0; k < TURNS; ++k) {
            const int u = k * PT_LOAD_WARPS + lw;
            if (u >= UNITS) break;
#pragma unroll
            for (int i = 0; i < CPU; ++i) {
              const uint32_t w[4] = {hold[k][i].x, hold[k][i].y, hold[k][i].z, hold[k][i].w};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w0 = w[2 * h], w1 = w[2 * h + 1];
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + u * 1024 + at[i][h]),
                             "r"(e4m3_to_half2((uint16_t)w0)), "r"(e4m3_to_half2((uint16_t)(w0 >> 16))),
                             "r"(e4m3_to_half2((uint16_t)w1)), "r"(e4m3_to_half2((uint16_t)(w1 >> 16)))
                             : "memory");
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&kv_full[slot]);
        }
      }
      page = next_page;
      tb = next_tb;
    }
  } else if (!KV8 && warp >= PT_LOAD_WARP) {
    // ------------------------------ K and V, 16-bit: one warp, tile copies of 16 rows x 64 elements ------------------------------
    if (warp == PT_LOAD_WARP) {
      constexpr int RB = D * 2, CPR = RB / 16, RPI = 32 / CPR;
      const int ch = lane % CPR, row0 = lane / CPR;
      int page, tb, next_page, next_tb;
      find_tile(0, page, tb, true);
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        next_page = next_tb = -1;
        if (j + 1 < n) find_tile(j + 1, next_page, next_tb, true);
        // lanes 0-7, a 16-row tile each: seen whole by somebody of this CTA's rows, or to be copied row by row
        const int row = ((max(page, 0) * a.kv.kv_heads + kvh) << a.kv.page_shift) + (max(tb, 0) & ((1 << a.kv.page_shift) - 1));
        const bool whole = tb >= 0 && tb + PA_TILE <= t.sp.kv_len && (tb >= t.sp.lo_min || tb + PA_TILE <= a.sinks);
        const unsigned mask = __ballot_sync(MUI_FULL_MASK, lane < PT_SUB && whole);
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const int it = 2 * j + which, slot = it % PT_SLOTS;
          const uint32_t dst = ring + slot * KT;
          if (it >= PT_SLOTS) ok = __all_sync(MUI_FULL_MASK, wait(&kv_empty[slot], it / PT_SLOTS - 1, 0x100 + slot));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[slot], __popc(mask) * (PA_TILE * RB));
          __syncwarp();
          if (mask >> lane & 1) {
            const CUtensorMap* map = which == 0 ? &map_k : &map_v;
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              asm volatile(
                  "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                      dst + h * BLOCK + lane * (PA_TILE * 128)),
                  "l"(reinterpret_cast<uint64_t>(map)), "r"(h * 64), "r"(row), "r"(smem_u32(&kv_full[slot]))
                  : "memory");
          }
          // the others: rows that nobody of this tile sees are zeros (what they hold must not matter)
          for (unsigned left = ~mask & ((1u << PT_SUB) - 1); left; left &= left - 1) {
            const int sub = __ffs(left) - 1;
            const int first = __shfl_sync(MUI_FULL_MASK, tb, sub), from = __shfl_sync(MUI_FULL_MASK, row, sub);
            const unsigned char* src = reinterpret_cast<const unsigned char*>(which == 0 ? a.kv.k_pages : a.kv.v_pages) +
                                       static_cast<size_t>(from) * RB + ch * 16;
#pragma unroll
            for (int r = row0; r < PA_TILE; r += RPI) {
              const int jr = first + r;
              const bool see = first >= 0 && jr < t.sp.kv_len && (jr >= t.sp.lo_min || jr < a.sinks);
              copy16(dst + (ch >> 3) * BLOCK + (sub * PA_TILE + r) * 128 + (((ch & 7) ^ (r & 7)) << 4), src + r * RB, see ? 16 : 0);
            }
          }
          // arrives when this lane's copies, if any, have landed
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&kv_full[slot])) : "memory");
        }
        page = next_page;
        tb = next_tb;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (!ok) {  // leave no tile copy in flight behind: the last four items that were begun
        int none = 0;
        for (int i = 0; i < PT_SLOTS; ++i) (void)mbar_wait_bounded(&kv_full[i], 0, &none);
      }
    }
  } else if (warp == PT_MMA_WARP) {
    // ------------------------------ MMAs ------------------------------
    {
      const int bf = std::is_same<M, __nv_bfloat16>::value;
      const uint32_t id_s = f16_idesc(bf, PT_KEYS, 0), id_o = f16_idesc(bf, D, 1);
      // one thread issues: a descriptor per operand, its address field (16-byte units) moved on
      auto scores = [&](int g, int slot) {
        const uint64_t da = sw128_desc(tiles + g * QT, 16), db = sw128_desc(ring + slot * KT, 16);
        const uint32_t d = tmem + TM_S + g * PT_KEYS;
        if (elect_one())
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = ((k >> 2) * BLOCK + (k & 3) * 32) >> 4;
          mma_ss(d, da + off, db + off, id_s, k != 0);
        }
      };
      auto output = [&](int g, int slot, int half, bool more) {
        const uint64_t db = sw128_desc(ring + slot * KT + half * (PT_KEYS / 2) * 128, BLOCK);
        const uint32_t d = tmem + TM_O + g * D, p = tmem + TM_S + g * PT_KEYS + half * (PT_KEYS / 4);
        if (elect_one()) {
          mma_ts(d, p, db, id_o, more);
#pragma unroll
          for (int k = 1; k < PT_KEYS / 32; ++k) mma_ts(d, p + k * 8, db + k * (2048 >> 4), id_o, 1);
        }
      };
      bool ok = n == 0 || __all_sync(MUI_FULL_MASK, wait(&kv_full[0], 0, 0x200));
      // the whole warp waits and one lane, always the same, issues and commits
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit_to(bar);
        __syncwarp();
      };
      // what cp.async wrote is ordered before the tensor cores' reads by a fence on this side (tile copies need none)
      auto fence = [&]() {
        tc_after();
        if (!KV8) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      };
      if (ok && n > 0) {
        fence();
        scores(0, 0);
        commit(&s_full[0]);
        if (two) {
          scores(1, 0);
          commit(&s_full[1]);
        }
        commit(&kv_empty[0]);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 2, vs = vi % PT_SLOTS, ks = ki % PT_SLOTS;
        ok = __all_sync(MUI_FULL_MASK, wait(&kv_full[vs], vi / PT_SLOTS, 0x210) && wait(&p_half[0], j, 0x220));
        if (!ok) break;
        fence();
        output(0, vs, 0, j > 0);
        ok = __all_sync(MUI_FULL_MASK, wait(&p_full[0], j, 0x221));
        if (!ok) break;
        tc_after();
        output(0, vs, 1, true);
        commit(&pv_done[0]);
        if (j + 1 < n) {
          ok = __all_sync(MUI_FULL_MASK, wait(&kv_full[ks], ki / PT_SLOTS, 0x230));
          if (!ok) break;
          fence();
          scores(0, ks);
          commit(&s_full[0]);
        }
        if (two) {
          ok = __all_sync(MUI_FULL_MASK, wait(&p_half[1], j, 0x240));
          if (!ok) break;
          tc_after();
          output(1, vs, 0, j > 0);
          ok = __all_sync(MUI_FULL_MASK, wait(&p_full[1], j, 0x241));
          if (!ok) break;
          tc_after();
          output(1, vs, 1, true);
          commit(&pv_done[1]);
        }
        commit(&kv_empty[vs]);
        if (j + 1 < n) {
          if (two) {
            scores(1, ks);
            commit(&s_full[1]);
          }
          commit(&kv_empty[ks]);
        }
      }
      if (!ok) {  // leave no MMA in flight behind (slot 0's barrier is not waited for by anyone any more)
        commit(&pv_done[0]);
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ softmax: a thread per row ------------------------------
    const int g = warp >> 2, row = (warp & 3) * 32 + lane;
    if (g == 0 || two) {
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + TM_S + g * PT_KEYS, to = tmem + lanes + TM_O + g * D;
      const int rr = t.r0 + g * PT_GROUP + row;
      const bool mine = rr < t.R;
      const int pos = t.ctx + (mine ? rr / a.G : 0);
      const int hi = mine ? pos : -1, lo = a.window > 0 ? pos - a.window + 1 : 0;
      // what all rows of the group see without looking: rows from lo_all (or sinks) to hi_all
      const int last_row = min(t.R, t.r0 + (g + 1) * PT_GROUP) - 1;
      const int hi_all = t.ctx + (t.r0 + g * PT_GROUP) / a.G;
      const int lo_all = a.window > 0 ? t.ctx + last_row / a.G - a.window + 1 : 0;
      const float sc = KV8 ? a.scale_log2 * q_back[g * PT_GROUP + row] : fmaxf(a.scale_log2, 1e-37f);
      // references of the sum and, over e4m3 pages, of the output: there what is rounded is the probability times V's scale, against
      // the row's own largest such product
      float ref = -INFINITY, vref = -INFINITY, l = 0.f;
      int page, tb, next_page, next_tb;
      float ks = 0.f, vs = 0.f;
      auto scales = [&](int p, float& k, float& v) {
        k = v = 0.f;
        if (KV8 && p >= 0) {
          const size_t head = static_cast<size_t>(p) * a.kv.kv_heads + kvh;
          k = __ldcg(a.kv.k_scales + head);
          v = __ldcg(a.kv.v_scales + head);
        }
      };
      find_tile(0, page, tb, false);
      scales(page, ks, vs);
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        next_page = next_tb = -1;
        if (j + 1 < n) find_tile(j + 1, next_page, next_tb, false);
        // every row of the step is seen by every row of the group
        const bool whole = lane >= PT_SUB || (tb >= 0 && tb + PA_TILE - 1 <= hi_all && (tb >= lo_all || tb + PA_TILE <= a.sinks));
        const bool open = __all_sync(MUI_FULL_MASK, whole);
        ok = __all_sync(MUI_FULL_MASK, wait(&s_full[g], j, 0x300 + g));
        if (!ok) break;
        tc_after();
        // factor of the scores of 16 columns; above 0, since -infinity stands for what a row does not see
        auto factor_of = [&](int sub) { return KV8 ? fmaxf(sc * __shfl_sync(MUI_FULL_MASK, ks, sub), 1e-37f) : sc; };
        const float lv = KV8 ? log2f(vs) : 0.f;
        float mx = -INFINITY, mv = -INFINITY;
        auto see_top = [&](int sub, float x) {  // the largest score of 16 columns
          mx = fmaxf(mx, x);
          if (KV8) mv = fmaxf(mv, x + __shfl_sync(MUI_FULL_MASK, lv, sub));
        };
        if (open) {
          uint32_t s0[32], s1[32];
          auto top = [&](int c, const uint32_t(&s)[32]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float m0 = __uint_as_float(s[16 * h]), m1 = __uint_as_float(s[16 * h + 1]);
#pragma unroll
              for (int e = 2; e < 16; e += 2) {
                m0 = fmaxf(m0, __uint_as_float(s[16 * h + e]));
                m1 = fmaxf(m1, __uint_as_float(s[16 * h + e + 1]));
              }
              see_top(2 * c + h, fmaxf(m0, m1) * factor_of(2 * c + h));
            }
          };
          tmem_ask32(ts, s0);
          tmem_load_wait(s0);
          tmem_ask32(ts + 32, s1);
          top(0, s0);
          tmem_load_wait(s1);
          tmem_ask32(ts + 64, s0);
          top(1, s1);
          tmem_load_wait(s0);
          tmem_ask32(ts + 96, s1);
          top(2, s0);
          tmem_load_wait(s1);
          top(3, s1);
        } else {
          // masked scores are written back, so that what follows need not know
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            tmem_load32(ts + c * 32, s);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = factor_of(2 * c + h);
              const int b0 = __shfl_sync(MUI_FULL_MASK, tb, 2 * c + h);
              // bit e: this row sees column b0 + e
              auto below = [&](int x) { return (1u << min(max(x, 0), PA_TILE)) - 1u; };
              const unsigned see =
                  b0 < 0 ? 0u : below(hi - b0 + 1) & (~below(lo - b0) | below(min(a.sinks, 0x7fffffff - PA_TILE) - b0));
              uint32_t w[16];
              float top = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x = see >> e & 1 ? s[16 * h + e] : -INFINITY;
                top = fmaxf(top, x);
                w[e] = __float_as_uint(x);
              }
              see_top(2 * c + h, top * f);
              tmem_store16(ts + c * 32 + 16 * h, w);
            }
          }
          tmem_store_wait();
        }
        float factor = 1.f;  // of the output so far
        if (mx > ref + PT_SLACK || ref == -INFINITY) {
          factor = ref == -INFINITY ? 0.f : ex2(ref - mx);
          l *= factor;
          ref = mx;
        }
        if (KV8) {
          factor = 1.f;
          if (mv > vref + PT_SLACK || vref == -INFINITY) {
            factor = vref == -INFINITY ? 0.f : ex2(vref - mv);
            vref = mv;
          }
        }
        if (j > 0 && __any_sync(MUI_FULL_MASK, factor != 1.f)) {
          ok = __all_sync(MUI_FULL_MASK, wait(&pv_done[g], j - 1, 0x310 + g));
          if (!ok) break;
          tc_after();
          // a row without anything so far has nothing in O
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_load32(to + c * 32, o);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[16 * h + e] * factor);
              tmem_store16(to + c * 32 + 16 * h, w);
            }
          }
        }
        const float ref0 = ref == -INFINITY ? 0.f : ref, use = PT_LIFT - ref0;
        const float turn = KV8 ? ref0 - (vref == -INFINITY ? 0.f : vref) : 0.f;
        {
          uint32_t s0[32], s1[32];
          float2 sum = make_float2(0.f, 0.f);
          auto weigh = [&](int c, const uint32_t(&s)[32]) {
            uint32_t w[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = factor_of(2 * c + h);
              // finite: 0 stays 0
              const float pf = KV8 ? ex2(fminf(turn + __shfl_sync(MUI_FULL_MASK, lv, 2 * c + h), 120.f)) : 1.f;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float2 p = fma2(make_float2(__uint_as_float(s[16 * h + e]), __uint_as_float(s[16 * h + e + 1])),
                                make_float2(f, f), make_float2(use, use));
                p.x = ex2(p.x);
                p.y = ex2(p.y);
                sum = add2(sum, p);
                w[8 * h + e / 2] = KV8 ? Elt<M>::pack2(p.x * pf, p.y * pf) : Elt<M>::pack2(p.x, p.y);
              }
            }
            tmem_store16(ts + c * 16, w);  // columns that have been read
          };
          tmem_ask32(ts, s0);
          tmem_load_wait(s0);
          tmem_ask32(ts + 32, s1);
          weigh(0, s0);
          tmem_load_wait(s1);
          tmem_ask32(ts + 64, s0);
          weigh(1, s1);
          tmem_load_wait(s0);
          tmem_store_wait();
          tc_before();
          mbar_arrive(&p_half[g]);  // the first 64 cache rows can be multiplied
          tmem_ask32(ts + 96, s1);
          weigh(2, s0);
          tmem_load_wait(s1);
          weigh(3, s1);
          l += sum.x + sum.y;
        }
        tmem_store_wait();
        tc_before();
        mbar_arrive(&p_full[g]);
        page = next_page;
        tb = next_tb;
        scales(page, ks, vs);
      }
      if (ok && n > 0) ok = __all_sync(MUI_FULL_MASK, wait(&pv_done[g], n - 1, 0x320 + g));
      tc_after();
      if (ok) {
        const bool direct = t.active == 1;
        l *= exp2_int(-static_cast<int>(PT_LIFT));
        const float back = !KV8 ? exp2_int(-static_cast<int>(PT_LIFT)) : vref == -INFINITY ? 0.f : ex2(vref - ref - PT_LIFT);
        const float norm = direct ? (l != 0.f ? back / l : 0.f) : back;
        const size_t out_row = static_cast<size_t>(t.first + rr / a.G) * a.Hq + kvh * a.G + rr % a.G;
        float* part = a.partials + (out_row * a.splits + split) * (D + 2);
        if (mine && !direct) {
          part[0] = ref;
          part[1] = l;
        }
        float2 check[4] = {};  // NaN when any element is infinite or NaN
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (n > 0) {
            tmem_load32(to + c * 32, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (!mine) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= norm;
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            check[e / 2 & 3] = fma2(make_float2(o[e], o[e + 1]), make_float2(0.f, 0.f), check[e / 2 & 3]);
          if (direct) {
            uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + out_row * D + c * 32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              out[e] = make_uint4(Elt<T>::pack2(o[8 * e], o[8 * e + 1]), Elt<T>::pack2(o[8 * e + 2], o[8 * e + 3]),
                                  Elt<T>::pack2(o[8 * e + 4], o[8 * e + 5]), Elt<T>::pack2(o[8 * e + 6], o[8 * e + 7]));
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              *reinterpret_cast<float2*>(part + 2 + c * 32 + 2 * e) = make_float2(o[2 * e], o[2 * e + 1]);
          }
        }
        check[0] = add2(add2(check[0], check[1]), add2(check[2], check[3]));
        if (check[0].x + check[0].y != 0.f) redo_s = 1;
      }
    }
  }
  tc_before();
  __syncthreads();
  if (redo_s && tid < PT_ROWS) prompt_again<T, KV8, D>(a, tiles, q_back);
  if (warp == PT_MMA_WARP) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the splits of the prompt kernel in order: a warp per (new token, query head).
template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS) paged_prompt_merge_kernel(const PaArgs a) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * PA_WARPS + (threadIdx.x >> 5);
  const int tok = static_cast<int>(row / a.Hq), head = static_cast<int>(row % a.Hq);
  int active = 0;
  if (tok < a.kv.total) {
    const int32_t* cu = a.kv.cu;
    const int b = warp_count_le(a.kv.batch, tok, [&](int k) { return __ldcg(cu + 1 + k); });
    if (b < a.kv.batch) {
      int first, count;
      paged_new_tokens(a.kv, b, first, count);
      const int x = ((tok - first) * a.G + head % a.G) / PT_ROWS;
      PromptTile t;
      const int start = static_cast<int>(static_cast<long long>(__ldcg(cu + b)) * a.G / PT_ROWS) + b;
      if (prompt_tile(a, start + x, t)) active = t.active;
    }
  }
  pdl_wait_prior_grid();  // every thread, also one without work: this grid must not be done before the attention kernel is
  if (active <= 1) return;
  const float* p = a.partials + static_cast<size_t>(row) * a.splits * (D + 2);
  float m[PT_MAX_SPLITS], mm = -INFINITY;
#pragma unroll
  for (int s = 0; s < PT_MAX_SPLITS; ++s) {
    m[s] = s < active ? __ldcg(p + s * (D + 2)) : -INFINITY;
    mm = fmaxf(mm, m[s]);
  }
  const float use = mm == -INFINITY ? 0.f : mm;
  float l = 0.f, o[D / 32] = {};
#pragma unroll
  for (int s = 0; s < PT_MAX_SPLITS; ++s) {
    if (s >= active) break;
    const float f = ex2(m[s] - use);
    l = fmaf(__ldcg(p + s * (D + 2) + 1), f, l);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(p + s * (D + 2) + 2) + e * 32 + lane);
      o[2 * e] = fmaf(v.x, f, o[2 * e]);
      o[2 * e + 1] = fmaf(v.y, f, o[2 * e + 1]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(a.out) + static_cast<size_t>(row) * (D / 2);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[e * 32 + lane] = Elt<T>::pack2(o[2 * e] * inv, o[2 * e + 1] * inv);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
// What a call launches and the scratch it needs, from sizes alone.
struct PaPlan {
  // Up to 32 rows per sequence: the decode kernel; more: the prompt kernel. Where short and long sequences can meet in one call
  // both run, each on its own (mixed).
  bool decode, prompt;
  int block, row_blocks, ctas;  // decode: rows per block (8, else blocks of 16)
  int tiles, splits;            // prompt
  size_t begins_at, decode_bytes, bytes;  // begins_at: offset of the table of first places, 0: none
};
bool pa_plan(const MuiDeviceInfo& di, int total, int batch, int Hq, int kv_heads, int D, int max_new, int max_context,
             int window, int sinks, PaPlan& p) {
  const int G = Hq / kv_heads;
  long long span = max_context;
  if (window > 0) span = std::min<long long>(span, static_cast<long long>(window) + max_new + sinks);
  p = {};
  p.prompt = static_cast<long long>(G) * max_new > PA_MAX_DECODE_ROWS;
  // at least one short sequence fits beside sequences of max_new tokens only if the total leaves room for it
  p.decode = !p.prompt ||
             (batch > 1 && total <= static_cast<long long>(batch - 1) * max_new + PA_MAX_DECODE_ROWS / G);
  if (p.decode) {
    const int rows = p.prompt ? PA_MAX_DECODE_ROWS : G * max_new;
    p.block = rows <= 8 ? 8 : 16;
    p.row_blocks = (rows + p.block - 1) / p.block;
    const long long pairs = static_cast<long long>(batch) * kv_heads * p.row_blocks;
    if (pairs * p.block > 0x7fffffff) return false;
    // as many CTAs as fit the GPU at once, fewer when the longest sequence expected leaves them without PA_MIN_TILES tiles each
    const long long tiles = ((span + PA_TILE - 1) / PA_TILE + 2) * pairs;
    const long long most = static_cast<long long>(di.sm_count) * (p.block == 8 ? 3 : 2);
    p.ctas = static_cast<int>(std::max<long long>(1, std::min(most, (tiles + PA_MIN_TILES - 1) / PA_MIN_TILES)));
    if (p.ctas > 1) p.decode_bytes = (static_cast<size_t>(p.ctas) * 2 * p.block * (D + 2) * sizeof(float) + 255) / 256 * 256;
    if (p.ctas > 1 && batch > PA_THREADS) {
      p.begins_at = p.decode_bytes;
      p.decode_bytes += ((static_cast<size_t>(batch) + 1) * sizeof(long long) + 255) / 256 * 256;
    }
  }
  p.bytes = p.decode_bytes;
  if (p.prompt) {
    const long long tiles = static_cast<long long>(total) * G / PT_ROWS + batch;
    if (tiles * kv_heads > 0x7fffffff) return false;
    p.tiles = static_cast<int>(tiles);
    // the rows' spans are split where whole ones would leave SMs idle
    const long long fit = di.sm_count / std::max<long long>(1, tiles * kv_heads);
    p.splits = static_cast<int>(std::max<long long>(1, std::min<long long>({fit, span / (2 * PT_KEYS), PT_MAX_SPLITS})));
    if (p.splits > 1) p.bytes += static_cast<size_t>(total) * Hq * p.splits * (D + 2) * sizeof(float);
  }
  return true;
}

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
mui_status_t launch_prompt(cudaStream_t stream, const PaArgs& a, int tiles, int pdl, int device) {
  constexpr size_t smem = 2 * PT_GROUP * D * 2 + PT_SLOTS * PT_KEYS * D * 2 + 1024;
  static std::atomic<unsigned long long> configured{0};  // one bit per device
  const unsigned long long bit = 1ull << (device & 63);
  if (!(configured.load() & bit)) {
    MUI_CUDA_CHECK(cudaFuncSetAttribute(paged_prompt_kernel<T, KV8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(smem)));
    configured.fetch_or(bit);
  }
  CUtensorMap maps[2] = {};
  if (!KV8) {
    // the pool as rows of head_dim elements; boxes of 16 rows x 64 elements, which never cross a page
    EncodeTiledFn enc = encode_tiled_fn();
    MUI_REQUIRE(enc != nullptr, MUI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const long long rows = (static_cast<long long>(a.kv.num_pages) * a.kv.kv_heads) << a.kv.page_shift;
    MUI_REQUIRE(rows <= 0x7fffffff, MUI_ERR_UNSUPPORTED, "%lld cache rows in a pool (at most 2^31 - 1)", rows);
    const cuuint64_t dims[2] = {D, static_cast<cuuint64_t>(rows)}, stride[1] = {D * 2};
    const cuuint32_t box[2] = {64, PA_TILE}, step[2] = {1, 1};
    for (int i = 0; i < 2; ++i) {
      const CUresult r = enc(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, i == 0 ? a.kv.k_pages : a.kv.v_pages, dims, stride, box,
                             step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
      MUI_REQUIRE(r == CUDA_SUCCESS, MUI_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", static_cast<int>(r));
    }
  }
  MUI_CUDA_CHECK(mui_launch(paged_prompt_kernel<T, KV8, D>, dim3(tiles * a.kv.kv_heads, a.splits), dim3(PT_THREADS), smem,
                            stream, pdl, maps[0], maps[1], a));
  if (a.splits > 1) {
    const long long rows = static_cast<long long>(a.kv.total) * a.Hq;
    MUI_CUDA_CHECK(mui_launch(paged_prompt_merge_kernel<T, D>, dim3(static_cast<unsigned>((rows + PA_WARPS - 1) / PA_WARPS)),
                              dim3(PA_THREADS), 0, stream, 1, a));
  }
  return MUI_OK;
}

template <typename T, bool KV8, int D>
mui_status_t launch_attention(cudaStream_t stream, PaArgs a, const PaPlan& p, void* workspace, int pdl, int device) {
  if (p.decode) {
    a.partials = reinterpret_cast<float*>(workspace);
    if (p.begins_at) a.begins = reinterpret_cast<long long*>(reinterpret_cast<char*>(workspace) + p.begins_at);
    const mui_status_t s = p.block == 8 ? launch_decode<T, KV8, D, 1>(stream, a, pdl, device)
                                        : launch_decode<T, KV8, D, 2>(stream, a, pdl, device);
    if (s != MUI_OK) return s;
    pdl = 0;
  }
  if (!p.prompt) return MUI_OK;
  a.partials = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + p.decode_bytes);
  return launch_prompt<T, KV8, D>(stream, a, p.tiles, pdl, device);
}

}  // namespace

extern "C" {

size_t mui_paged_attention_workspace_bytes(int total_tokens, int batch, int num_q_heads, int kv_heads, int head_dim,
                                           int max_new_tokens, int max_context, int window, int sinks) {
  if (total_tokens <= 0 || batch <= 0 || num_q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_new_tokens <= 0 ||
      max_context <= 0)
    return 0;
  const MuiDeviceInfo* di = mui_current_device_info();
  if (num_q_heads < kv_heads || !di) return 0;
  auto bytes = [&](int max_new) {
    PaPlan p;
    return pa_plan(*di, total_tokens, batch, num_q_heads, kv_heads, head_dim, max_new, max_context, window, sinks, p) ? p.bytes
                                                                                                                       : 0;
  };
  // as many tokens as sequences may stand for a call without cu_tokens, which counts max_new_tokens as 1
  return std::max(bytes(max_new_tokens), total_tokens == batch ? bytes(1) : 0);
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
  if (cache->cu_tokens == nullptr) max_new_tokens = 1;  // a looser bound would launch the prompt kernel, which reads cu_tokens
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
  // a negative scale is taken as a positive one of -q
  a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  a.scale_log2 = (scale < 0.f ? -scale : scale) * 1.44269504088896341f;
  // a tile is 16 rows of K and of V
  a.lead = PA_TRIPLE_COST * 4096 / (2 * PA_TILE * cache->head_dim * (cache->format == MUI_KV_E4M3 ? 1 : 2));
  PaPlan p;
  MUI_REQUIRE(pa_plan(*di, cache->total_tokens, cache->batch, num_q_heads, cache->kv_heads, cache->head_dim, max_new_tokens,
                      max_context, window, sinks, p),
              MUI_ERR_UNSUPPORTED, "batch=%d, total_tokens=%d and kv_heads=%d are too large", cache->batch,
              cache->total_tokens, cache->kv_heads);
  MUI_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes &&
                               (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
              MUI_ERR_INVALID_ARG, "workspace of %zu bytes (16-byte aligned) needed, %zu given", p.bytes,
              workspace ? workspace_bytes : static_cast<size_t>(0));
  a.row_blocks = p.row_blocks;
  a.ctas = p.ctas;
  a.splits = p.splits;
  a.mixed = p.decode && p.prompt;
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define PA_GO(T, D)                                                            \
  (cache->format == MUI_KV_E4M3 ? launch_attention<T, true, D>(st, a, p, workspace, pdl, di->device) \
                                : launch_attention<T, false, D>(st, a, p, workspace, pdl, di->device))
  if (dtype == MUI_F16) return cache->head_dim == 128 ? PA_GO(__half, 128) : PA_GO(__half, 64);
  return cache->head_dim == 128 ? PA_GO(__nv_bfloat16, 128) : PA_GO(__nv_bfloat16, 64);
#undef PA_GO
}

}  // extern "C"
