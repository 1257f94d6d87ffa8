// Drawing a token from each row of logits: temperature, top-k, top-p, min-p, inverse transform of a given uniform number.
//
// With z = (logit - largest) / temperature and w = exp(z), the kept tokens are a run from the front of the ranking by
// (logit descending, index ascending), so two numbers describe them: kept is key > T, or key == T and index <= T_idx. No
// sort is needed, only that threshold.
//
// Sums of weights decide which token is drawn, so they must not depend on the order in which threads add: w is taken in
// fp64 and rounded once to an integer with S fraction bits (S = min(50, 62 - ceil(log2 vocab)); 44 for 200 k tokens; no sum
// overflows), and integers are summed. A weight that rounds to 0 can never be drawn. Against real arithmetic a boundary is
// off by sqrt(vocab) * 2^-S of the largest weight or so, 3e-11 for 200 k tokens.
//
// A cluster of up to eight CTAs works on a row (one CTA when there are rows enough to fill the GPU). Passes over the row:
//   1. the largest logit (from HBM; the later passes find the row in L2);
//   2. a histogram of z in 4096 equal bins down to the smallest z that still has weight. Counts give the bin that holds
//      the top_k-th token exactly; counts times the bin centre's weight tell the bin in which top_p ends, nearly always;
//   3. exact sums of the weight above and between these two bins; the bins' own tokens (some hundred) are collected in rank
//      0's shared memory, sorted, and give T and T_idx; where the estimate was off, again with the neighbouring bin;
//   4. the kept weight of every run of 256 tokens; the run that holds the drawn point is then walked by one warp.
// Without top-k and top-p only 1 and 4 run. Where a bin has more tokens than the list holds (long ties, very high
// temperatures) T and T_idx are found by bisection over keys and indices instead: slower, same result.
//
// Bound: rows * vocab * size bytes for large batches, then 13 fp64 operations a weight; for few rows the chain of passes and
// cluster barriers.
#include "common.cuh"

#include <atomic>
#include <cmath>
#include <type_traits>

MUI_STATUS_ACCESSOR(sample)

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_CHUNK = 256;    // tokens of one warp step: eight consecutive ones per lane
constexpr int SM_BINS = 4096;
constexpr int SM_LIST = 4096;    // tokens collected per boundary bin
constexpr int SM_RUNS = 1024;    // runs of chunks whose kept weight a CTA holds
constexpr int SM_MAX_CLUSTER = 8;
// what rank 0 finds in the collected bins: the threshold, that top-p ends further up or down the ranking, or too many tokens
enum : uint32_t { SM_FOUND, SM_UP, SM_DOWN, SM_BISECT };

struct SampleArgs {
  const void* logits;
  long long stride;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t* top_k;
  int64_t* tokens;
  float* logprobs;
  int V, frac_bits, cluster, chunks_per_run;
};

// order-preserving key of a logit: larger logit, larger key; -0 equals +0; NaN is below everything (key 0)
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// ---- cluster helpers (also right for a cluster of one) ----
__device__ __forceinline__ unsigned cta_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* local, unsigned rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* local, unsigned rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer_u64(const u64* local, unsigned rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(local, rank)) : "memory");
  return v;
}

struct Shared {
  uint32_t bins[SM_BINS];    // this CTA's counts
  u64 list[2][SM_LIST];      // rank 0: key << 32 | ~index of the tokens in the two boundary bins: larger ranks first
  u64 list_w[SM_LIST];
  u64 runs[SM_RUNS];
  u64 part[SM_WARPS][3];
  u64 sums[2][3];            // this CTA's sums, two turns so that one barrier per exchange is enough
  u64 fwarp[SM_WARPS];
  double mwarp[SM_WARPS];
  uint32_t list_n[2];
  uint32_t verdict;          // rank 0: threshold found
  uint32_t T, T_idx;
  int bin_k, bin_p;
  uint32_t before_k;
  double est_total;
  int hit;
};

// The eight tokens from i on as fp32; NaN behind the end of the row.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int i, int V, bool vec, float (&x)[8]) {
  if (vec && i + 8 <= V) {
    if (sizeof(T) == 4) {
      const uint4 a = ld_act16(reinterpret_cast<const char*>(row) + static_cast<size_t>(i) * 4);
      const uint4 b = ld_act16(reinterpret_cast<const char*>(row) + static_cast<size_t>(i) * 4 + 16);
      x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
      x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
    } else {
      using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
      unpack8<H>(ld_act16(row + i), x);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = __int_as_float(0x7fffffff);
    if (i + e < V) {
      if (sizeof(T) == 4) x[e] = __ldcg(reinterpret_cast<const float*>(row) + i + e);
      else {
        using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
        x[e] = ld_act_f32<H>(reinterpret_cast<const H*>(row) + i + e);
      }
    }
  }
}

// Weights of one row. table: lane j of every warp holds 2^(j / 32).
struct Weigh {
  float top, bin_scale;
  double inv_t, table;
  int frac_bits;
  // bin of z; SM_BINS and above: the weight rounds to 0. Non-decreasing in the distance from the largest logit.
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    const float b = (top - x) * bin_scale;
    return b < static_cast<float>(SM_BINS) ? static_cast<int>(b) : SM_BINS;  // NaN: SM_BINS
  }
  // 2^S exp(z), rounded; whole warp, x of lanes with use == false is not looked at. z = (32 n + j) ln2 / 32 + r with |r| <=
  // ln2 / 64: exp(z) = 2^n * 2^(j/32) * exp(r), the last one by its Taylor polynomial of degree 5 (r^6 / 720 < 3e-15).
  __device__ __forceinline__ u64 operator()(float x, bool use) const {
    const double z = use && x != top ? (static_cast<double>(x) - static_cast<double>(top)) * inv_t : 0.0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number, in the low bits
    const double km = fma(z, 46.166241308446828, magic);  // 32 / ln 2
    const int k = __double2loint(km);
    const double r = fma(km - magic, -0.021660849392498290, z);  // ln 2 / 32
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    p *= __shfl_sync(MUI_FULL_MASK, table, k & 31);
    p = __hiloint2double(__double2hiint(p) + (((k >> 5) + frac_bits) << 20), __double2loint(p));
    // p < 2^51: adding 2^52 leaves the rounded integer in the mantissa
    const u64 bits = static_cast<u64>(__double_as_longlong(p + 4503599627370496.0)) & 0xfffffffffffffull;
    return use ? bits : 0ull;
  }
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(MUI_FULL_MASK, v, o);
  return v;
}

template <typename T>
struct Row {
  const T* p;
  int V, c0, c1;  // this CTA's chunks
  bool vec;
  // f(first token of the lane, its eight logits) for every chunk of this CTA; warps take chunks in turn
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int c = c0 + warp;
    for (; c + SM_WARPS < c1; c += 2 * SM_WARPS) {  // two chunks of loads in flight
      float x[8], y[8];
      load8<T>(p, c * SM_CHUNK + lane * 8, V, vec, x);
      load8<T>(p, (c + SM_WARPS) * SM_CHUNK + lane * 8, V, vec, y);
      f(c * SM_CHUNK + lane * 8, x);
      f((c + SM_WARPS) * SM_CHUNK + lane * 8, y);
    }
    if (c < c1) {
      float x[8];
      load8<T>(p, c * SM_CHUNK + lane * 8, V, vec, x);
      f(c * SM_CHUNK + lane * 8, x);
    }
  }
};

// Sums of three numbers over the cluster; every thread gets them. `turn` alternates from call to call.
__device__ __forceinline__ void cluster_sum3(Shared& s, int cluster, int& turn, u64 (&v)[3]) {
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 3; ++i) v[i] = warp_sum_u64(v[i]);
  if ((threadIdx.x & 31) == 0)
    for (int i = 0; i < 3; ++i) s.part[warp][i] = v[i];
  __syncthreads();
  if (threadIdx.x < 3) {
    u64 t = 0;
    for (int w = 0; w < SM_WARPS; ++w) t += s.part[w][threadIdx.x];
    s.sums[turn][threadIdx.x] = t;
  }
  if (cluster > 1) cluster_sync();
  else __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = 0;
    for (int r = 0; r < cluster; ++r) v[i] += cluster > 1 ? peer_u64(&s.sums[turn][i], r) : s.sums[turn][i];
  }
  turn ^= 1;
}

// The boundary of top-k and top-p by bisection: 32 steps over keys for each, then over indices for the ties.
template <typename T>
__device__ void threshold_by_bisection(Shared& s, const SampleArgs& a, const Row<T>& row, const Weigh& w, int& turn,
                                       uint32_t best, bool use_k, uint32_t k, bool use_p, double top_p, uint32_t& T_key,
                                       uint32_t& T_idx) {
  // count and weight of the tokens with key >= pivot
  auto from = [&](uint32_t pivot, u64& count, u64& mass) {
    u64 v[3] = {0, 0, 0};
    row.each([&](int i, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = i + e < a.V && logit_key(x[e]) >= pivot;
        v[0] += in;
        v[1] += w(x[e], in && w.bin(x[e]) < SM_BINS);
      }
    });
    cluster_sum3(s, a.cluster, turn, v);
    count = v[0];
    mass = v[1];
  };
  auto weight_of = [&](uint32_t key) {
    const float x = key_logit(key);
    return w(x, x == x && w.bin(x) < SM_BINS);
  };
  u64 ties = ~0ull, total = 0, n, m;
  T_key = 0;
  if (use_k) {
    uint32_t lo = 0, hi = best;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      from(mid, n, m);
      if (n >= k) lo = mid;
      else hi = mid - 1;
    }
    T_key = lo;
    from(lo + 1, n, m);  // lo <= best < 2^32 - 1 (a NaN has key 0)
    ties = k - n;
    total = m + ties * weight_of(lo);
  } else if (use_p) {
    from(0, n, total);
  }
  if (use_p) {
    const double target = top_p * static_cast<double>(total);
    uint32_t lo = T_key, hi = best;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      from(mid, n, m);
      if (static_cast<double>(m) >= target) lo = mid;
      else hi = mid - 1;
    }
    from(lo + 1, n, m);
    const double each = static_cast<double>(weight_of(lo));
    u64 need = 1;
    if (each > 0.0) {
      const double q = ceil((target - static_cast<double>(m)) / each);
      need = q < 1.0 ? 1ull : (q > 4.0e9 ? ~0ull : static_cast<u64>(q));
    }
    ties = lo > T_key || need < ties ? need : ties;
    T_key = lo;
  }
  // index of the last tie that is kept
  uint32_t lo = 0, hi = a.V - 1;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    u64 v[3] = {0, 0, 0};
    row.each([&](int i, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[0] += i + e < a.V && i + e <= static_cast<int>(mid) && logit_key(x[e]) == T_key;
    });
    cluster_sum3(s, a.cluster, turn, v);
    if (v[0] >= ties) hi = mid;
    else lo = mid + 1;
  }
  T_idx = lo;
}

// Sorts a collected bin into ranking order and leaves in list_w[i] the weight of its tokens before the i-th; returns the
// weight of all of them. One CTA. A bitonic sort: 8192 exchanges of the largest list are 2 per thread and step.
__device__ u64 rank_bin(Shared& s, u64* list, int n, const Weigh& w) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int m = 2;
  while (m < n) m <<= 1;
  for (int i = n + tid; i < m; i += SM_THREADS) list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= m; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int p = tid; p < m / 2; p += SM_THREADS) {
        const int i = 2 * p - (p & (j - 1)), o = i + j;
        const u64 x = list[i], y = list[o];
        if ((x < y) == ((i & k) == 0)) {
          list[i] = y;
          list[o] = x;
        }
      }
      __syncthreads();
    }
  constexpr int PER = SM_LIST / SM_THREADS;
  u64 q[PER], sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = tid * PER + e;
    q[e] = w(i < n ? key_logit(static_cast<uint32_t>(list[i] >> 32)) : 0.f, i < n);
    sum += q[e];
  }
  u64 run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(MUI_FULL_MASK, run, o);
    if (lane >= o) run += y;
  }
  if (lane == 31) s.fwarp[warp] = run;
  __syncthreads();
  u64 all = 0;
  run -= sum;
  for (int i = 0; i < SM_WARPS; ++i) {
    if (i < warp) run += s.fwarp[i];
    all += s.fwarp[i];
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    s.list_w[tid * PER + e] = run;
    run += q[e];
  }
  __syncthreads();
  return all;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  Shared& s = *reinterpret_cast<Shared*>(sample_smem);
  const int C = a.cluster, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned rank = C > 1 ? cta_rank() : 0;
  const int r = blockIdx.x / C;
  int turn = 0;
  pdl_wait_prior_grid();
  pdl_launch_dependents();

  Row<T> row;
  row.p = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  row.V = a.V;
  row.vec = (reinterpret_cast<uintptr_t>(row.p) & 15) == 0;
  const int chunks = (a.V + SM_CHUNK - 1) / SM_CHUNK, per_cta = (chunks + C - 1) / C;
  row.c0 = min(chunks, static_cast<int>(rank) * per_cta);
  row.c1 = min(chunks, row.c0 + per_cta);
  const float t = a.temperature ? __ldcg(a.temperature + r) : 1.f;
  const int k_raw = a.top_k ? __ldcg(a.top_k + r) : 0;
  const float top_p = a.top_p ? __ldcg(a.top_p + r) : 1.f;
  const float min_p = a.min_p ? __ldcg(a.min_p + r) : 0.f;
  const bool use_k = k_raw > 0 && k_raw < a.V, use_p = top_p < 1.f, greedy = !(t > 0.f);

  // 1. the largest logit; its lowest index where that is the answer
  u64 best = 0;  // key << 32 | ~index
  if (greedy) {
    row.each([&](int i, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 v = static_cast<u64>(logit_key(x[e])) << 32 | ~static_cast<uint32_t>(i + e);
        best = i + e < a.V && v > best ? v : best;
      }
    });
  } else {
    float m = -INFINITY;
    row.each([&](int, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
    });
    best = static_cast<u64>(logit_key(m)) << 32 | 0xffffffffu;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(MUI_FULL_MASK, best, o);
    best = y > best ? y : best;
  }
  if (lane == 0) s.fwarp[warp] = best;
  for (int i = tid; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0;
  if (tid < 2) s.list_n[tid] = 0;
  __syncthreads();
  for (int i = 0; i < SM_WARPS; ++i) best = s.fwarp[i] > best ? s.fwarp[i] : best;
  if (C > 1) {
    if (tid == 0) s.sums[1][0] = best;
    cluster_sync();
    for (int i = 0; i < C; ++i) {
      const u64 y = peer_u64(&s.sums[1][0], i);
      best = y > best ? y : best;
    }
  }
  const uint32_t best_key = static_cast<uint32_t>(best >> 32);
  Weigh w;
  w.top = key_logit(best_key);
  const bool nothing = !(w.top > -INFINITY);  // key 0 (all NaN) reads as NaN
  if (greedy || nothing) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = nothing ? 0 : static_cast<int64_t>(~static_cast<uint32_t>(best));
      if (a.logprobs) a.logprobs[r] = nothing ? -INFINITY : 0.f;
    }
    if (C > 1) cluster_sync();  // peers may still be reading this CTA's memory
    return;
  }
  w.frac_bits = a.frac_bits;
  w.inv_t = 1.0 / static_cast<double>(t);
  w.table = exp2(static_cast<double>(lane) / 32.0);
  // z below -(S + 2) ln 2 has a weight under a quarter of the last bit
  const float z_range = (a.frac_bits + 2) * 0.693147181f;
  w.bin_scale = static_cast<float>(SM_BINS) / z_range / t;
  const u64 one = 1ull << a.frac_bits;
  // min-p in the integers of the weights; the largest token has weight 1 and always stays
  const u64 w_min = min_p > 0.f ? static_cast<u64>(ceil(fmin(static_cast<double>(min_p), 1.0) * static_cast<double>(one))) : 1ull;

  uint32_t T_key = 0, T_idx = 0;  // nothing to cut: every key that has weight is above 0
  if (use_k || use_p) {
    // 2. histogram
    row.each([&](int, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int b = w.bin(x[e]);
        if (b < SM_BINS) atomicAdd(&s.bins[b], 1u);
      }
    });
    if (tid == 0) {
      s.bin_k = s.bin_p = SM_BINS;
      s.before_k = 0;
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    // prefix sums over the cluster's bins, four per thread: counts, and weights of the bin centres
    constexpr int PER = SM_BINS / SM_THREADS;
    uint32_t n[PER], nc = 0;
    double m[PER], mc = 0.0;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
      n[h] = 0;
      for (int i = 0; i < C; ++i) n[h] += C > 1 ? peer_u32(&s.bins[PER * tid + h], i) : s.bins[PER * tid + h];
      m[h] = n[h] * static_cast<double>(exp2f(-(PER * tid + h + 0.5f) * (z_range * 1.44269504f / SM_BINS)));
      nc += n[h];
      mc += m[h];
    }
    uint32_t nb = nc;
    double mb = mc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(MUI_FULL_MASK, nb, o);
      const double q = __shfl_up_sync(MUI_FULL_MASK, mb, o);
      if (lane >= o) {
        nb += y;
        mb += q;
      }
    }
    if (lane == 31) {
      s.fwarp[warp] = nb;
      s.mwarp[warp] = mb;
    }
    __syncthreads();
    double all = 0.0;
    nb -= nc;
    mb -= mc;
    for (int i = 0; i < SM_WARPS; ++i) {
      if (i < warp) {
        nb += static_cast<uint32_t>(s.fwarp[i]);
        mb += s.mwarp[i];
      }
      all += s.mwarp[i];
    }
    const uint32_t k = static_cast<uint32_t>(k_raw);
    if (use_k) {
      if (tid == 0) s.est_total = all;
      __syncthreads();
      uint32_t at = nb;
      double am = mb;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        if (at < k && at + n[h] >= k) {  // one thread at most
          s.bin_k = PER * tid + h;
          s.before_k = at;
          s.est_total = am + m[h] * (k - at) / n[h];
        }
        at += n[h];
        am += m[h];
      }
      __syncthreads();
      all = s.est_total;
    }
    if (use_p) {
      const double target = static_cast<double>(top_p) * all;
      uint32_t at = nb;
      double am = mb;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        // the first occupied bin with which the sum reaches the target
        if (n[h] > 0 && am + m[h] >= target && (am < target || at == 0)) atomicMin(&s.bin_p, PER * tid + h);
        at += n[h];
        am += m[h];
      }
      __syncthreads();
    }
    const int bin_k = s.bin_k;
    int bin_p = use_p ? min(s.bin_p, bin_k) : bin_k;
    uint32_t verdict = use_p || bin_k < SM_BINS ? SM_BISECT : SM_FOUND;  // a top_p next to 1 may end in no bin
    for (int attempt = 0; attempt < 4 && bin_p < SM_BINS; ++attempt) {
      // 3. exact sums: [0] above bin_p, [1] between the bins; tokens of the bins go to rank 0
      u64 v[3] = {0, 0, 0};
      const uint32_t count_at[2] = {peer_addr(&s.list_n[0], 0), peer_addr(&s.list_n[1], 0)};
      const uint32_t list_at[2] = {peer_addr(&s.list[0][0], 0), peer_addr(&s.list[1][0], 0)};
      row.each([&](int i, float(&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int b = w.bin(x[e]);
          const bool sum = use_p && b < bin_k && b != bin_p && b < SM_BINS;
          if (__any_sync(MUI_FULL_MASK, sum)) {
            const u64 q = w(x[e], sum);
            v[0] += b < bin_p ? q : 0ull;
            v[1] += b < bin_p ? 0ull : q;
          }
          if (b < SM_BINS && (b == bin_p || b == bin_k)) {
            const int which = b == bin_p ? 0 : 1;
            uint32_t at;
            asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count_at[which]) : "memory");
            if (at < SM_LIST) {
              const u64 entry = static_cast<u64>(logit_key(x[e])) << 32 | ~static_cast<uint32_t>(i + e);
              asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list_at[which] + at * 8), "l"(entry) : "memory");
            }
          }
        }
      });
      cluster_sum3(s, C, turn, v);  // its barrier also publishes the lists
      if (rank == 0) {
        const int n0 = s.list_n[0], n1 = s.list_n[1];
        const bool same = bin_p == bin_k;
        uint32_t say = SM_BISECT;
        if (n0 <= SM_LIST && n1 <= SM_LIST) {
          const uint32_t left = k - s.before_k;  // tokens of bin_k within the top-k
          u64 in_k = 0;
          u64 last = 0;
          if (!same && bin_k < SM_BINS) {
            const u64 bin_mass = rank_bin(s, s.list[1], n1, w);
            in_k = left < static_cast<uint32_t>(n1) ? s.list_w[left] : bin_mass;
            __syncthreads();
          }
          const int n_p = same ? static_cast<int>(min(left, static_cast<uint32_t>(n0))) : n0;  // of bin_p within the top-k
          u64 in_p = rank_bin(s, s.list[0], n0, w);
          if (n_p < n0) in_p = s.list_w[n_p];
          if (!use_p) {
            last = s.list[0][n_p - 1];
            say = SM_FOUND;
          } else {
            const double target = static_cast<double>(top_p) * static_cast<double>(v[0] + v[1] + in_p + in_k);
            // the estimate of step 2 may be a bin off
            if (v[0] != 0 && static_cast<double>(v[0]) >= target) say = SM_UP;
            else if (static_cast<double>(v[0] + in_p) < target) say = SM_DOWN;
            else {
              // tokens whose predecessors do not reach the target are kept, the first of all in any case
              int lo = 1, hi = n_p;
              while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (static_cast<double>(v[0] + s.list_w[mid - 1]) < target) lo = mid;
                else hi = mid - 1;
              }
              last = s.list[0][lo - 1];
              say = SM_FOUND;
            }
          }
          if (tid == 0) {
            s.T = static_cast<uint32_t>(last >> 32);
            s.T_idx = ~static_cast<uint32_t>(last);
          }
        }
        __syncthreads();
        if (tid == 0) s.verdict = say;
        if (tid < 2) s.list_n[tid] = 0;
      }
      if (C > 1) cluster_sync();
      else __syncthreads();
      verdict = C > 1 ? peer_u32(&s.verdict, 0) : s.verdict;
      if (verdict != SM_UP && verdict != SM_DOWN) break;
      // the neighbour that holds tokens (every CTA finds the same one)
      const int was = bin_p;
      if (tid == 0) s.bin_p = verdict == SM_UP ? -1 : SM_BINS;
      __syncthreads();
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        const int bin = PER * tid + h;
        if (n[h] > 0 && verdict == SM_UP && bin < was) atomicMax(&s.bin_p, bin);
        if (n[h] > 0 && verdict == SM_DOWN && bin > was) atomicMin(&s.bin_p, bin);
      }
      __syncthreads();
      bin_p = s.bin_p;
      verdict = SM_BISECT;
      if (bin_p < 0 || bin_p > bin_k) break;
      if (C > 1) cluster_sync();  // rank 0's list is empty before anyone adds to it; verdicts have been read
    }
    if (verdict == SM_FOUND) {
      if (bin_p < SM_BINS) {
        T_key = C > 1 ? peer_u32(&s.T, 0) : s.T;
        T_idx = C > 1 ? peer_u32(&s.T_idx, 0) : s.T_idx;
      }
    } else {
      threshold_by_bisection<T>(s, a, row, w, turn, best_key, use_k, k, use_p, static_cast<double>(top_p), T_key, T_idx);
    }
  }

  // 4. kept weight by runs of chunks
  __syncthreads();
  for (int i = tid; i < SM_RUNS; i += SM_THREADS) s.runs[i] = 0;
  __syncthreads();
  const float T_logit = T_key ? key_logit(T_key) : -INFINITY;
  auto kept_weight = [&](float x, int i) {
    const bool in = w.bin(x) < SM_BINS && (x > T_logit || (x == T_logit && i <= static_cast<int>(T_idx)));
    u64 q = 0;
    if (__any_sync(MUI_FULL_MASK, in)) q = w(x, in);
    return q >= w_min ? q : 0ull;
  };
  u64 v[3] = {0, 0, 0};
  row.each([&](int i, float(&x)[8]) {
    u64 q = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) q += kept_weight(x[e], i + e);
    if (__any_sync(MUI_FULL_MASK, q != 0)) {
      v[0] += q;
      q = warp_sum_u64(q);
      if (lane == 0) atomicAdd(&s.runs[(i / SM_CHUNK - row.c0) / a.chunks_per_run], q);
    }
  });
  const int my_turn = turn;
  cluster_sum3(s, C, turn, v);
  const u64 total = v[0];
  u64 before = 0, mine = 0;
  for (int i = 0; i < C; ++i) {
    const u64 y = C > 1 ? peer_u64(&s.sums[my_turn][0], i) : s.sums[my_turn][0];
    if (i < static_cast<int>(rank)) before += y;
    if (i == static_cast<int>(rank)) mine = y;
  }
  // uniform numbers lie in [0, 1); what does not is brought to the nearest fp32 that does
  const float u = fminf(fmaxf(__ldcg(a.uniforms + r), 0.f), 0.99999994f);
  const double want = static_cast<double>(u) * static_cast<double>(total);
  if (C > 1) cluster_sync();  // the last look at a peer's memory
  if (mine == 0 || static_cast<double>(before) > want || static_cast<double>(before + mine) <= want) return;

  // this CTA holds the drawn point: first its run, then its chunk and token
  {
    u64 q = tid < SM_RUNS ? s.runs[tid] : 0;
    u64 c = q;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(MUI_FULL_MASK, c, o);
      if (lane >= o) c += y;
    }
    if (lane == 31) s.fwarp[warp] = c;
    __syncthreads();
    u64 at = before;
    for (int i = 0; i < warp; ++i) at += s.fwarp[i];
    if (q != 0 && static_cast<double>(at + c) > want && static_cast<double>(at + c - q) <= want) {
      s.hit = tid;
      s.sums[my_turn ^ 1][0] = at + c - q;  // weight in front of the run
    }
    __syncthreads();
  }
  if (warp != 0) return;
  u64 at = s.sums[my_turn ^ 1][0];
  const int first = row.c0 + s.hit * a.chunks_per_run, last = min(row.c1, first + a.chunks_per_run);
  for (int c = first; c < last; ++c) {
    float x[8];
    u64 q[8], sum = 0;
    const int i = c * SM_CHUNK + lane * 8;
    load8<T>(row.p, i, a.V, row.vec, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = kept_weight(x[e], i + e);
      sum += q[e];
    }
    u64 run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(MUI_FULL_MASK, run, o);
      if (lane >= o) run += y;
    }
    const unsigned hit = __ballot_sync(MUI_FULL_MASK, sum != 0 && static_cast<double>(at + run) > want);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        u64 p = at + run - sum;
        int e = 0;
#pragma unroll
        for (int h = 7; h >= 0; --h) {  // the first token at which the running weight exceeds the point
          u64 upto = p;
          for (int j = 0; j <= h; ++j) upto += q[j];
          if (q[h] != 0 && static_cast<double>(upto) > want) e = h;
        }
        a.tokens[r] = i + e;
        u64 mine_w = 0;
#pragma unroll
        for (int h = 0; h < 8; ++h) mine_w = h == e ? q[h] : mine_w;
        if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(mine_w) / static_cast<double>(total)));
      }
      return;
    }
    at += __shfl_sync(MUI_FULL_MASK, run, 31);
  }
}

template <typename T>
mui_status_t launch_sample(cudaStream_t stream, const SampleArgs& a, int rows, int pdl, int device) {
  static std::atomic<u64> configured{0};  // one bit per device
  const u64 bit = 1ull << (device & 63);
  if (!(configured.load() & bit)) {
    MUI_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(sizeof(Shared))));
    configured.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * a.cluster);
  cfg.blockDim = dim3(SM_THREADS);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  MUI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a));
  return MUI_OK;
}

}  // namespace

extern "C" mui_status_t mui_sample_tokens(void* stream, int dtype, int rows, int vocab, const void* logits,
                                          int64_t row_stride, const float* temperature, const int32_t* top_k,
                                          const float* top_p, const float* min_p, const float* uniforms,
                                          int64_t* tokens, float* logprobs, unsigned flags) {
  MUI_REQUIRE(dtype == MUI_F16 || dtype == MUI_BF16 || dtype == MUI_COMM_F32, MUI_ERR_UNSUPPORTED,
              "dtype %d unsupported", dtype);
  MUI_REQUIRE(rows >= 0 && rows <= (1 << 24) && vocab >= 1 && vocab <= (1 << 24) && row_stride >= 0,
              MUI_ERR_INVALID_ARG, "bad sizes rows=%d (0..2^24) vocab=%d (1..2^24) row_stride=%lld", rows, vocab,
              (long long)row_stride);
  if (rows == 0) return MUI_OK;
  MUI_REQUIRE(logits && uniforms && tokens, MUI_ERR_INVALID_ARG, "logits, uniforms and tokens must be non-null");
  const MuiDeviceInfo* di = mui_current_device_info();
  if (!di) return MUI_ERR_CUDA;
  SampleArgs a;
  a.logits = logits;
  a.stride = row_stride;
  a.temperature = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniforms = uniforms;
  a.top_k = top_k;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.V = vocab;
  int lg = 0;
  while ((1 << lg) < vocab) ++lg;
  a.frac_bits = 62 - lg < 50 ? 62 - lg : 50;
  // CTAs per row: as many as the rows leave SMs for, each with two steps of all its warps at least
  a.cluster = 1;
  while (a.cluster < SM_MAX_CLUSTER && rows * static_cast<long long>(a.cluster) * 2 <= di->sm_count &&
         vocab > a.cluster * SM_CHUNK * SM_WARPS)
    a.cluster *= 2;
  const int chunks = (vocab + SM_CHUNK - 1) / SM_CHUNK, per_cta = (chunks + a.cluster - 1) / a.cluster;
  a.chunks_per_run = (per_cta + SM_RUNS - 1) / SM_RUNS;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  if (dtype == MUI_F16) return launch_sample<__half>(st, a, rows, pdl, di->device);
  if (dtype == MUI_BF16) return launch_sample<__nv_bfloat16>(st, a, rows, pdl, di->device);
  return launch_sample<float>(st, a, rows, pdl, di->device);
}
