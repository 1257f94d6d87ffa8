// Drawing a token from each row of logits: temperature, top-k, top-p, min-p, inverse transform of a given uniform number.
//
// With z = (logit - largest) / temperature and w = exp(z), the kept tokens are a run from the front of the ranking by
// (logit descending, index ascending), so two numbers describe them: kept is key > T, or key == T and index <= T_idx.
//
// Sums of weights decide which token is drawn, so they must not depend on the order in which threads add: w is taken in
// fp64 and rounded once to an integer with S fraction bits (S = min(48, 62 - ceil(log2 vocab)); 44 for 200 k tokens; no sum
// overflows), and integers are summed. A weight that rounds to 0 can never be drawn. Against real arithmetic a boundary is
// off by sqrt(vocab) * 2^-S of the largest weight or so, 3e-11 for 200 k tokens.
//
// A cluster of up to eight CTAs works on a row (one CTA when there are rows enough to fill the GPU). Passes over the row:
//   1. the largest logit (from HBM; the later passes find the row in L2);
//   2. with top-k or top-p, a histogram of z in 2048 equal bins down to the smallest z that still has weight. Counts give the
//      bin that holds the top_k-th token exactly; counts times the bin centre's weight tell the bin in which top_p ends,
//      nearly always. Not needed where min-p alone leaves few tokens, nor for a top_k of at most the number of threads: there
//      the threads' own largest logits, known from 1, are counted instead of all, and give a bin that is far enough down;
//   3. all tokens up to that bin (or above min-p's cut) are collected in rank 0's shared memory if they are at most 16384, with
//      the weight of the whole row where top-p asks for it (with min-p first roughly, in fp32: mostly the list is certain to
//      end before top-p does). Rank 0 sums them by bins of z, sorts the bins in which top-k and
//      top-p end, sums the kept ones by parts of the index range and sorts the part that holds the drawn point.
// More tokens than that (a wide nucleus, a temperature without cuts):
//   3'. exact sums of the weight above and between the boundary bins, whose own tokens are collected and sorted to give T and
//      T_idx; where the estimate of 2 was off, again with the neighbouring bin;
//   4'. the kept weight of every run of 256 tokens; the run that holds the drawn point is then walked by one warp.
// Where even one bin has more tokens than the list holds (long ties, very high temperatures) T and T_idx are found by
// bisection over keys and indices instead: slower, same result.
//
// Bound: rows * vocab * size bytes for large batches, then eleven fp64 operations a weight (fp64 runs at half the fp32 rate);
// for few rows the chain of passes and cluster barriers.
// Measured (device time): one row of 128256 fp16 logits, top-k 50 and top-p 0.9, 12 us (floor 0.04 us: five dependent steps of
// about 2 us); 128 rows of 202048 fp32 logits, top-p 0.95 and min-p 0.02, 90 us (floor 15.8 us; 60 us for most rows, the one with
// the longest list sets the time; with the row's weight in fp64 instead of roughly, 113 us). Of 128256 fp16 logits: 32 rows with top-k 50
// and top-p 0.9, 16 us, 96 rows 25 us; one row with top-p 0.9 alone, 35 us, 64 rows with 0.95, 104 us; 64 rows without cuts, 28 us; the
// largest logit of one row, 4.9 us.
#include "common.cuh"

#include <atomic>
#include <cmath>
#include <type_traits>

MUI_STATUS_ACCESSOR(sample)

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_CHUNK = 256;    // tokens of one warp step: eight consecutive ones per lane
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 16384;   // tokens collected at most
constexpr int SM_SMALL = 2048;   // tokens of one bin at most
constexpr int SM_MAX_VOCAB = 1 << 22;  // a part of an index range in SM_BINS parts fits the small list
constexpr int SM_FEW = 256;      // tokens that are compared pair by pair
constexpr int SM_RUNS = SM_THREADS;  // runs of chunks whose kept weight a CTA holds
constexpr int SM_MAX_CLUSTER = 8;
// what rank 0 finds in the collected tokens: the threshold, that top-p ends further up or down the ranking, or too many tokens
enum : uint32_t { SM_FOUND, SM_UP, SM_DOWN, SM_BISECT };
constexpr u64 SM_ENDLESS = ~0ull;  // a row's weight so large that top-p keeps all that was collected

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
// a token in ranking order: larger is further in front
__device__ __forceinline__ u64 rank_entry(float x, int i) {
  return static_cast<u64>(logit_key(x)) << 32 | ~static_cast<uint32_t>(i);
}

// ---- cluster helpers (also right for a cluster of one) ----
__device__ __forceinline__ unsigned cta_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync(int cluster) {
  if (cluster == 1) {
    __syncthreads();
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A peer's shared memory may be touched only once the peer runs: every thread says so first, and waits for the others' word
// before its CTA's first access, which costs nothing where there is work in between.
__device__ __forceinline__ void cluster_started(int cluster) {
  if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait_started(int cluster) {
  if (cluster > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* local, unsigned rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_peer_u64(u64* local, unsigned rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer_addr(local, rank)), "l"(v) : "memory");
}

struct Shared {
  u64 list[SM_LIST];                   // rank 0: rank_entry of collected tokens
  u64 small[SM_SMALL];                 // rank 0: those of one bin
  u64 small_w[SM_SMALL];               // weight of the sorted small list in front of each
  u64 mass[SM_BINS];
  uint32_t count[SM_BINS];
  uint32_t bins[SM_BINS];              // rank 0: the cluster's counts
  u64 runs[SM_RUNS];
  u64 part[SM_WARPS][3];
  u64 sums[2][SM_MAX_CLUSTER][3];      // every CTA's sums, two turns so that one barrier per exchange is enough
  u64 best[SM_MAX_CLUSTER];
  u64 warp_u64[SM_WARPS];
  float warp_f32[SM_WARPS];
  uint32_t warp_u32[SM_WARPS];
  uint32_t list_n[2];
  // rank 0's findings, and their copy in every CTA
  struct Say {
    uint32_t verdict, before_k, collect, small_bins, T, T_idx;
    int bin_k, bin_p;
  } say, said;
  float est_total;
  // a bin that rank 0 looks for, with what lies in front of it
  int bin;
  uint32_t bin_count, small_n;
  u64 bin_mass;
  int hit;
};

// Rank 0 hands its findings to every CTA of the cluster (all of them call this).
__device__ __forceinline__ void tell(Shared& s, int cluster, unsigned rank) {
  constexpr int WORDS = sizeof(Shared::Say) / 4;
  if (rank == 0) {
    __syncthreads();
    const int to = threadIdx.x / WORDS, word = threadIdx.x % WORDS;
    if (to < cluster)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(reinterpret_cast<uint32_t*>(&s.said) + word, to)),
                   "r"(reinterpret_cast<const uint32_t*>(&s.say)[word])
                   : "memory");
  }
  cluster_sync(cluster);
}

// Eight tokens as they sit in memory: 16 bytes, or twice 16 bytes of fp32. A lane's eight tokens of a chunk are consecutive
// 16-bit ones, or four and another four half a chunk on, so that a warp reads whole lines: token e is i + e + gap<T>(e).
struct Raw {
  uint4 a, b;
};
template <typename T>
__device__ __forceinline__ constexpr int gap(int e) {
  return sizeof(T) == 4 && e >= 4 ? SM_CHUNK / 2 - 4 : 0;
}
template <typename T>
__device__ __forceinline__ int lane_first(int chunk) {  // the lane's first token of a chunk
  return chunk * SM_CHUNK + static_cast<int>(threadIdx.x & 31) * (sizeof(T) == 4 ? 4 : 8);
}
template <typename T>
__device__ __forceinline__ Raw load_raw(const T* row, int i, int V, bool vec) {
  Raw r;
  if (vec && i + 8 + gap<T>(7) <= V) {
    const char* p = reinterpret_cast<const char*>(row) + static_cast<size_t>(i) * sizeof(T);
    r.a = ld_act16(p);
    if (sizeof(T) == 4) r.b = ld_act16(p + SM_CHUNK * 2);
    return r;
  }
  uint32_t w[8];  // NaN behind the end of the row
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int n = i + e + gap<T>(e);
    if (sizeof(T) == 4) w[e] = n < V ? __ldcg(reinterpret_cast<const uint32_t*>(row) + n) : 0x7fffffffu;
    else w[e] = i + e < V ? __ldcg(reinterpret_cast<const unsigned short*>(row) + i + e) : 0x7fffu;
  }
  if (sizeof(T) == 4) {
    r.a = make_uint4(w[0], w[1], w[2], w[3]);
    r.b = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack_raw(const Raw& r, float (&x)[8]) {
  if (sizeof(T) == 4) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
  } else {
    using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
    unpack8<H>(r.a, x);
  }
}

template <typename T>
struct Row {
  const T* p;
  int V, c0, c1;  // this CTA's chunks
  bool vec;
  // The largest logit is +infinity or the lowest finite number, so that nothing finite is below it: 0 stands for it then, and
  // -infinity for everything else. (Below the lowest number there would be no place for logits without weight.)
  bool alone;
  float peak;  // that logit
  __device__ __forceinline__ float stand_in(float x) const { return x == peak ? 0.f : -INFINITY; }
  __device__ __forceinline__ void unpack(const Raw& r, float (&x)[8]) const {
    unpack_raw<T>(r, x);
    if (alone) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = stand_in(x[e]);
    }
  }
  // f(first token of the lane, its eight logits) for every chunk of this CTA; warps take chunks in turn, the next four in
  // flight (64 KiB per CTA of fp32 logits: a round trip to L2 takes about a microsecond)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    int c = c0 + (threadIdx.x >> 5);
    auto get = [&](int n) {
      Raw q = {};
      if (n < c1) q = load_raw<T>(p, lane_first<T>(n), V, vec);
      return q;
    };
    Raw q0 = get(c), q1 = get(c + SM_WARPS), q2 = get(c + 2 * SM_WARPS), q3 = get(c + 3 * SM_WARPS);
#pragma unroll 1
    for (; c < c1; c += SM_WARPS) {
      float x[8];
      unpack(q0, x);
      q0 = q1;
      q1 = q2;
      q2 = q3;
      q3 = get(c + 4 * SM_WARPS);
      f(lane_first<T>(c), x);
    }
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights of one row. table: lane j of every warp holds 2^(j / 32).
struct Weigh {
  float top, floor, bin_scale;  // floor: at and below it a weight rounds to 0
  double scale, table;          // 32 / (ln 2 * temperature)
  int frac_bits;
  // bin of z; SM_BINS and above: no weight. Non-decreasing in the distance from the largest logit.
  __device__ __forceinline__ int bin(float x) const {
    const float b = (top - x) * bin_scale;
    return b < static_cast<float>(SM_BINS) ? static_cast<int>(b) : SM_BINS;  // NaN: SM_BINS
  }
  // 2^S exp(z) before rounding of N logits, x above the floor; whole warp. (logit - largest) * scale = 32 n + j + f, |f| <= 1/2: the
  // weight is 2^n * 2^(j/32) * 2^(f/32), the last one by its Taylor polynomial of degree 4 (error below 1.3e-12). Step by step
  // for all N, since one of these chains takes some 250 cycles.
  template <int N>
  __device__ __forceinline__ void values(const float (&x)[N], double (&p)[N]) const {
    constexpr double L = 0.021660849392498290;  // ln 2 / 32
    const double magic = 6755399441055744.0;    // 1.5 * 2^52: adding it rounds to a whole number, in the low bits
    double d[N], km[N];
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] = static_cast<double>(fmaxf(x[e], floor)) - static_cast<double>(top);
#pragma unroll
    for (int e = 0; e < N; ++e) km[e] = fma(d[e], scale, magic);
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] = fma(d[e], scale, magic - km[e]);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = fma(d[e], L * L * L * L / 24.0, L * L * L / 6.0);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = fma(p[e], d[e], L * L / 2.0);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = fma(p[e], d[e], L);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = fma(p[e], d[e], 1.0);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int k = __double2loint(km[e]);
      p[e] *= __shfl_sync(MUI_FULL_MASK, table, k);
      p[e] = __hiloint2double(__double2hiint(p[e]) + ((k >> 5) + frac_bits) * (1 << 20), __double2loint(p[e]));
    }
  }
  // 2^S exp(z) in fp32: off by less than 2^-14 of itself (z up to 46 with three roundings of 2^-24, and ex2's own error)
  __device__ __forceinline__ float rough(float x) const {
    return ex2((fmaxf(x, floor) - top) * static_cast<float>(scale * (1.0 / 32.0)) + static_cast<float>(frac_bits));
  }
  // values below 2^51 added to 2^52 leave their rounded sum in the mantissa
  static __device__ __forceinline__ u64 bits(double v) {
    return static_cast<u64>(__double_as_longlong(v)) & 0xfffffffffffffull;
  }
  // the weight as an integer; whole warp
  __device__ __forceinline__ u64 operator()(float x, bool use) const {
    const float in[1] = {x};
    double p[1];
    values(in, p);
    return use ? bits(p[0] + 4503599627370496.0) : 0ull;
  }
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(MUI_FULL_MASK, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_scan(V v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(MUI_FULL_MASK, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
// Exclusive sum over the CTA's threads; s_warp: one element per warp, free again after the next barrier.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* s_warp, V& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const V inc = warp_scan(v);
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  const V w = warp_scan(lane < SM_WARPS ? s_warp[lane] : V(0));
  all = __shfl_sync(MUI_FULL_MASK, w, 31);
  const V before = __shfl_sync(MUI_FULL_MASK, w, warp - 1);
  return inc - v + (warp ? before : V(0));
}

// Sums of three numbers over the cluster; every thread gets them. `turn` alternates from call to call.
__device__ __forceinline__ void cluster_sum3(Shared& s, int cluster, unsigned rank, int& turn, u64 (&v)[3]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 3; ++i) v[i] = warp_sum_u64(v[i]);
  if (lane == 0)
    for (int i = 0; i < 3; ++i) s.part[warp][i] = v[i];
  __syncthreads();
  if (warp < 3) {
    const u64 t = warp_sum_u64(lane < SM_WARPS ? s.part[lane][warp] : 0ull);
    if (lane < cluster) store_peer_u64(&s.sums[turn][rank][warp], lane, t);
  }
  cluster_sync(cluster);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = 0;
    for (int r = 0; r < cluster; ++r) v[i] += s.sums[turn][r][i];
  }
  turn ^= 1;
}

// The boundary of top-k and top-p by bisection: 32 steps over keys for each, then over indices for the ties.
template <typename T>
__device__ void threshold_by_bisection(Shared& s, const SampleArgs& a, const Row<T>& row, const Weigh& w, unsigned rank,
                                       int& turn, uint32_t best, bool use_k, uint32_t k, bool use_p, double top_p, uint32_t& T_key,
                                       uint32_t& T_idx) {
  // count and weight of the tokens with key >= pivot
  auto from = [&](uint32_t pivot, u64& count, u64& mass) {
    u64 v[3] = {0, 0, 0};
    row.each([&](int i, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = i + e + gap<T>(e) < a.V && logit_key(x[e]) >= pivot;
        v[0] += in;
        v[1] += w(x[e], in && w.bin(x[e]) < SM_BINS);
      }
    });
    cluster_sum3(s, a.cluster, rank, turn, v);
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
      for (int e = 0; e < 8; ++e) {
        const int n = i + e + gap<T>(e);
        v[0] += n < a.V && n <= static_cast<int>(mid) && logit_key(x[e]) == T_key;
      }
    });
    cluster_sum3(s, a.cluster, rank, turn, v);
    if (v[0] >= ties) hi = mid;
    else lo = mid + 1;
  }
  T_idx = lo;
}

// Sorts n entries, largest first. One CTA. A bitonic sort: two exchanges per thread and step for the largest list.
__device__ void sort_list(u64* list, int n) {
  const int tid = threadIdx.x;
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
      // exchanges closer than 64 entries stay within a warp, as does the step after such a one
      if (j > 32 || (j == 1 && 2 * k > 64)) __syncthreads();
      else __syncwarp();
    }
  __syncthreads();
}

// Leaves in w_before[i] the weight of the sorted list's tokens in front of the i-th; returns the weight of all of them. SHIFT:
// where the keys sit in the entries. One CTA.
template <int SHIFT>
__device__ u64 weigh_list(Shared& s, const u64* list, u64* w_before, int n, const Weigh& w) {
  const int per = (n + SM_THREADS - 1) / SM_THREADS, i0 = threadIdx.x * per;
  u64 sum = 0, all;
#pragma unroll 1
  for (int e = 0; e < per; ++e) {
    const bool in = i0 + e < n;
    const u64 q = w(in ? key_logit(static_cast<uint32_t>(list[i0 + e] >> SHIFT)) : 0.f, in);
    if (in) w_before[i0 + e] = q;
    sum += q;
  }
  u64 run = block_scan(sum, s.warp_u64, all);
#pragma unroll 1
  for (int e = 0; e < per; ++e)
    if (i0 + e < n) {
      const u64 q = w_before[i0 + e];
      w_before[i0 + e] = run;
      run += q;
    }
  __syncthreads();
  return all;
}

// number of leading entries i < n for which test(i) holds (it holds for a run from the front)
template <typename F>
__device__ __forceinline__ int leading(int n, F test) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (test(mid)) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  Shared& s = *reinterpret_cast<Shared*>(sample_smem);
  const int C = a.cluster, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned rank = C > 1 ? cta_rank() : 0;
  const int r = blockIdx.x / C;
  int turn = 0;
  cluster_started(C);
  pdl_wait_prior_grid();
  pdl_launch_dependents();

  Row<T> row;
  row.p = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  row.V = a.V;
  row.vec = (reinterpret_cast<uintptr_t>(row.p) & 15) == 0;
  row.alone = false;
  const int chunks = (a.V + SM_CHUNK - 1) / SM_CHUNK, per_cta = (chunks + C - 1) / C;
  row.c0 = min(chunks, static_cast<int>(rank) * per_cta);
  row.c1 = min(chunks, row.c0 + per_cta);
  float t = a.temperature ? __ldcg(a.temperature + r) : 1.f;
  const int k_raw = a.top_k ? __ldcg(a.top_k + r) : 0;
  const float top_p = a.top_p ? __ldcg(a.top_p + r) : 1.f;
  const float min_p = a.min_p ? __ldcg(a.min_p + r) : 0.f;
  const float uniform = __ldcg(a.uniforms + r);
  const bool use_k = k_raw > 0 && k_raw < a.V, use_p = top_p < 1.f, greedy = !(t > 0.f);

  // 1. the largest logit; its lowest index where that is the answer
  for (int i = tid; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0;
  if (tid < 2) s.list_n[tid] = 0;
  u64 best = 0;
  float m = -INFINITY;  // the thread's own
  if (greedy) {
    row.each([&](int i, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int n = i + e + gap<T>(e);
        const u64 v = rank_entry(x[e], n);
        best = n < a.V && v > best ? v : best;
      }
    });
  } else {
    int c = row.c0 + warp;
    for (; c + 7 * SM_WARPS < row.c1; c += 8 * SM_WARPS) {  // eight chunks of loads in flight, 128 KiB per CTA of fp32
      Raw q[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) q[h] = load_raw<T>(row.p, lane_first<T>(c + h * SM_WARPS), a.V, row.vec);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        float x[8];
        unpack_raw<T>(q[h], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
      }
    }
    for (; c < row.c1; c += SM_WARPS) {
      float x[8];
      unpack_raw<T>(load_raw<T>(row.p, lane_first<T>(c), a.V, row.vec), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
    }
    best = rank_entry(m, 0);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(MUI_FULL_MASK, best, o);
    best = y > best ? y : best;
  }
  if (lane == 0) s.warp_u64[warp] = best;
  __syncthreads();
  cluster_wait_started(C);
  if (warp == 0) {
    best = lane < SM_WARPS ? s.warp_u64[lane] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 y = __shfl_xor_sync(MUI_FULL_MASK, best, o);
      best = y > best ? y : best;
    }
    if (lane < C) store_peer_u64(&s.best[rank], lane, best);
  }
  cluster_sync(C);
  best = 0;
  for (int i = 0; i < C; ++i) best = s.best[i] > best ? s.best[i] : best;
  Weigh w;
  w.top = key_logit(static_cast<uint32_t>(best >> 32));
  const bool nothing = !(w.top > -INFINITY);  // key 0 (all NaN) reads as NaN
  if (greedy || nothing) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = nothing ? 0 : static_cast<int64_t>(~static_cast<uint32_t>(best));
      if (a.logprobs) a.logprobs[r] = nothing ? -INFINITY : 0.f;
    }
    return;
  }
  if (w.top == INFINITY || w.top == -3.402823466e38f) {
    row.alone = true;
    row.peak = w.top;
    w.top = 0.f;
  }
  const uint32_t best_key = logit_key(w.top);
  w.frac_bits = a.frac_bits;
  // z below -(S + 2) ln 2 has a weight under a quarter of the last bit. A temperature so small that the next smaller logit
  // lies beyond that, or so large that all logits are alike, is brought to where this is just the case. (10^29: the range, 3.5 * 10^30,
  // is below the distance of the largest fp32 numbers, so that the floor stays above the lowest one.)
  const float z_range = (a.frac_bits + 2) * 0.693147181f;
  t = fmaxf(fmaxf(fminf(t, 1e29f), (w.top - key_logit(best_key - 1)) / z_range), 1.17549435e-38f);
  w.floor = fmaxf(fminf(w.top - z_range * t, key_logit(best_key - 1)), -3.402823466e38f);
  w.scale = 46.166241308446828 / static_cast<double>(t);  // 32 / ln 2
  w.table = exp2(static_cast<double>(lane) / 32.0);
  // finite, so that the largest logit is in bin 0: next to logits of 0 the smallest temperatures only make the bins wider
  w.bin_scale = fminf(static_cast<float>(SM_BINS) / z_range / t, 3.402823466e38f);
  const u64 one = 1ull << a.frac_bits;
  // min-p in the integers of the weights (the largest token has weight 1 and always stays), and a logit safely below its cut
  const float min_w = fminf(min_p, 1.f);
  const u64 w_min = min_p > 0.f ? static_cast<u64>(ceil(static_cast<double>(min_w) * static_cast<double>(one))) : 1ull;
  const float x_min = min_p > 0.f ? w.top + t * (logf(min_w) - 1e-3f) - fabsf(w.top) * 1e-6f : -INFINITY;
  // uniform numbers lie in [0, 1); what does not is brought to the nearest fp32 that does
  const double u = static_cast<double>(fminf(fmaxf(uniform, 0.f), 0.99999994f));

  // Rank 0 turns a complete list of the tokens in front (n of them, `total` the weight of the row for top-p without top-k) into
  // the drawn token. cut_p: the list ends where top-p was expected to end; false is returned when it does not.
  // Few tokens, one per thread: the tokens in front of each, by rank and then by index, are found by looking at all of them.
  auto finish_few = [&](int n, u64 total, bool cut_p) {
    const u64 mine = tid < n ? s.list[tid] : 0;
    const u64 q = w(tid < n ? key_logit(static_cast<uint32_t>(mine >> 32)) : 0.f, tid < n);
    if (tid < n) s.small_w[tid] = q;
    __syncthreads();
    int place = 0;
    u64 front = 0;
    if (tid < n)
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const bool before = s.list[j] > mine;
        place += before;
        front += before ? s.small_w[j] : 0ull;
      }
    bool keep = tid < n && (!use_k || place < k_raw);
    u64 within;
    if (use_p) {
      block_scan(keep ? q : 0ull, s.warp_u64, within);
      const double target = static_cast<double>(top_p) * static_cast<double>(use_k ? within : total);
      if (cut_p && static_cast<double>(within) < target) return false;
      keep = keep && (place == 0 || static_cast<double>(front) < target);
    }
    keep = keep && q >= w_min;
    __syncthreads();
    if (tid < n) s.small_w[tid] = keep ? q : 0ull;
    u64 mass;
    block_scan(keep ? q : 0ull, s.warp_u64, mass);  // and a barrier
    if (!keep) return true;
    front = 0;
    const uint32_t index = ~static_cast<uint32_t>(mine);
#pragma unroll 4
    for (int j = 0; j < n; ++j) front += ~static_cast<uint32_t>(s.list[j]) < index ? s.small_w[j] : 0ull;
    // the first token at which the running weight exceeds the point
    const double want = u * static_cast<double>(mass);
    if (static_cast<double>(front + q) > want && static_cast<double>(front) <= want) {
      a.tokens[r] = static_cast<int64_t>(index);
      if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(q) / static_cast<double>(mass)));
    }
    return true;
  };
  // Inlined in every place: as a function it takes all of the state through memory (one row of fp16 logits 12 -> 20 us).
  auto finish = [&](int n, u64 total, bool cut_p) __attribute__((always_inline)) {
    if (n <= SM_FEW) return finish_few(n, total, cut_p);
    constexpr int PER = SM_BINS / SM_THREADS;
    uint32_t cn[PER], cb = 0;
    u64 mn[PER], mb = 0, all = 0;
    auto clear = [&]() {
      for (int i = tid; i < SM_BINS; i += SM_THREADS) {
        s.mass[i] = 0;
        s.count[i] = 0;
      }
      if (tid == 0) {
        s.bin = SM_BINS;
        s.small_n = 0;
      }
      __syncthreads();
    };
    // g(entry, its weight) for every token of the list; whole warps
    auto tokens = [&](auto g) {
#pragma unroll 1
      for (int base = 0; base < n; base += SM_THREADS) {
        const int i = base + tid;
        const u64 e = i < n ? s.list[i] : 0;
        const u64 q = w(i < n ? key_logit(static_cast<uint32_t>(e >> 32)) : 0.f, i < n);
        if (i < n) g(e, q);
      }
    };
    auto prefix = [&]() {
      __syncthreads();
      cb = 0;
      mb = 0;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        cn[h] = s.count[tid * PER + h];
        mn[h] = s.mass[tid * PER + h];
        cb += cn[h];
        mb += mn[h];
      }
      uint32_t unused;
      cb = block_scan(cb, s.warp_u32, unused);
      mb = block_scan(mb, s.warp_u64, all);
    };
    // the first bin for which hit(count in front, its count, weight in front, its weight) holds
    auto find = [&](auto hit) {
      uint32_t c = cb;
      u64 m = mb;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        if (cn[h] > 0 && hit(c, cn[h], m, mn[h])) atomicMin(&s.bin, tid * PER + h);
        c += cn[h];
        m += mn[h];
      }
      __syncthreads();
      c = cb;
      m = mb;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        if (s.bin == tid * PER + h) {
          s.bin_count = c;
          s.bin_mass = m;
        }
        c += cn[h];
        m += mn[h];
      }
      __syncthreads();
      return s.bin;
    };
    auto bin_of = [&](u64 e) { return min(w.bin(key_logit(static_cast<uint32_t>(e >> 32))), SM_BINS - 1); };
    // the tokens of a bin, sorted, with the weight in front of each; their number, over SM_SMALL: too many
    auto open_bin = [&](int bin) {
      for (int i = tid; i < n; i += SM_THREADS)
        if (bin_of(s.list[i]) == bin) {
          const uint32_t at = atomicAdd(&s.small_n, 1u);
          if (at < SM_SMALL) s.small[at] = s.list[i];
        }
      __syncthreads();
      const int m = s.small_n;
      __syncthreads();
      if (tid == 0) {
        s.small_n = 0;
        s.bin = SM_BINS;
      }
      if (m <= SM_SMALL) {
        sort_list(s.small, m);
        weigh_list<32>(s, s.small, s.small_w, m, w);
      }
      return m;
    };

    u64 edge = 0;  // entries from here on are kept
    bool cut = use_k || use_p;
    if (!use_k && use_p && total == SM_ENDLESS) {
      cut = false;
    } else if (!use_k && !cut_p && use_p) {  // less weight than top-p asks for: all are kept
      u64 sum = 0;
      tokens([&](u64, u64 q) { sum += q; });
      block_scan(sum, s.warp_u64, all);
      __syncthreads();
      cut = !(static_cast<double>(all) < static_cast<double>(top_p) * static_cast<double>(total));
    }
    if (cut) {
      clear();
      tokens([&](u64 e, u64 q) {
        const int b = bin_of(e);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], q);
      });
      prefix();
      u64 within = use_k ? all : total;
      if (use_k && n > k_raw) {
        const uint32_t k = static_cast<uint32_t>(k_raw);
        const int bin = find([&](uint32_t c, uint32_t nc, u64, u64) { return c < k && c + nc >= k; });
        const uint32_t left = k - s.bin_count;
        const u64 front = s.bin_mass;
        const int m = open_bin(bin);
        if (m > SM_SMALL) return false;
        edge = s.small[left - 1];
        const u64 last = w(key_logit(static_cast<uint32_t>(edge >> 32)), true);
        within = front + s.small_w[left - 1] + last;
        __syncthreads();
      }
      if (use_p) {
        const double target = static_cast<double>(top_p) * static_cast<double>(within);
        if (cut_p && static_cast<double>(all) < target) return false;
        const int bin = find([&](uint32_t c, uint32_t, u64 f, u64 m) {
          return static_cast<double>(f + m) >= target && (static_cast<double>(f) < target || c == 0);
        });
        if (bin < SM_BINS) {
          const u64 front = s.bin_mass;
          const int m = open_bin(bin);
          if (m > SM_SMALL) return false;
          // tokens whose predecessors do not reach the target are kept, the first of all in any case
          const int kept = max(1, leading(m, [&](int i) { return static_cast<double>(front + s.small_w[i]) < target; }));
          const u64 e = s.small[kept - 1];
          edge = e > edge ? e : edge;
          __syncthreads();
        }
      }
    }
    // the kept ones by index
    clear();
    int shift = 0;
    while ((a.V - 1) >> shift >= SM_BINS) ++shift;
    auto index_of = [](u64 e) { return static_cast<int>(~static_cast<uint32_t>(e)); };
    tokens([&](u64 e, u64 q) {
      if (e >= edge && q >= w_min) {
        atomicAdd(&s.count[index_of(e) >> shift], 1u);
        atomicAdd(&s.mass[index_of(e) >> shift], q);
      }
    });
    prefix();
    const double want = u * static_cast<double>(all);
    const int part = find([&](uint32_t, uint32_t, u64 f, u64 m) {
      return static_cast<double>(f + m) > want && static_cast<double>(f) <= want;
    });
#pragma unroll 1
    for (int base = 0; base < n; base += SM_THREADS) {
      const int i = base + tid;
      const u64 e = i < n ? s.list[i] : 0;
      const bool here = i < n && e >= edge && index_of(e) >> shift == part;
      if (!__any_sync(MUI_FULL_MASK, here)) continue;
      const u64 q = w(here ? key_logit(static_cast<uint32_t>(e >> 32)) : 0.f, here);
      if (here && q >= w_min) s.small[atomicAdd(&s.small_n, 1u)] = e << 32 | e >> 32;  // ~index, key
    }
    __syncthreads();
    const int m = s.small_n;
    sort_list(s.small, m);
    const u64 in_part = weigh_list<0>(s, s.small, s.small_w, m, w);
    for (int i = tid; i < m; i += SM_THREADS) {
      // the first token at which the running weight exceeds the point
      const u64 from = s.bin_mass + s.small_w[i], to = s.bin_mass + (i + 1 < m ? s.small_w[i + 1] : in_part);
      if (static_cast<double>(to) > want && static_cast<double>(from) <= want) {
        a.tokens[r] = static_cast<int64_t>(~static_cast<uint32_t>(s.small[i] >> 32));
        if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(to - from) / static_cast<double>(all)));
      }
    }
    return true;
  };
  // Collects the tokens that in(x) names in rank 0's list. v[0]: the weight of the whole row if asked for, v[1]: their number if
  // asked for (over SM_LIST: the list is incomplete).
  const uint32_t count_at[2] = {peer_addr(&s.list_n[0], 0), peer_addr(&s.list_n[1], 0)};
  const uint32_t list_at[2] = {peer_addr(s.list, 0), peer_addr(s.small, 0)};
  auto put = [&](int which, float x, int i, uint32_t room) {
    uint32_t at;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count_at[which]) : "memory");
    if (at < room)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list_at[which] + at * 8), "l"(rank_entry(x, i)) : "memory");
  };
  u64 v[3];
  enum { NO_WEIGHT, ROUGH, EXACT };
  auto collect = [&](auto in, int weigh, bool count) {
    v[0] = v[1] = v[2] = 0;
    float rough = 0.f;
    row.each([&](int i, float(&x)[8]) {
      if (weigh == ROUGH) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += w.rough(x[e]);
        rough += sum;
      } else if (weigh == EXACT) {
        double p[8], sum = 4503599627370496.0;  // 2^52
        w.values(x, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += p[e];
        v[0] += Weigh::bits(sum);
      }
      // places in the list are taken once for the warp
      unsigned mine = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) mine |= in(x[e]) ? 1u << e : 0u;
      if (__any_sync(MUI_FULL_MASK, mine != 0)) {
        const uint32_t upto = warp_scan(static_cast<uint32_t>(__popc(mine)));
        uint32_t at = 0;
        if (C == 1) {
          if ((tid & 31) == 31) at = atomicAdd(&s.list_n[0], upto);
        } else if ((tid & 31) == 31)
          asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(at) : "r"(count_at[0]), "r"(upto) : "memory");
        at = __shfl_sync(MUI_FULL_MASK, at, 31) + upto - __popc(mine);
        v[1] += __popc(mine);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (mine >> e & 1) {
            if (at < SM_LIST)
              asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list_at[0] + at * 8), "l"(rank_entry(x[e], i + e + gap<T>(e)))
                           : "memory");
            ++at;
          }
      }
    });
    if (weigh == ROUGH) v[0] = static_cast<u64>(rough);
    // a barrier of the cluster either way: it publishes the list
    if (weigh != NO_WEIGHT || count) cluster_sum3(s, C, rank, turn, v);
    else cluster_sync(C);
  };

  uint32_t T_key = 0, T_idx = 0;  // nothing to cut: every key that has weight is above 0
  bool bisect = false;
  if (min_p > 0.f && !use_k) {
    // Where the collected tokens are certain to end before top-p does, a rough weight of the row is enough: it is off by less
    // than 2^-14, and as much again for the fp32 sums of a thread (at most 2^22 / 4096 + 8 additions). Less 2^-10 it is a bound.
    collect([&](float x) { return x >= x_min; }, use_p ? ROUGH : NO_WEIGHT, true);
    if (v[1] <= SM_LIST) {
      const int n = static_cast<int>(v[1]);
      bool cuts = use_p;  // top-p may end within the list
      if (use_p) {
        if (rank == 0) {
          const u64 least = v[0] - (v[0] >> 10);
          u64 sum = 0, listed;
#pragma unroll 1
          for (int base = 0; base < n; base += SM_THREADS) {
            const int i = base + tid;
            sum += w(i < n ? key_logit(static_cast<uint32_t>(s.list[i] >> 32)) : 0.f, i < n);
          }
          block_scan(sum, s.warp_u64, listed);
          const bool sure = static_cast<double>(listed) < static_cast<double>(top_p) * static_cast<double>(least);
          v[0] = SM_ENDLESS;
          if (tid == 0) s.say.verdict = sure ? SM_FOUND : SM_BISECT;
        }
        tell(s, C, rank);
        cuts = s.said.verdict != SM_FOUND;
        if (cuts) collect([](float) { return false; }, EXACT, false);
      }
      // a list that is not cut, or of few tokens, is always brought to an end
      const bool ends = !cuts || n <= SM_FEW;
      if (ends && rank != 0) return;
      if (rank == 0) {
        const bool ok = finish(n, v[0], false);
        if (ends) return;
        __syncthreads();
        if (tid == 0) s.say.verdict = ok ? SM_FOUND : SM_UP;
      }
      tell(s, C, rank);
      if (s.said.verdict == SM_FOUND) return;
      // top-p ends in a bin of more tokens than are sorted
    }
    if (tid == 0) s.list_n[0] = 0;  // a barrier follows before the next token is put there
  }
  // bins of all CTAs summed in rank 0's
  auto join_bins = [&]() {
    if (rank != 0) {
      __syncthreads();
      for (int i = tid; i < SM_BINS; i += SM_THREADS)
        if (const uint32_t n = s.bins[i])
          asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(peer_addr(&s.bins[i], 0)), "r"(n) : "memory");
    }
    cluster_sync(C);
  };
  if (use_k && k_raw <= C * SM_THREADS) {
    // The largest logits of k threads are k tokens: whatever the bin of the k-th of them, the top-k lie in the bins up to it.
    if (row.alone) m = row.stand_in(m);
    const int mine = w.bin(m);
    if (mine < SM_BINS) atomicAdd(&s.bins[mine], 1u);
    join_bins();
    if (rank == 0) {
      constexpr int PER = SM_BINS / SM_THREADS;
      const uint32_t k = static_cast<uint32_t>(k_raw);
      uint32_t n[PER], at = 0, all;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        n[h] = s.bins[PER * tid + h];
        at += n[h];
      }
      if (tid == 0) s.say.bin_k = SM_BINS;
      at = block_scan(at, s.warp_u32, all);
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        if (at < k && at + n[h] >= k) s.say.bin_k = PER * tid + h;  // one thread at most
        at += n[h];
      }
    }
    tell(s, C, rank);
    const int last = s.said.bin_k;
    collect([&](float x) { return w.bin(x) <= min(last, SM_BINS - 1); }, NO_WEIGHT, true);
    if (v[1] <= SM_LIST) {
      // few tokens are always brought to an end
      if (rank != 0 && v[1] <= SM_FEW) return;
      if (rank == 0) {
        const bool ok = finish(static_cast<int>(v[1]), 0, false);
        if (v[1] <= SM_FEW) return;
        __syncthreads();
        if (tid == 0) s.say.verdict = ok ? SM_FOUND : SM_UP;
      }
      tell(s, C, rank);
      if (s.said.verdict == SM_FOUND) return;
    }
    for (int i = tid; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0;
    if (tid == 0) s.list_n[0] = 0;
    cluster_sync(C);
  }
  if (use_k || use_p) {
    // 2. histogram
    row.each([&](int, float(&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int b = w.bin(x[e]);
        if (b < SM_BINS) atomicAdd(&s.bins[b], 1u);
      }
    });
    join_bins();
    constexpr int PER = SM_BINS / SM_THREADS;
    const uint32_t k = static_cast<uint32_t>(k_raw);
    if (rank == 0) {
      // prefix sums over the bins, four per thread: counts, and weights of the bin centres
      if (tid == 0) {
        s.say.bin_k = s.say.bin_p = SM_BINS;
        s.say.before_k = 0;
        s.say.small_bins = 1;
      }
      uint32_t n[PER], nc = 0, n_all;
      float m[PER], mc = 0.f, all;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        n[h] = s.bins[PER * tid + h];
        m[h] = n[h] * exp2f(-(PER * tid + h + 0.5f) * (z_range * 1.44269504f / SM_BINS));
        nc += n[h];
        mc += m[h];
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < PER; ++h)
        if (n[h] > SM_SMALL) s.say.small_bins = 0;
      const uint32_t nb = block_scan(nc, s.warp_u32, n_all);
      const float mb = block_scan(mc, s.warp_f32, all);
      if (use_k) {
        if (tid == 0) s.est_total = all;
        __syncthreads();
        uint32_t at = nb;
        float am = mb;
#pragma unroll
        for (int h = 0; h < PER; ++h) {
          if (at < k && at + n[h] >= k) {  // one thread at most
            s.say.bin_k = PER * tid + h;
            s.say.before_k = at;
            s.est_total = am + m[h] * (k - at) / n[h];
          }
          at += n[h];
          am += m[h];
        }
        __syncthreads();
        all = s.est_total;
      }
      const int bin_k = s.say.bin_k;
      if (use_p) {
        const float target = top_p * all;
        uint32_t at = nb;
        float am = mb;
#pragma unroll
        for (int h = 0; h < PER; ++h) {
          // the first occupied bin with which the sum reaches the target
          if (n[h] > 0 && am + m[h] >= target && (am < target || at == 0)) atomicMin(&s.say.bin_p, PER * tid + h);
          at += n[h];
          am += m[h];
        }
        __syncthreads();
      }
      const int bin_p = use_p ? min(s.say.bin_p, bin_k) : bin_k;
      // tokens up to the last bin that matters; top-p without top-k takes a bin more, since it is an estimate
      const int last = use_k ? bin_k : min(bin_p + 1, SM_BINS);
      if (last < SM_BINS && tid == last / PER) {
        uint32_t upto = nb;
#pragma unroll
        for (int h = 0; h < PER; ++h)
          if (PER * tid + h <= last) upto += n[h];
        s.say.collect = upto <= SM_LIST;
      } else if (last >= SM_BINS && tid == 0) {
        s.say.collect = n_all <= SM_LIST;
      }
      __syncthreads();
      if (tid == 0) s.say.bin_p = bin_p;
    }
    tell(s, C, rank);
    const int bin_k = s.said.bin_k;
    int bin_p = s.said.bin_p;
    const uint32_t before_k = s.said.before_k;
    if (s.said.collect) {
      // 3. the tokens in front
      const int last = use_k ? bin_k : min(bin_p + 1, SM_BINS);
      collect([&](float x) { return w.bin(x) < SM_BINS && w.bin(x) <= last; }, use_p && !use_k ? EXACT : NO_WEIGHT, false);
      // with top-k the list is complete for sure: only rank 0 goes on
      const bool sure = use_k && s.said.small_bins;
      if (sure && rank != 0) return;
      if (rank == 0) {
        const bool ok = finish(static_cast<int>(s.list_n[0]), v[0], use_p && !use_k && last < SM_BINS);
        if (sure) return;
        __syncthreads();
        if (tid == 0) {
          s.say.verdict = ok ? SM_FOUND : SM_UP;
          s.list_n[0] = 0;
        }
      }
      tell(s, C, rank);
      if (s.said.verdict == SM_FOUND) return;
    }
    bisect = use_p || bin_k < SM_BINS;  // a top_p next to 1 may end in no bin
    for (int attempt = 0; attempt < 4 && bin_p < SM_BINS; ++attempt) {
      // 3'. exact sums: [0] above bin_p, [1] between the bins; tokens of the bins go to rank 0
      v[0] = v[1] = v[2] = 0;
      row.each([&](int i, float(&x)[8]) {
        double above = 4503599627370496.0, between = above;
        bool mine = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int b = w.bin(x[e]);
          mine |= use_p && b < bin_k && b != bin_p && b < SM_BINS;
          if (b < SM_BINS && (b == bin_p || b == bin_k)) put(b == bin_p ? 0 : 1, x[e], i + e + gap<T>(e), SM_SMALL);
        }
        if (__any_sync(MUI_FULL_MASK, mine)) {
          double p[8];
          w.values(x, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int b = w.bin(x[e]);
            above += b < bin_p ? p[e] : 0.0;
            between += b > bin_p && b < bin_k ? p[e] : 0.0;
          }
          v[0] += Weigh::bits(above);
          v[1] += Weigh::bits(between);
        }
      });
      cluster_sum3(s, C, rank, turn, v);  // its barrier also publishes the lists
      if (rank == 0) {
        const int n0 = s.list_n[0], n1 = s.list_n[1];
        const bool same = bin_p == bin_k;
        uint32_t say = SM_BISECT;
        int next = bin_p;
        if (n0 <= SM_SMALL && n1 <= SM_SMALL) {
          const uint32_t left = k - before_k;  // tokens of bin_k within the top-k
          u64 in_k = 0;
          u64 last = 0;
          if (!same && bin_k < SM_BINS) {
            sort_list(s.small, n1);
            const u64 bin_mass = weigh_list<32>(s, s.small, s.small_w, n1, w);
            in_k = left < static_cast<uint32_t>(n1) ? s.small_w[left] : bin_mass;
            __syncthreads();
          }
          const int n_p = same ? static_cast<int>(min(left, static_cast<uint32_t>(n0))) : n0;  // of bin_p within the top-k
          sort_list(s.list, n0);
          u64 in_p = weigh_list<32>(s, s.list, s.small_w, n0, w);
          if (n_p < n0) in_p = s.small_w[n_p];
          if (!use_p) {
            last = s.list[n_p - 1];
            say = SM_FOUND;
          } else {
            const double target = static_cast<double>(top_p) * static_cast<double>(v[0] + v[1] + in_p + in_k);
            // the estimate of step 2 may be a bin off
            if (v[0] != 0 && static_cast<double>(v[0]) >= target) say = SM_UP;
            else if (static_cast<double>(v[0] + in_p) < target) say = SM_DOWN;
            else {
              // tokens whose predecessors do not reach the target are kept, the first of all in any case
              const int kept = leading(n_p, [&](int i) { return static_cast<double>(v[0] + s.small_w[i]) < target; });
              last = s.list[max(1, kept) - 1];
              say = SM_FOUND;
            }
          }
          if (say == SM_UP || say == SM_DOWN) {  // the neighbour that holds tokens
            const int step = say == SM_UP ? -1 : 1;
            do next += step;
            while (next >= 0 && next < SM_BINS && s.bins[next] == 0);
            if (next < 0 || next > bin_k || next >= SM_BINS) say = SM_BISECT;
          }
          if (tid == 0) {
            s.say.T = static_cast<uint32_t>(last >> 32);
            s.say.T_idx = ~static_cast<uint32_t>(last);
          }
        }
        __syncthreads();
        if (tid == 0) {
          s.say.verdict = say;
          s.say.bin_p = next;
        }
        if (tid < 2) s.list_n[tid] = 0;
      }
      tell(s, C, rank);
      const uint32_t verdict = s.said.verdict;
      bin_p = s.said.bin_p;
      T_key = s.said.T;
      T_idx = s.said.T_idx;
      cluster_sync(C);  // the findings have been read before rank 0 has others
      bisect = verdict != SM_FOUND;
      if (verdict == SM_FOUND || verdict == SM_BISECT) break;
    }
    if (bisect)
      threshold_by_bisection<T>(s, a, row, w, rank, turn, best_key, use_k, k, use_p, static_cast<double>(top_p), T_key, T_idx);
  }

  // 4'. kept weight by runs of chunks
  for (int i = tid; i < SM_RUNS; i += SM_THREADS) s.runs[i] = 0;
  __syncthreads();
  const float T_logit = T_key ? key_logit(T_key) : -INFINITY;
  const float x_low = fmaxf(fmaxf(T_logit, x_min), w.floor);
  // weights of the lane's eight tokens that are kept; whole warp
  auto kept_weights = [&](int i, const float(&x)[8], u64(&q)[8]) {
    double p[8];
    w.values(x, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = x[e] > T_logit || (x[e] == T_logit && i + e + gap<T>(e) <= static_cast<int>(T_idx));
      q[e] = Weigh::bits(p[e] + 4503599627370496.0);
      q[e] = in && q[e] >= w_min ? q[e] : 0ull;
    }
  };
  v[0] = v[1] = v[2] = 0;
  row.each([&](int i, float(&x)[8]) {
    bool some = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) some |= x[e] >= x_low;
    if (__any_sync(MUI_FULL_MASK, some)) {
      u64 q[8], sum = 0;
      kept_weights(i, x, q);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += q[e];
      v[0] += sum;
      sum = warp_sum_u64(sum);
      if (lane == 0 && sum) atomicAdd(&s.runs[(i / SM_CHUNK - row.c0) / a.chunks_per_run], sum);
    }
  });
  const int my_turn = turn;
  cluster_sum3(s, C, rank, turn, v);
  const u64 total = v[0], mine = s.sums[my_turn][rank][0];
  u64 before = 0;
  for (unsigned i = 0; i < rank; ++i) before += s.sums[my_turn][i][0];
  const double want = u * static_cast<double>(total);
  if (mine == 0 || static_cast<double>(before) > want || static_cast<double>(before + mine) <= want) return;

  // this CTA holds the drawn point: first its run, then its chunk and token
  {
    const u64 q = s.runs[tid];
    u64 all;
    const u64 at = before + block_scan(q, s.warp_u64, all);
    if (q != 0 && static_cast<double>(at + q) > want && static_cast<double>(at) <= want) {
      s.hit = tid;
      s.best[0] = at;  // weight in front of the run
    }
    __syncthreads();
  }
  if (warp != 0) return;
  u64 at = s.best[0];
  const int first = row.c0 + s.hit * a.chunks_per_run, last = min(row.c1, first + a.chunks_per_run);
  for (int c = first; c < last; ++c) {
    float x[8];
    u64 q[8];
    const int i = lane_first<T>(c);
    row.unpack(load_raw<T>(row.p, i, a.V, row.vec), x);
    kept_weights(i, x, q);
    // tokens in index order: all eight of a lane, or the first four of all lanes and then the other four
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, N = 8 / PARTS;
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) sum += q[h * N + e];
      const u64 run = warp_scan(sum);
      const unsigned hit = __ballot_sync(MUI_FULL_MASK, sum != 0 && static_cast<double>(at + run) > want);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          u64 upto = at + run;
          int token = 0;
          u64 weight = 0;
#pragma unroll
          for (int e = N - 1; e >= 0; --e) {  // the first token at which the running weight exceeds the point
            const u64 mine_w = q[h * N + e];
            if (mine_w != 0 && static_cast<double>(upto) > want) {
              token = i + h * N + e + gap<T>(h * N + e);
              weight = mine_w;
            }
            upto -= mine_w;
          }
          a.tokens[r] = token;
          if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(weight) / static_cast<double>(total)));
        }
        return;
      }
      at += __shfl_sync(MUI_FULL_MASK, run, 31);
    }
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
  MUI_REQUIRE(rows >= 0 && rows <= (1 << 24) && vocab >= 1 && vocab <= SM_MAX_VOCAB && row_stride >= 0,
              MUI_ERR_INVALID_ARG, "bad sizes rows=%d (0..2^24) vocab=%d (1..2^22) row_stride=%lld", rows, vocab,
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
  a.frac_bits = 62 - lg < 48 ? 62 - lg : 48;
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
