// Drawing a token from each row of logits: temperature, top-k, top-p, min-p, inverse transform of a given uniform number.
//
// With d = (logit - largest) / temperature and w = exp(d), the kept tokens are a run from the front of the ranking by
// (logit descending, index ascending): all tokens above a threshold logit and the first few at it. No sort is needed, only
// the threshold: the largest key T for which the tokens >= T number top_k, or weigh top_p of the total.
//
// Sums of weights decide which token is drawn, so they must not depend on the order in which threads add: w is taken in
// fp64 and rounded once to a 64-bit integer with S fraction bits (S = 62 - ceil(log2 vocab), 44 for 200 k tokens: no sum
// overflows), and integers are summed. Against real arithmetic a boundary is off by at most vocab * 2^-(S+1) of the largest
// weight, about 1e-8 in the worst case and sqrt(vocab) * 2^-S in practice.
#include "common.cuh"

#include <cmath>

MUI_STATUS_ACCESSOR(sample)

namespace {

constexpr int SM_THREADS = 1024;
constexpr int SM_WARPS = SM_THREADS / 32;

struct SampleArgs {
  const void* logits;
  long long stride;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t* top_k;
  int64_t* tokens;
  float* logprobs;
  int V, frac_bits;
};

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int i) {
  return ld_act_f32<T>(row + i);
}
template <>
__device__ __forceinline__ float logit_at<float>(const float* row, int i) {
  return __ldcg(row + i);
}

// order-preserving key of a logit: larger logit, larger key; -0 equals +0; NaN is below everything (key 0)
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;  // key of -infinity; at or below it a token has no weight

struct Weigh {
  double inv_t;
  float top;
  double one;  // 2^frac_bits
  __device__ __forceinline__ double real(float x) const {
    if (x == top) return 1.0;
    return exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
  }
  __device__ __forceinline__ unsigned long long operator()(uint32_t key) const {
    if (key <= KEY_NEG_INF) return 0ull;
    return static_cast<unsigned long long>(__double2ll_rn(real(key_logit(key)) * one));
  }
};

struct Sums {
  unsigned long long count, mass;
};
// block-wide sum over all tokens with key >= pivot
template <typename T>
__device__ Sums sum_from(const T* row, int V, uint32_t pivot, const Weigh& w, bool want_mass, Sums* s_part) {
  Sums r = {0, 0};
  for (int i = threadIdx.x; i < V; i += SM_THREADS) {
    const uint32_t k = logit_key(logit_at<T>(row, i));
    if (k >= pivot) {
      r.count += 1;
      if (want_mass) r.mass += w(k);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    r.count += __shfl_xor_sync(MUI_FULL_MASK, r.count, o);
    r.mass += __shfl_xor_sync(MUI_FULL_MASK, r.mass, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = r;
  __syncthreads();
  r = {0, 0};
  for (int i = 0; i < SM_WARPS; ++i) {
    r.count += s_part[i].count;
    r.mass += s_part[i].mass;
  }
  return r;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleArgs a) {
  __shared__ Sums s_part[SM_WARPS];
  __shared__ uint32_t s_key[SM_WARPS];
  __shared__ int s_idx[SM_WARPS];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int r = blockIdx.x, V = a.V, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  // largest key, lowest index
  uint32_t best = 0;
  int best_i = 0x7fffffff;
  for (int i = tid; i < V; i += SM_THREADS) {
    const uint32_t k = logit_key(logit_at<T>(row, i));
    if (k > best || (k == best && i < best_i)) {
      best = k;
      best_i = i;
    }
  }
  auto fold = [&](uint32_t ok, int oi) {
    if (ok > best || (ok == best && oi < best_i)) {
      best = ok;
      best_i = oi;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    fold(__shfl_xor_sync(MUI_FULL_MASK, best, o), __shfl_xor_sync(MUI_FULL_MASK, best_i, o));
  if (lane == 0) {
    s_key[warp] = best;
    s_idx[warp] = best_i;
  }
  __syncthreads();
  for (int i = 0; i < SM_WARPS; ++i) fold(s_key[i], s_idx[i]);
  const float t = a.temperature ? __ldcg(a.temperature + r) : 1.f;
  if (best <= KEY_NEG_INF || !(t > 0.f)) {
    if (tid == 0) {
      a.tokens[r] = best <= KEY_NEG_INF ? 0 : best_i;
      if (a.logprobs) a.logprobs[r] = best <= KEY_NEG_INF ? -INFINITY : 0.f;
    }
    return;
  }
  Weigh w;
  w.inv_t = 1.0 / static_cast<double>(t);
  w.top = key_logit(best);
  w.one = static_cast<double>(1ull << a.frac_bits);

  // top-k: largest T with at least k tokens at or above it
  const int k_raw = a.top_k ? __ldcg(a.top_k + r) : 0;
  const bool use_k = k_raw > 0 && k_raw < V;
  const float top_p = a.top_p ? __ldcg(a.top_p + r) : 1.f;
  const float min_p = a.min_p ? __ldcg(a.min_p + r) : 0.f;
  uint32_t T_key = 0;                     // kept: key > T_key, and the first `ties` at it
  unsigned long long ties = ~0ull;
  unsigned long long above_mass = 0;
  if (use_k) {
    uint32_t lo = 0, hi = best;  // count(>= lo) >= k
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (sum_from<T>(row, V, mid, w, false, s_part).count >= static_cast<unsigned long long>(k_raw)) lo = mid;
      else hi = mid - 1;
    }
    T_key = lo;
    const Sums up = lo == 0xffffffffu ? Sums{0, 0} : sum_from<T>(row, V, lo + 1, w, true, s_part);
    ties = k_raw - up.count;
    above_mass = up.mass;
  }
  if (top_p < 1.f) {
    const unsigned long long total =
        use_k ? above_mass + ties * w(T_key) : sum_from<T>(row, V, 0, w, true, s_part).mass;
    const double target = static_cast<double>(top_p) * static_cast<double>(total);
    // largest P whose tokens at or above (within the top-k) weigh the target
    auto mass_from = [&](uint32_t p) {
      if (use_k && p <= T_key) return total;
      return sum_from<T>(row, V, p, w, true, s_part).mass;
    };
    uint32_t lo = T_key, hi = best;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (static_cast<double>(mass_from(mid)) >= target) lo = mid;
      else hi = mid - 1;
    }
    const Sums up = lo == 0xffffffffu ? Sums{0, 0} : sum_from<T>(row, V, lo + 1, w, true, s_part);
    const double each = static_cast<double>(w(lo));
    unsigned long long n = 1;
    if (each > 0.0) {
      const double need = ceil((target - static_cast<double>(up.mass)) / each);
      n = need < 1.0 ? 1ull : (need > 4.0e9 ? ~0ull : static_cast<unsigned long long>(need));
    }
    if (lo > T_key || !use_k) {
      T_key = lo;
      ties = n;
    } else {
      ties = n < ties ? n : ties;
    }
  }
  // the smallest key that min-p keeps is found by evaluating w itself
  const double min_w = min_p > 0.f ? static_cast<double>(min_p) : -1.0;
  auto keeps = [&](uint32_t k) { return k > KEY_NEG_INF && (min_w < 0.0 || w.real(key_logit(k)) >= min_w || k == best); };

  // each warp takes a run of the row: ties and weight above the threshold in it
  const int per = (V + SM_WARPS - 1) / SM_WARPS, i0 = warp * per, i1 = min(V, i0 + per);
  Sums mine = {0, 0};
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t k = logit_key(logit_at<T>(row, i));
    if (k == T_key) mine.count += 1;
    else if (k > T_key && keeps(k)) mine.mass += w(k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mine.count += __shfl_xor_sync(MUI_FULL_MASK, mine.count, o);
    mine.mass += __shfl_xor_sync(MUI_FULL_MASK, mine.mass, o);
  }
  __syncthreads();
  if (lane == 0) s_part[warp] = mine;
  __syncthreads();
  const unsigned long long tie_w = keeps(T_key) ? w(T_key) : 0ull;
  unsigned long long left = ties, before = 0, total = 0, my_left = 0;
  for (int i = 0; i < SM_WARPS; ++i) {
    if (i == warp) {
      my_left = left;
      before = total;
    }
    const unsigned long long n = s_part[i].count < left ? s_part[i].count : left;
    left -= n;
    total += s_part[i].mass + n * tie_w;
    if (i == warp) mine.mass = s_part[i].mass + n * tie_w;
  }
  const float u = a.uniforms ? __ldcg(a.uniforms + r) : 0.f;
  // uniform numbers lie in [0, 1); what does not is brought to the nearest fp32 that does
  const double want = static_cast<double>(fminf(fmaxf(u, 0.f), 0.99999994f)) * static_cast<double>(total);
  // the warp whose run holds the point walks it
  if (mine.mass == 0 || static_cast<double>(before) > want || static_cast<double>(before + mine.mass) <= want) return;
  unsigned long long run = before;
  for (int base = i0; base < i1; base += 32) {
    const int i = base + lane;
    const uint32_t k = i < i1 ? logit_key(logit_at<T>(row, i)) : 0u;
    const unsigned tie_mask = __ballot_sync(MUI_FULL_MASK, i < i1 && k == T_key);
    const unsigned long long rank = __popc(tie_mask & ((1u << lane) - 1));
    unsigned long long x = 0;
    if (i < i1) {
      if (k == T_key) x = rank < my_left ? tie_w : 0ull;
      else if (k > T_key && keeps(k)) x = w(k);
    }
    my_left -= min(my_left, static_cast<unsigned long long>(__popc(tie_mask)));
    unsigned long long c = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(MUI_FULL_MASK, c, o);
      if (lane >= o) c += y;
    }
    const unsigned hit = __ballot_sync(MUI_FULL_MASK, static_cast<double>(run + c) > want);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.tokens[r] = i;
        if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(x) / static_cast<double>(total)));
      }
      return;
    }
    run += __shfl_sync(MUI_FULL_MASK, c, 31);
  }
}

}  // namespace

extern "C" mui_status_t mui_sample_tokens(void* stream, int dtype, int rows, int vocab, const void* logits,
                                          int64_t row_stride, const float* temperature, const int32_t* top_k,
                                          const float* top_p, const float* min_p, const float* uniforms,
                                          int64_t* tokens, float* logprobs, unsigned flags) {
  MUI_REQUIRE(dtype == MUI_F16 || dtype == MUI_BF16 || dtype == MUI_COMM_F32, MUI_ERR_UNSUPPORTED,
              "dtype %d unsupported", dtype);
  MUI_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= (1 << 24) && row_stride >= 0, MUI_ERR_INVALID_ARG,
              "bad sizes rows=%d vocab=%d (1..2^24) row_stride=%lld", rows, vocab, (long long)row_stride);
  if (rows == 0) return MUI_OK;
  MUI_REQUIRE(logits && uniforms && tokens, MUI_ERR_INVALID_ARG, "logits, uniforms and tokens must be non-null");
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
  a.frac_bits = 62 - lg;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int pdl = (flags & MUI_FLAG_PDL) ? 1 : 0;
  const dim3 grid(rows), block(SM_THREADS);
  if (dtype == MUI_F16) {
    MUI_CUDA_CHECK(mui_launch(sample_kernel<__half>, grid, block, 0, st, pdl, a));
  } else if (dtype == MUI_BF16) {
    MUI_CUDA_CHECK(mui_launch(sample_kernel<__nv_bfloat16>, grid, block, 0, st, pdl, a));
  } else {
    MUI_CUDA_CHECK(mui_launch(sample_kernel<float>, grid, block, 0, st, pdl, a));
  }
  return MUI_OK;
}
