// The next token of every row from its logits and one given random number.
//
// Row r with temperature t > 0: a token weighs w = exp((l - max l) / t). Tokens are ordered by falling logit,
// equal ones by index. Of them top-k keeps the first k; top-p of those the shortest beginning whose weight reaches
// the share p of theirs; min-p of those the ones with w >= min_p. The token is the least index at which the kept
// weights' running sum passes u times their total. What is kept is therefore a border in the order: all logits
// above one value, and of those equal to it the first few by index.
//
// Weights are whole numbers, w 2^S rounded, S = 62 - log2 of the vocabulary's size (48 at most), and sums of them 64-bit
// whole numbers: exact, the same in any order, and comparable with a border that lies next to them. 32-bit sums
// would move the borders by 2^-24 of the total, which is the weight of whole tokens in a wide row.
#include "cdb_common.cuh"

namespace cdb {
namespace sample {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
typedef unsigned long long u64;

struct Params {
  const void* logits;
  int64_t stride;
  int vocab;
  const float* uniform;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* ids;
  float* logp;
  int scale_bits;  // S
};

// Keys that order as the logits do; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  x += 0.f;
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ (key & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kMinusInf = 0x007fffffu;  // key_of(-inf)

template <typename T>
__device__ __forceinline__ uint32_t load_key(const void* row, int i) {
  if constexpr (sizeof(T) == 2) return key_of(bf16_to_f(static_cast<const __nv_bfloat16*>(row)[i]));
  else return key_of(static_cast<const float*>(row)[i]);
}

struct Weigher {
  double top, inv;
  float bits;
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    const double l = (double)logit_of(key);
    const double d = l == top ? 0. : l - top;  // (+inf - +inf)
    if (!(d >= -1e300)) return 0ull;
    return (u64)__double2ll_rn(exp(d * inv) * exp2((double)bits));
  }
};

__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

// The product of a share in [0, 1] and a sum, rounded down.
__device__ __forceinline__ u64 share_of(float share, u64 sum) {
  const double s = fmin(fmax((double)share, 0.), 1.);
  const u64 m = (u64)(s * 9007199254740992.);  // 2^53 s, whole
  return (__umul64hi(m, sum) << 11) | ((m * sum) >> 53);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  __shared__ u64 red[kWarps];
  __shared__ int found;
  const int r = blockIdx.x, tid = threadIdx.x, v = p.vocab;
  const T* row = static_cast<const T*>(p.logits) + (int64_t)r * p.stride;
  uint32_t top = 0;
  for (int i = tid; i < v; i += kThreads) top = max(top, load_key<T>(row, i));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = max(top, (uint32_t)red[i]);
  if (top == kMinusInf) {
    if (tid == 0) {
      p.ids[r] = -1;
      if (p.logp) p.logp[r] = NAN;
    }
    return;
  }
  const float t = p.temperature[r];
  const bool greedy = !(t > 0.f);
  Weigher weigh;
  weigh.top = (double)logit_of(top);
  weigh.inv = greedy ? 0. : 1. / (double)t;
  weigh.bits = (float)p.scale_bits;
  // the border: tokens of keys above `edge` are kept, and the first `ties` at it
  uint32_t edge = 0;
  u64 ties = ~0ull;
  if (greedy) {
    edge = top;
    ties = 1;
  }
  const int k = p.top_k ? p.top_k[r] : 0;
  if (!greedy && k > 0 && k < v) {
    // the largest key that at least k tokens reach
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = edge | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < v; i += kThreads) n += load_key<T>(row, i) >= probe;
      n = block_sum(n, red);
      if (n >= (u64)k) edge = probe;
      else above = n;
    }
    ties = (u64)k - above;
  }
  const float tp = p.top_p ? p.top_p[r] : 1.f;
  if (!greedy && tp < 1.f) {
    u64 total = 0;
    const u64 at_edge = weigh(edge) * (ties == ~0ull ? 0 : ties);
    for (int i = tid; i < v; i += kThreads) {
      const uint32_t key = load_key<T>(row, i);
      if (key > edge) total += weigh(key);
    }
    total = block_sum(total, red) + at_edge;
    const u64 want = share_of(tp, total);  // kept: tokens before which less than p of the weight lies
    uint32_t e = 0;
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = e | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < v; i += kThreads) {
        const uint32_t key = load_key<T>(row, i);
        if (key >= probe && key > edge) n += weigh(key);
      }
      n = block_sum(n, red);
      if (probe <= edge) n += at_edge;
      if (n >= want && n > 0) e = probe;
      else above = n;
    }
    const u64 w = weigh(e);
    const u64 room = want > above ? want - above : 0;
    u64 m = w ? (room + w - 1) / w : 1;
    if (m == 0) m = 1;
    if (e != edge || m < ties) ties = m;
    edge = e;
  }
  const float mp = p.min_p ? p.min_p[r] : 0.f;
  const bool cut = !greedy && mp > 0.f;
  const double floor_w = cut ? fmin((double)mp, 1.) : 0.;
  auto heavy = [&](uint32_t key) {
    const double l = (double)logit_of(key);
    return !cut || key == top || exp((l - weigh.top) * weigh.inv) >= floor_w;
  };
  // index order: each thread a stretch of the row
  const int per = (v + kThreads - 1) / kThreads;
  const int lo = min(v, tid * per), hi = min(v, lo + per);
  auto scan = [&](u64 mine, u64& all) {  // sum of the threads before this one
    u64 x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, x, o);
      if ((tid & 31) >= o) x += y;
    }
    __syncthreads();
    if ((tid & 31) == 31) red[tid >> 5] = x;
    __syncthreads();
    u64 before = x - mine;
    all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < (tid >> 5)) before += red[i];
      all += red[i];
    }
    return before;
  };
  u64 n = 0, all;
  for (int i = lo; i < hi; ++i) n += load_key<T>(row, i) == edge;
  const u64 ties_before = scan(n, all);
  auto walk = [&](auto f) {
    u64 seen = ties_before;
    for (int i = lo; i < hi; ++i) {
      const uint32_t key = load_key<T>(row, i);
      bool keep = key > edge;
      if (key == edge) keep = seen++ < ties;
      if (keep && heavy(key)) f(i, greedy ? 1ull : weigh(key));
    }
  };
  u64 mine = 0;
  walk([&](int, u64 w) { mine += w; });
  u64 run = scan(mine, all);
  if (tid == 0) found = -1;
  __syncthreads();
  u64 want = share_of(p.uniform[r], all);
  if (want >= all) want = all - 1;
  if (run <= want && want < run + mine) {
    walk([&](int i, u64 w) {
      if (run <= want && want < run + w) {
        found = i;
        p.ids[r] = i;
        const double l = (double)logit_of(load_key<T>(row, i)), d = l == weigh.top ? 0. : (l - weigh.top) * weigh.inv;
        if (p.logp) p.logp[r] = greedy ? 0.f : (float)(d - log((double)all) + p.scale_bits * 0.69314718055994530942);
      }
      run += w;
    });
  }
}

}  // namespace sample
}  // namespace cdb

extern "C" int cdb_sample_tokens(const void* logits, int logits_fp32, int64_t logits_stride, int num_rows, int vocab,
                                 const float* uniform, const float* temperature, const int32_t* top_k,
                                 const float* top_p, const float* min_p, int64_t* out_ids, float* out_logprobs,
                                 void* stream) {
  using namespace cdb;
  using namespace cdb::sample;
  if (num_rows < 0 || vocab <= 0 || logits_stride < 0) return CDB_ERR_INVALID_ARGUMENT;
  if (vocab > (1 << 24)) return CDB_ERR_UNSUPPORTED;
  if (num_rows == 0) return CDB_OK;
  if (logits == nullptr || uniform == nullptr || temperature == nullptr || out_ids == nullptr)
    return CDB_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(logits) & (logits_fp32 ? 3 : 1)) return CDB_ERR_INVALID_ARGUMENT;
  Params p;
  p.logits = logits;
  p.stride = logits_stride;
  p.vocab = vocab;
  p.uniform = uniform;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.ids = out_ids;
  p.logp = out_logprobs;
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  p.scale_bits = 62 - bits < 48 ? 62 - bits : 48;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* kernel = logits_fp32 ? sample_kernel<float> : sample_kernel<__nv_bfloat16>;
  return launch_pdl(kernel, dim3(num_rows), dim3(kThreads), 0, st, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}
