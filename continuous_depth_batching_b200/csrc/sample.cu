// The next token of every row from its logits and one given random number.
//
// Row r with temperature t > 0: a token weighs w = exp((l - max l) / t). Tokens are ordered by falling logit,
// equal ones by index. Of them top-k keeps the first k; top-p of those the shortest beginning whose weight reaches
// the share p of theirs; min-p of those the ones with w >= min_p. The token is the least index at which the kept
// weights' running sum passes u times their total. What is kept is therefore a border in the order: all logits
// above one value, and of those equal to it the first few by index.
//
// Weights are whole numbers, w 2^S rounded, S = 62 - log2 of the vocabulary's size (46 at most), and sums of them 64-bit
// whole numbers: exact, the same in any order, and comparable with a border that lies next to them. 32-bit sums
// would move the borders by 2^-24 of the total, which is the weight of whole tokens in a wide row.
//
// A CTA takes a row and reads it up to four times, the first from memory and the others from L2:
//   1. its largest and least logit;
//   2. (top-k, top-p; bf16 always) how many tokens each of 8192 bins has: the upper 16 bits of the logit's 32, so
//      for bf16 a bin holds one value, over the 32 octaves below the row's largest magnitude, either sign;
//   3. the kept weights of every warp's stretch of the row. bf16 looks a bin's weight up. fp32 computes it, and where
//      the border falls into a bin, its neighbourhood's tokens are collected, sorted and summed exactly;
//   4. the stretch in which the target lies, a few tokens to a thread.
// Rows that this does not fit (an infinite largest logit, bf16 logits over more than 32 octaves, a border among more
// fp32 tokens than the list holds) take `slow_row`, which finds its borders by bisection, a bit of the key a pass.
#include "cdb_common.cuh"

namespace cdb {
namespace sample {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kHalf = 4096;              // bins of one sign: 32 octaves of 128
constexpr int kBins = 2 * kHalf + 1;     // largest logits first; bin kHalf holds 0
constexpr int kPerThread = (kBins + kThreads - 1) / kThreads;
constexpr int kBinsPadded = kPerThread * kThreads;
constexpr int kList = 8192;              // fp32 tokens next to a border
constexpr int kNone = kBinsPadded;       // no bin: weighs nothing
constexpr uint32_t kAll = 0xffffffffu;
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
constexpr uint32_t kPlusInf = 0xff800000u;

template <typename T>
__device__ __forceinline__ float load_one(const void* row, int i) {
  if constexpr (sizeof(T) == 2) return bf16_to_f(static_cast<const __nv_bfloat16*>(row)[i]);
  else return static_cast<const float*>(row)[i];
}
template <typename T>
__device__ __forceinline__ uint32_t load_key(const void* row, int i) {
  return key_of(load_one<T>(row, i));
}

// The row as vectors of 16 bytes: vector j holds tokens j * N - shift .. of which those in [0, vocab) count.
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  const T* at;
  int vocab, shift, vectors;
  __device__ __forceinline__ Row(const Params& p, int r) {
    at = static_cast<const T*>(p.logits) + (int64_t)r * p.stride;
    vocab = p.vocab;
    shift = (int)((reinterpret_cast<uintptr_t>(at) & 15) / sizeof(T));
    vectors = (vocab + shift + N - 1) / N;
  }
  // Tokens outside the row come as NaN, which weighs nothing.
  __device__ __forceinline__ void load(int j, float (&x)[N]) const {
    const int i = j * N - shift;
    if (i >= 0 && i + N <= vocab) {
      const uint4 w = *reinterpret_cast<const uint4*>(at + i);
      if constexpr (N == 8) {
        x[0] = bf16lo(w.x), x[1] = bf16hi(w.x), x[2] = bf16lo(w.y), x[3] = bf16hi(w.y);
        x[4] = bf16lo(w.z), x[5] = bf16hi(w.z), x[6] = bf16lo(w.w), x[7] = bf16hi(w.w);
      } else {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = i + k >= 0 && i + k < vocab ? load_one<T>(at, i + k) : NAN;
    }
  }
};

// ---------------------------------------------------------------------------------- sums over the CTA

struct Scratch {
  u64 sum[kWarps];
  u64 sum2[kWarps];
  int found;
};

// Sum of the threads before this one, and of all.
__device__ __forceinline__ u64 scan(u64 mine, u64& all, u64* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(kAll, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  u64 before = x - mine;
  all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += red[i];
    all += red[i];
  }
  return before;
}
__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

// The product of a share in [0, 1] and a sum, rounded down (a running sum passes it where it passes the product) or up
// (one is below it where it is below the product). NaN: 0.
__device__ __forceinline__ u64 share_of(float share, u64 sum, bool up = false) {
  const double s = fmin(fmax((double)share, 0.), 1.);
  const u64 m = (u64)(s * 9007199254740992.);  // 2^53 s, whole
  const u64 low = m * sum;
  return ((__umul64hi(m, sum) << 11) | (low >> 53)) + (up && (low & ((1ull << 53) - 1)) != 0);
}

// ---------------------------------------------------------------------------------- weights

// In 64 bits, for a few tokens or bins.
struct Weigher {
  double top, inv, one;  // one: 2^S
  __device__ __forceinline__ double share(float l) const {
    const double d = (double)l == top ? 0. : (double)l - top;  // (+inf - +inf)
    return d >= -1e300 ? exp(d * inv) : 0.;
  }
  __device__ __forceinline__ u64 operator()(float l) const { return (u64)__double2ll_rn(share(l) * one); }
};

// The same to 2^-30 of each weight from 32-bit operations, for every token of a row. With y = (top - l) log2(e) / t as a
// sum of two floats: 2^-y = 2^-n 2^-(j / 256) 2^-r, the second from a table, the third from its series, |r| <= 2^-9.
struct FastWeigher {
  float top, c, c_low;  // log2(e) / t in two floats
  int bits;             // S - 31
  const uint2* table;   // {2^31 2^-(j / 256) whole, as a float}
  __device__ __forceinline__ u64 operator()(float l) const {
    const float d = top - l;
    // what the subtraction rounded away
    const float back = d - top;
    const float low = (top - (d - back)) - (l + back);
    const float y = __fmul_rn(d, c);
    if (!(y < 62.f)) return d == 0.f ? 1ull << (bits + 31) : 0ull;  // (also NaN: 0 / a tiny temperature, -inf)
    const float e = fmaf(low, c, fmaf(d, c_low, fmaf(d, c, -y)));
    const float round = y + 49152.f;  // to whole 1 / 256
    const int step = __float_as_int(round) - __float_as_int(49152.f);
    const float r = ((y - (round - 49152.f)) + e) * 0.693147180559945f;
    const float q = r * fmaf(r, fmaf(r, 0.16666667f, -0.5f), 1.f);  // 1 - 2^-r
    const uint2 t = table[step & 255];
    const float less = fmaf(__uint_as_float(t.y), q, 12582912.f);  // + 1.5 * 2^23: its low bits are the whole number
    const uint32_t m = t.x - (uint32_t)(__float_as_int(less) - __float_as_int(12582912.f));
    return ((u64)m << bits) >> (step >> 8);
  }
};

// ---------------------------------------------------------------------------------- any row, slowly

template <typename T>
__device__ __noinline__ void slow_row(const Params& p, int r, uint32_t top, float t, Scratch& sc) {
  const int tid = threadIdx.x, v = p.vocab;
  const void* row = static_cast<const T*>(p.logits) + (int64_t)r * p.stride;
  const bool greedy = !(t > 0.f);
  Weigher weigh;
  weigh.top = (double)logit_of(top);
  weigh.inv = greedy ? 0. : 1. / (double)t;
  weigh.one = (double)(1ull << p.scale_bits);
  // tokens of keys above `edge` are kept, and the first `ties` at it
  uint32_t edge = greedy ? top : 0;
  u64 ties = greedy ? 1 : ~0ull;
  const int k = p.top_k ? p.top_k[r] : 0;
  if (!greedy && k > 0 && k < v) {
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {  // the largest key that at least k tokens reach
      const uint32_t probe = edge | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < v; i += kThreads) n += load_key<T>(row, i) >= probe;
      n = block_sum(n, sc.sum);
      if (n >= (u64)k) edge = probe;
      else above = n;
    }
    ties = (u64)k - above;
  }
  const float tp = p.top_p ? p.top_p[r] : 1.f;
  if (!greedy && tp < 1.f) {
    const u64 at_edge = ties == ~0ull ? 0 : weigh(logit_of(edge)) * ties;
    u64 total = 0;
    for (int i = tid; i < v; i += kThreads) {
      const uint32_t key = load_key<T>(row, i);
      if (key > edge) total += weigh(logit_of(key));
    }
    total = block_sum(total, sc.sum) + at_edge;
    const u64 want = share_of(tp, total, true);
    uint32_t e = 0;
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = e | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < v; i += kThreads) {
        const uint32_t key = load_key<T>(row, i);
        if (key >= probe && key > edge) n += weigh(logit_of(key));
      }
      n = block_sum(n, sc.sum);
      if (probe <= edge) n += at_edge;
      if (n >= want && n > 0) e = probe;
      else above = n;
    }
    const u64 w = weigh(logit_of(e));
    const u64 room = want > above ? want - above : 0;
    u64 m = w ? (room + w - 1) / w : 1;
    if (m == 0) m = 1;
    if (e != edge || m < ties) ties = m;
    edge = e;
  }
  const float mp = p.min_p ? p.min_p[r] : 0.f;
  const bool cut = !greedy && mp > 0.f;
  const double least = cut ? fmin((double)mp, 1.) : 0.;
  // index order: each thread a stretch of the row
  const int per = (v + kThreads - 1) / kThreads;
  const int lo = min(v, tid * per), hi = min(v, lo + per);
  u64 n = 0, all;
  for (int i = lo; i < hi; ++i) n += load_key<T>(row, i) == edge;
  const u64 ties_before = scan(n, all, sc.sum);
  auto walk = [&](auto f) {
    u64 seen = ties_before;
    for (int i = lo; i < hi; ++i) {
      const uint32_t key = load_key<T>(row, i);
      bool keep = key > edge;
      if (key == edge) keep = seen++ < ties;
      if (keep && (!cut || key == top || weigh.share(logit_of(key)) >= least)) f(i, greedy ? 1ull : weigh(logit_of(key)));
    }
  };
  u64 mine = 0;
  walk([&](int, u64 w) { mine += w; });
  u64 run = scan(mine, all, sc.sum);
  u64 want = share_of(p.uniform[r], all);
  if (want >= all) want = all - 1;
  if (run <= want && want < run + mine) {
    walk([&](int i, u64 w) {
      if (run <= want && want < run + w) {
        p.ids[r] = i;
        const double l = (double)load_one<T>(row, i), d = l == weigh.top ? 0. : (l - weigh.top) * weigh.inv;
        if (p.logp) p.logp[r] = greedy ? 0.f : (float)(d - log((double)all / weigh.one));
      }
      run += w;
    });
  }
}

// ---------------------------------------------------------------------------------- bins

// `low`: (least biased exponent of the bins' 32 octaves) * 128, at least 0.
// Logits of smaller magnitude share 0's bin (bf16 rows that have such go the slow way), larger ones have none.
__device__ __forceinline__ int bin_of(float x, int low) {
  const uint32_t b = __float_as_uint(x);
  const int mag = (int)((b >> 16) & 0x7fffu);
  const int off = max(mag - low + 1, 0) * (mag != 0);
  const int bin = (int32_t)b < 0 ? kHalf + off : kHalf - off;
  return x == x && off <= kHalf ? bin : kNone;
}
// The least magnitude of a bin's logits, signed.
__device__ __forceinline__ float logit_of_bin(int bin, int low) {
  if (bin == kHalf) return 0.f;
  const int off = bin < kHalf ? kHalf - bin : bin - kHalf;
  const uint32_t mag = (uint32_t)(off - 1 + low) << 16;
  return __uint_as_float(bin < kHalf ? mag : mag | 0x80000000u);
}

struct Shared {
  Scratch sc;
  uint32_t red[2 * kWarps];
  uint2 table[256];
  int edge_bin, edge_count;  // the border: of that bin's tokens the first few are kept
  int lo_bin, hi_bin;        // fp32: the bins whose tokens are collected
  int list_n, list_over;
  int k_border;              // fp32: top-k ends among the binned tokens
  u64 edge;                  // fp32: the last token kept, as the list has it
  u64 above;
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
  constexpr bool WIDE = sizeof(T) == 4;
  constexpr int N = Row<T>::N;
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* counts = reinterpret_cast<uint32_t*>(smem);                        // [kBinsPadded + 1]
  u64* weights = reinterpret_cast<u64*>(smem + (kBinsPadded + 4) * 4);         // bf16: [kBinsPadded + 1]
  u64* list = weights;                                                         // fp32: [kList] {key, ~index}
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x;
  for (int i = tid; i < (kBinsPadded + 4) / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
  if (WIDE && tid < 256) {
    const double x = 2147483648. * exp2(-(double)tid / 256.);
    sh.table[tid] = make_uint2((uint32_t)__double2ll_rn(x), __float_as_uint((float)x));
  }
  pdl_wait();
  const Row<T> row(p, r);
  const float t = p.temperature[r];
  const bool greedy = !(t > 0.f);

  // ---- the largest logit, and the least above -inf
  uint32_t top = 0, least = kAll;
#pragma unroll 4
  for (int j = tid; j < row.vectors; j += kThreads) {
    float x[N];
    row.load(j, x);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t key = key_of(x[k]);
      top = max(top, key);
      if (key > kMinusInf) least = min(least, key);
    }
  }
  top = __reduce_max_sync(kAll, top);
  least = __reduce_min_sync(kAll, least);
  if (lane == 0) sh.red[warp] = top, sh.red[kWarps + warp] = least;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    top = max(top, sh.red[i]);
    least = min(least, sh.red[kWarps + i]);
  }
  if (top <= kMinusInf) {
    if (tid == 0) {
      p.ids[r] = -1;
      if (p.logp) p.logp[r] = NAN;
    }
    return;
  }
  if (greedy) {
    int first = INT32_MAX;
    for (int j = tid; j < row.vectors; j += kThreads) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int k = N - 1; k >= 0; --k)
        if (key_of(x[k]) == top) first = min(first, j * N - row.shift + k);
    }
    first = __reduce_min_sync(kAll, first);
    __syncthreads();
    if (lane == 0) sh.red[warp] = (uint32_t)first;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int i = 1; i < kWarps; ++i) first = min(first, (int)sh.red[i]);
      p.ids[r] = first;
      if (p.logp) p.logp[r] = 0.f;
    }
    return;
  }
  if (top == kPlusInf) {
    slow_row<T>(p, r, top, t, sh.sc);
    return;
  }
  const int k = p.top_k ? p.top_k[r] : 0;
  const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < p.vocab, by_p = tp < 1.f, by_m = mp > 0.f;
  Weigher weigh;
  weigh.top = (double)logit_of(top);
  weigh.inv = 1. / (double)t;
  weigh.one = (double)(1ull << p.scale_bits);
  // below this no weight is left
  const double cutoff = weigh.top - (double)t * 0.6931471805599453 * (p.scale_bits + 2);
  const float lowest = fmaxf(logit_of(least), (float)fmax(cutoff, -3.4e38));
  const float widest = fmaxf(fabsf(logit_of(top)), fabsf(lowest));
  const int low = max((int)(__float_as_uint(widest) >> 23) - 31, 0) * 128;
  const bool bins = !WIDE || by_k || by_p;

  // ---- bins
  if (bins) {
    bool strange = false;
#pragma unroll 2
    for (int j = tid; j < row.vectors; j += kThreads) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of(x[i], low);
        if (!WIDE) strange |= bin == kHalf && x[i] != 0.f;
        if (bin != kNone) atomicAdd(&counts[bin], 1u);
      }
    }
    if (__syncthreads_or(strange)) {
      slow_row<T>(p, r, top, t, sh.sc);
      return;
    }
    // Each thread a few neighbouring bins, largest logits first.
    const int b0 = tid * kPerThread;
    uint32_t n[kPerThread];
    u64 w[kPerThread], mine_n = 0, mine_w = 0, all_n, all_w;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      n[i] = counts[b0 + i];
      mine_n += n[i];
      w[i] = 0;
    }
    u64 before = scan(mine_n, all_n, sh.sc.sum);
    // tokens of each bin that top-k leaves; fp32 takes the middle of a bin for all of its tokens
    if (tid == 0) sh.edge_bin = kNone, sh.edge_count = 0, sh.lo_bin = kBinsPadded, sh.hi_bin = -1, sh.list_n = 0, sh.list_over = 0, sh.k_border = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const uint32_t had = n[i];
      if (by_k) {
        n[i] = before >= (u64)k ? 0u : (uint32_t)min((u64)n[i], (u64)k - before);
        if ((n[i] < had && n[i] > 0) || (before + had == (u64)k && had > 0)) {
          if (!WIDE) sh.edge_bin = b0 + i, sh.edge_count = (int)n[i];
          else atomicMin(&sh.lo_bin, b0 + i), atomicMax(&sh.hi_bin, b0 + i), sh.k_border = 1;
        }
      }
      before += had;
      if (n[i] > 0) {
        float l = logit_of_bin(b0 + i, low);
        if (WIDE) {
          const float next = b0 + i < kHalf ? logit_of_bin(b0 + i - 1, low) : logit_of_bin(b0 + i + 1, low);
          l = b0 + i == kHalf ? 0.f : fminf(0.5f * l + 0.5f * next, logit_of(top));
        }
        w[i] = weigh(l);
        mine_w += w[i] * n[i];
      }
    }
    if (by_p || !WIDE) {
      u64 mass = scan(mine_w, all_w, sh.sc.sum);
      const u64 want = by_p ? share_of(tp, all_w, true) : ~0ull;
      // fp32: the border is somewhere within 2^-8 of the total (checked later); 2^-12 where bins are narrow would do
      const u64 slack = WIDE ? (all_w >> 8) + 1 : 0;
      const u64 want_lo = want > slack ? want - slack : 0, want_hi = want + slack;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        if (n[i] == 0) continue;
        const u64 here = w[i] * n[i];
        if (by_p && !WIDE) {
          const uint32_t had = n[i];
          if (mass >= want) n[i] = 0;
          else if (w[i] > 0 && mass + here >= want) n[i] = (uint32_t)min((u64)had, (want - mass + w[i] - 1) / w[i]);
          if (mass == 0 && n[i] == 0) n[i] = 1;  // the first token always stays
          if (n[i] > 0 && (n[i] < had || mass + here >= want)) sh.edge_bin = b0 + i, sh.edge_count = (int)n[i];
        } else if (by_p) {
          // bins that the border may fall into
          if (mass <= want_hi && mass + here >= want_lo) atomicMin(&sh.lo_bin, b0 + i), atomicMax(&sh.hi_bin, b0 + i);
        }
        mass += here;
      }
    }
    __syncthreads();
    if (!WIDE) {
      const float floor_w = by_m ? fminf(mp, 1.f) : 0.f;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        bool keep = n[i] > 0;
        if (by_m && keep) {
          const float l = logit_of_bin(b0 + i, low);
          keep = l == logit_of(top) || weigh.share(l) >= (double)floor_w;
        }
        // the border's bin is counted token by token
        weights[b0 + i] = keep && b0 + i != sh.edge_bin ? w[i] : 0;
        if (b0 + i == sh.edge_bin) sh.above = keep ? w[i] : 0;
      }
      if (tid == 0) weights[kNone] = 0;
      __syncthreads();
    }
  }

  // ---- kept weights of every warp's stretch
  const int per_warp = (row.vectors + kWarps - 1) / kWarps;
  const int v0 = min(row.vectors, warp * per_warp), v1 = min(row.vectors, v0 + per_warp);
  if constexpr (!WIDE) {
    const int edge = sh.edge_bin;
    const u64 edge_w = edge == kNone ? 0 : sh.above;
    const u64 edge_n = (u64)sh.edge_count;
    u64 sum = 0;
    uint32_t ties = 0;
#pragma unroll 2
    for (int j = v0 + lane; j < v1; j += 32) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of(x[i], low);
        sum += weights[bin];
        ties += bin == edge;
      }
    }
    if (edge == kNone) ties = 0;
    ties = __reduce_add_sync(kAll, ties);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    if (lane == 0) sh.sc.sum[warp] = sum, sh.sc.sum2[warp] = ties;
    __syncthreads();
    // stretch by stretch: ties before it, and the weight with those that stay
    u64 run = 0, seen = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 stay = seen >= edge_n ? 0 : min(sh.sc.sum2[i], edge_n - seen);
      seen += sh.sc.sum2[i];
      all += sh.sc.sum[i] + stay * edge_w;
    }
    u64 want = share_of(p.uniform[r], all);
    if (want >= all) want = all - 1;
    seen = 0;
    int in = 0;
    u64 run_in = 0, seen_in = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 stay = seen >= edge_n ? 0 : min(sh.sc.sum2[i], edge_n - seen);
      const u64 here = sh.sc.sum[i] + stay * edge_w;
      if (run <= want && want < run + here) in = i, run_in = run, seen_in = seen;
      seen += sh.sc.sum2[i];
      run += here;
    }
    __syncthreads();
    // ---- the stretch with the target, a vector or a few to a thread
    const int s0 = min(row.vectors, in * per_warp), s1 = min(row.vectors, s0 + per_warp);
    const int per = (s1 - s0 + kThreads - 1) / kThreads;
    const int j0 = min(s1, s0 + tid * per), j1 = min(s1, j0 + per);
    u64 mine = 0, mine_ties = 0, dummy;
    for (int j = j0; j < j1; ++j) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of(x[i], low);
        mine += weights[bin];
        mine_ties += bin == edge && edge != kNone;
      }
    }
    u64 my_seen = seen_in + scan(mine_ties, dummy, sh.sc.sum);
    const u64 my_stay = my_seen >= edge_n ? 0 : min(mine_ties, edge_n - my_seen);
    mine += my_stay * edge_w;
    u64 my_run = run_in + scan(mine, dummy, sh.sc.sum);
    if (my_run <= want && want < my_run + mine) {
      for (int j = j0; j < j1; ++j) {
        float x[N];
        row.load(j, x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int bin = bin_of(x[i], low);
          u64 w = weights[bin];
          if (bin == edge && edge != kNone && my_seen++ < edge_n) w = edge_w;
          if (my_run <= want && want < my_run + w) {
            p.ids[r] = j * N - row.shift + i;
            if (p.logp) p.logp[r] = (float)(((double)x[i] - weigh.top) * weigh.inv - log((double)all / weigh.one));
          }
          my_run += w;
        }
      }
    }
  } else {
    FastWeigher fast;
    {
      const double c = 1.4426950408889634 / (double)t;
      fast.top = logit_of(top);
      fast.c = (float)c;
      fast.c_low = isinf(fast.c) ? 0.f : (float)(c - (double)fast.c);
      fast.bits = p.scale_bits - 31;
      fast.table = sh.table;
    }
    const u64 least_w = by_m ? (u64)(fmin((double)mp, 1.) * weigh.one) : 0;
    auto heavy = [&](u64 w, float l) { return !by_m || w >= least_w || l == fast.top; };
    const bool edged = bins && sh.hi_bin >= 0;  // (top-k of more tokens than weigh anything leaves all)
    const int lo = edged ? sh.lo_bin : kNone, hi = edged ? sh.hi_bin : kNone;
    const bool all_rest = by_p && !sh.k_border;  // the total that top-p takes a share of goes on below the list
    u64 sum = 0, rest = 0, all_above = 0;
    uint32_t above_n = 0;
#pragma unroll 2
    for (int j = v0 + lane; j < v1; j += 32) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!edged) {
          const u64 w = fast(x[i]);
          if (heavy(w, x[i])) sum += w;
        } else {
          const int bin = bin_of(x[i], low);
          if (bin < lo) {
            const u64 w = fast(x[i]);
            ++above_n;
            all_above += w;
            if (heavy(w, x[i])) sum += w;
          } else if (bin <= hi) {
            const int at = atomicAdd(&sh.list_n, 1);
            if (at < kList) list[at] = (u64)key_of(x[i]) << 32 | (uint32_t)~(j * N - row.shift + i);
          } else if (all_rest) {
            rest += fast(x[i]);
          }
        }
      }
    }
    u64 edge = 0;  // tokens at or above it (key, then lower indexes) are kept
    if (edged) {
      const u64 above_w = block_sum(all_above, sh.sc.sum), rest_w = block_sum(rest, sh.sc.sum);
      const u64 n_above = block_sum(above_n, sh.sc.sum);
      const int n = sh.list_n;
      if (n > kList) {
        slow_row<T>(p, r, top, t, sh.sc);
        return;
      }
      // sort the list, largest first
      int size = 32;
      while (size < n) size <<= 1;
      for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
      __syncthreads();
      for (int run = 2; run <= size; run <<= 1)
        for (int step = run >> 1; step > 0; step >>= 1) {
          for (int i = tid; i < size / 2; i += kThreads) {
            const int a = 2 * i - (i & (step - 1)), b = a + step;
            const u64 x = list[a], y = list[b];
            if ((x < y) == ((a & run) == 0)) list[a] = y, list[b] = x;
          }
          __syncthreads();
        }
      // their weights, and what top-k, then top-p leaves of them
      const int per = (size + kThreads - 1) / kThreads, i0 = min(size, tid * per), i1 = min(size, i0 + per);
      const u64 left_k = by_k ? ((u64)k > n_above ? (u64)k - n_above : 0) : ~0ull;
      u64 mine = 0, all_w;
      for (int i = i0; i < i1; ++i)
        if (i < n && (u64)i < left_k) mine += fast(logit_of((uint32_t)(list[i] >> 32)));
      u64 mass = above_w + scan(mine, all_w, sh.sc.sum);
      const u64 total = above_w + all_w + rest_w;
      const u64 want = by_p ? share_of(tp, total, true) : ~0ull;
      if (tid == 0) sh.edge = 0, sh.list_over = 0;
      __syncthreads();
      // The last token kept; the first of all always is. A top-p border outside the list is a slow row.
      for (int i = i0; i < i1; ++i) {
        if (i >= n || (u64)i >= left_k) break;
        const u64 w = fast(logit_of((uint32_t)(list[i] >> 32)));
        const bool first = n_above == 0 && i == 0;
        if (mass < want || first) {
          const bool last = (u64)i + 1 >= left_k || (by_p && mass + w >= want);
          if (last || i + 1 == n) sh.edge = list[i];
          if (!last && i + 1 == n && by_p && rest_w > 0) sh.list_over = 1;  // the border lies below the list
        }
        mass += w;
      }
      if (by_p && tid == 0 && above_w >= want && n_above > 0) sh.list_over = 1;  // or above it
      __syncthreads();
      edge = sh.edge;
      if (sh.list_over || edge == 0) {
        slow_row<T>(p, r, top, t, sh.sc);
        return;
      }
    }
    auto kept = [&](float l, int i, u64& w) {
      w = 0;
      if (!(l > -INFINITY)) return;
      if (edged && ((u64)key_of(l) << 32 | (uint32_t)~i) < edge) return;
      w = fast(l);
      if (!heavy(w, l)) w = 0;
    };
    // the list's kept tokens belong to their stretches
    if (lane == 0) sh.sc.sum2[warp] = 0;
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    if (edged) {
      for (int i = tid; i < sh.list_n; i += kThreads) {
        if (list[i] < edge) continue;
        const int index = (int)~(uint32_t)list[i];
        u64 w;
        kept(logit_of((uint32_t)(list[i] >> 32)), index, w);
        if (w) atomicAdd(&sh.sc.sum2[(index + row.shift) / N / per_warp], w);
      }
    }
    if (lane == 0) sh.sc.sum[warp] = sum;
    __syncthreads();
    u64 all = 0, run = 0, run_in = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) all += sh.sc.sum[i] + sh.sc.sum2[i];
    u64 want = share_of(p.uniform[r], all);
    if (want >= all) want = all - 1;
    int in = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 here = sh.sc.sum[i] + sh.sc.sum2[i];
      if (run <= want && want < run + here) in = i, run_in = run;
      run += here;
    }
    __syncthreads();
    // ---- the stretch with the target, a vector or a few to a thread
    const int s0 = min(row.vectors, in * per_warp), s1 = min(row.vectors, s0 + per_warp);
    const int per = (s1 - s0 + kThreads - 1) / kThreads;
    const int j0 = min(s1, s0 + tid * per), j1 = min(s1, j0 + per);
    u64 mine = 0, dummy;
    for (int j = j0; j < j1; ++j) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u64 w;
        kept(x[i], j * N - row.shift + i, w);
        mine += w;
      }
    }
    u64 my_run = run_in + scan(mine, dummy, sh.sc.sum);
    if (my_run <= want && want < my_run + mine) {
      for (int j = j0; j < j1; ++j) {
        float x[N];
        row.load(j, x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          u64 w;
          kept(x[i], j * N - row.shift + i, w);
          if (my_run <= want && want < my_run + w) {
            p.ids[r] = j * N - row.shift + i;
            if (p.logp) p.logp[r] = (float)(((double)x[i] - weigh.top) * weigh.inv - log((double)all / weigh.one));
          }
          my_run += w;
        }
      }
    }
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
  p.scale_bits = 62 - bits < 46 ? 62 - bits : 46;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int smem = (kBinsPadded + 4) * 4 + (logits_fp32 ? kList : kBinsPadded + 1) * 8;
  auto* kernel = logits_fp32 ? sample_kernel<float> : sample_kernel<__nv_bfloat16>;
  if (allow_shared(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess) return CDB_ERR_CUDA;
  return launch_pdl(kernel, dim3(num_rows), dim3(kThreads), smem, st, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}
