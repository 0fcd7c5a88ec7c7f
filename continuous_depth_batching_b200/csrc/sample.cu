// The next token of every row from its logits and one given random number.
//
// Row r with temperature t > 0: a token weighs w = exp((l - max l) / t). Tokens are ordered by falling logit,
// equal ones by index. Of them top-k keeps the first k; top-p of those the shortest beginning whose weight reaches
// the share p of theirs; min-p of those the ones with w >= min_p. The token is the least index at which the kept
// weights' running sum passes u times their total. What is kept is therefore a border in the order: all logits
// above one value, and of those equal to it the first few by index.
//
// Weights are whole numbers, w 2^S rounded down, S = 62 - log2 of the vocabulary's size (46 at most), and sums of them 64-bit
// whole numbers: exact, the same in any order, and comparable with a border that lies next to them. 32-bit sums
// would move the borders by 2^-24 of the total, which is the weight of whole tokens in a wide row.
//
// A CTA takes a row and reads it a few times, the first from memory and the others from L2:
//   1. its largest and least logit, and every thread's largest;
//   2. with top-k of up to half the threads: the tokens at or above the k-th largest of the threads' largest, a few more
//      than k of them, which are sorted; the rest is done on them;
//   2. with top-p, or more of top-k: how many tokens each of 8192 bins has (fp32: 4096): the upper 16 bits of the logit's 32,
//      so for bf16 a bin holds one value, over the 32 (16) octaves below the row's largest magnitude, either sign;
//   3. the kept weights of every warp's stretch of the row. Behind bins bf16 looks a bin's weight up; fp32 computes it, and
//      where the border falls into a bin, its neighbourhood's tokens are collected, sorted and summed exactly;
//   4. the stretch in which the target lies, a few tokens to a thread.
// Rows that this does not fit (an infinite largest logit, bf16 logits over more than 32 octaves, a border among more
// fp32 tokens than the list holds) take `slow_row`, which finds its borders by bisection, a bit of the key a pass: 0.25 to
// 0.6 ms at 49152 tokens (all logits equal; a border in bf16 where some logit is 2^-32 of another). With fp32 and top-p the
// list holds what lies within 2^-11 of the total about the border, and five deviations of what the bins leave open, so near
// p = 1 it is a wide row's whole tail: rows of a language model's shape take the slow way from p = 0.998 on at 49152 tokens
// and temperature 0.7, or 0.995 at 151936 (256 rows: 0.13 ms at p = 0.995 and 1.1 at 0.998; 0.32 at 0.99 and 3.2 to 4.5 above).
//
// What bounds it: instructions, and for a few rows a chain of passes with a barrier or a scan after each. A weight is some
// 30 instructions, so 256 rows of 65536 plain take 35 us (5 of HBM; 0.58 instructions a cycle and scheduler); counting
// into bins 12 cycles a warp of tokens (shared atomics on 32 banks, most of the 18 us of that pass), so 256 fp32 rows of
// 49152 with top-p take 81 us. Their median row takes 62: 2 to begin, 10 the largest (memory), 18 bins, 6 their weights and
// sums, 18 the weights above and below the border, 5 its list, 3 the token; the last rows' lists of thousands take up to 25.
// One row with top-k of 50: 12 us, in steps of 1 to 2. With 32 octaves of bins
// for fp32, and every token's bin for its sums, those 81 us were 95; one CTA an SM for 256 rows is slower than two of 512 threads.
#include "cdb_common.cuh"

namespace cdb {
namespace sample {

constexpr int kMaxWarps = 32;
// Bins, 128 to an octave, largest logits first. fp32 does with 16 octaves: what is smaller is next to 0 and all but equal.
template <typename T>
struct Bins {
  static constexpr int kHalf = sizeof(T) == 4 ? 2048 : 4096;  // of one sign; bin kHalf holds 0
  static constexpr int kBins = 2 * kHalf + 1;
  static constexpr int kNone = kBins;  // no bin: weighs nothing
  template <int kThreads>
  static constexpr int kPadded = (kBins + kThreads) / kThreads * kThreads;  // and room for kNone
};
constexpr int kList = 8192;  // fp32 tokens next to a border
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
  // The vectors that lie in the row whole are [full0, full1); of one at either end `edge` gives a thread its own, or -1.
  __device__ __forceinline__ int full0() const { return shift != 0; }
  __device__ __forceinline__ int full1() const { return (vocab + shift) / N; }
  __device__ __forceinline__ int edge() const {
    const int at = threadIdx.x == 0 ? (shift ? 0 : -1) : threadIdx.x == 1 ? full1() : -1;
    return threadIdx.x == 1 && (at == vectors || at < full0()) ? -1 : at;
  }
  __device__ __forceinline__ uint4 whole(int j) const { return *reinterpret_cast<const uint4*>(at + (j * N - shift)); }
  // Largest, and least, of a whole vector.
  __device__ __forceinline__ static float largest(const uint4& w) {
    if constexpr (N == 8) {  // two at a time
      const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&w);
      const __nv_bfloat162 a = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
      return fmaxf(__low2float(a), __high2float(a));
    } else {
      return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
  }
  __device__ __forceinline__ static float least(const uint4& w) {
    if constexpr (N == 8) {
      const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&w);
      const __nv_bfloat162 a = __hmin2(__hmin2(v[0], v[1]), __hmin2(v[2], v[3]));
      return fminf(__low2float(a), __high2float(a));
    } else {
      return fminf(fminf(__uint_as_float(w.x), __uint_as_float(w.y)), fminf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
  }
  // f(token, logit) for every token of a vector.
  template <typename F>
  __device__ __forceinline__ void each(int j, F f) const {
#pragma unroll 1
    for (int i = max(j * N - shift, 0); i < min(j * N - shift + N, vocab); ++i) f(i, load_one<T>(at, i));
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
  u64 sum[kMaxWarps];
  u64 sum2[kMaxWarps];
  u64 sum3[kMaxWarps];
};

// Sum of the threads before this one, and of all.
template <int kThreads>
__device__ __forceinline__ u64 scan(u64 mine, u64& all, u64* red) {
  constexpr int kWarps = kThreads / 32;
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
  u64 w = lane < kWarps ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const u64 y = __shfl_up_sync(kAll, w, o);
    if (lane >= o) w += y;
  }
  all = __shfl_sync(kAll, w, kWarps - 1);
  const u64 before = __shfl_sync(kAll, w, (warp + 31) & 31);
  return (warp ? before : 0) + x - mine;
}
// Sums of three numbers over the CTA, to all threads.
template <int kThreads>
__device__ __forceinline__ void block_sums(u64& a, u64& b, u64& c, Scratch& sc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto over_warp = [&] {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(kAll, a, o);
      b += __shfl_xor_sync(kAll, b, o);
      c += __shfl_xor_sync(kAll, c, o);
    }
  };
  over_warp();
  __syncthreads();
  if (lane == 0) sc.sum[warp] = a, sc.sum2[warp] = b, sc.sum3[warp] = c;
  __syncthreads();
  const bool in = lane < kThreads / 32;
  a = in ? sc.sum[lane] : 0, b = in ? sc.sum2[lane] : 0, c = in ? sc.sum3[lane] : 0;
  over_warp();
}
template <int kThreads>
__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  u64 t = lane < kThreads / 32 ? red[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kAll, t, o);
  return t;
}

// The product of a share in [0, 1] and a sum, rounded down (a running sum passes it where it passes the product) or up
// (one is below it where it is below the product). NaN: 0. In whole numbers: 64-bit floating point takes longer here.
__device__ __forceinline__ u64 share_of(float share, u64 sum, bool up = false) {
  if (!(share > 0.f)) return 0;
  if (share >= 1.f) return sum;
  const uint32_t b = __float_as_uint(share);
  const u64 m = (b & 0x7fffffu) | (b >> 23 ? 0x800000u : 0u);
  const int s = 150 - max((int)(b >> 23), 1);  // share = m 2^-s, s > 23
  const u64 high = __umul64hi(m, sum), low = m * sum;
  u64 whole, cut;
  if (s < 64) whole = (high << (64 - s)) | (low >> s), cut = low << (64 - s);
  else whole = s < 128 ? high >> (s - 64) : 0, cut = low | (s < 128 ? s > 64 ? high << (128 - s) : 0 : high);
  return whole + (up && cut != 0);
}

// Sum of the lanes before this one.
__device__ __forceinline__ u64 lane_scan(u64 mine) {
  const int lane = threadIdx.x & 31;
  u64 x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(kAll, x, o);
    if (lane >= o) x += y;
  }
  return x - mine;
}
// Of stretches, one to a lane, the one in which the target lies.
struct Stretch {
  int at;
  u64 before, all, target;
};
__device__ __forceinline__ Stretch stretch_of(u64 mine, float share) {
  const u64 before = lane_scan(mine);
  Stretch s;
  s.all = __shfl_sync(kAll, before + mine, 31);
  s.target = share_of(share, s.all);
  if (s.target >= s.all) s.target = s.all - 1;
  s.at = __ffs(__ballot_sync(kAll, before <= s.target && s.target < before + mine)) - 1;
  s.before = __shfl_sync(kAll, before, s.at);
  return s;
}

// ---------------------------------------------------------------------------------- weights

// In 64 bits, for rows whose largest logit is infinite or whose temperature has no finite inverse in 32.
struct Weigher {
  double top, inv, one;  // one: 2^S
  __device__ __forceinline__ u64 operator()(float l) const {
    const double d = (double)l == top ? 0. : (double)l - top;  // (+inf - +inf)
    return d >= -1e300 ? (u64)(exp(d * inv) * one) : 0;
  }
};

// The same to 2^-30 of each weight from 32-bit operations, for every token of all other rows, whichever way they take: two
// ways with weights of their own would answer differently as the number of rows chooses between them. With y = (top - l) log2(e) / t as a
// sum of two floats: 2^-y = 2^-n 2^-(j / 1024) 2^-r, the second from a table, the third from its series, |r| <= 2^-11.
// What top - l rounds away belongs to that sum, of bf16 logits too: they lie up to 2^8 octaves apart, and past 2^15 their
// difference needs more than 24 bits. (Left out for them, 60000 tokens next to 0 under one at 12 were off by 2^-21 each.
// 256 plain rows of 65536 take 35.3 us with it and 31.1 without; only where a vector holds a logit next to 0, 34.7.)
constexpr int kTable = 1024;
struct Powers {
  uint2 at[kTable];
};
// 2^-(j / 1024) by products of 2^-(1 / 1024) in 64 bits: off by 2^-43 at most.
constexpr uint32_t float_bits(uint32_t whole) {  // of a whole number in [2^30, 2^31], rounded down
  return whole >= 0x80000000u ? 0x4f000000u : (0x4e800000u + ((whole - 0x40000000u) >> 7));
}
constexpr Powers powers() {
  Powers p{};
  double x = 2147483648.;
  for (int j = 0; j < kTable; ++j, x *= 0.99932332750265075) {
    p.at[j].x = (uint32_t)(x + 0.5);
    p.at[j].y = float_bits(p.at[j].x);
  }
  return p;
}
__device__ const Powers g_powers = powers();

struct FastWeigher {
  float top, c, c_low;  // log2(e) / t in two floats
  int down;             // 63 - S
  const uint2* table;   // {2^31 2^-(j / 1024) whole, as a float}
  __device__ __forceinline__ u64 operator()(float l) const {
    const float d = top - l;
    const float y = fminf(__fmul_rn(d, c), 63.f);  // (NaN comes as 63 too, and 2^-63 as 0 below)
    float e = fmaf(d, c_low, fmaf(d, c, -y));
    const float back = d - top;  // what the subtraction rounded away
    e = fmaf((top - (d - back)) - (l + back), c, e);
    const float round = y + 12288.f;  // to whole 1 / 1024
    const int step = __float_as_int(round) - __float_as_int(12288.f);
    const float r = (y - (round - 12288.f)) + e;
    const float q = r * fmaf(r, -0.240226507f, 0.693147181f);  // 1 - 2^-r
    const uint2 t = table[step & (kTable - 1)];
    const float less = fmaf(__uint_as_float(t.y), q, 12582912.f);  // + 1.5 * 2^23: its low bits are the whole number
    const uint32_t m = t.x - (uint32_t)(__float_as_int(less) - __float_as_int(12582912.f));
    u64 w;
    asm("shr.u64 %0, %1, %2;" : "=l"(w) : "l"((u64)m << 32), "r"(down + (step >> 10)));
    return w;
  }
};

// Sorts `size` (a power of two, at least 64) numbers, largest first; only zeros may stand more than once. Few of them
// by counting for each the larger ones, 4 threads or more to each (64: 0.3 us, where the steps below take 3).
template <int kThreads>
__device__ __forceinline__ void sort(u64* list, int size) {
  if (size * 2 <= kThreads) {
    const int parts = min(32, kThreads / size), at = threadIdx.x / parts, part = threadIdx.x % parts;
    const u64 mine = at < size ? list[at] : 0;
    int larger = 0;
    if (at < size) {
#pragma unroll 8
      for (int i = part; i < size; i += parts) larger += list[i] > mine;
    }
    for (int o = parts / 2; o > 0; o >>= 1) larger += __shfl_xor_sync(kAll, larger, o);
    __syncthreads();
    if (at < size && part == 0 && mine != 0) list[larger] = mine;
    __syncthreads();
    // zeros: behind the others, where some of those may have stood
    if (at < size && part == 0 && mine == 0) larger = -1;
    const int zeros = __syncthreads_count(at < size && part == 0 && larger == -1);
    if ((int)threadIdx.x < zeros) list[size - 1 - threadIdx.x] = 0;
    __syncthreads();
    return;
  }
  for (int run = 2; run <= size; run <<= 1)
    for (int step = run >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & run) == 0)) list[a] = y, list[b] = x;
      }
      // a warp's pairs stay within 64 places below that distance
      if (step > 32 || (step == 1 && run >= 64)) __syncthreads();
      else __syncwarp();
    }
}

// ---------------------------------------------------------------------------------- any row, slowly

// `weigh`: by value, since the address of the caller's would keep it out of registers.
template <typename T, int kThreads, typename W>
__device__ __noinline__ void slow_row(const Params& p, int r, float top, float t, const W weigh, u64 least_w, Scratch& sc) {
  const int tid = threadIdx.x, v = p.vocab;
  const void* row = static_cast<const T*>(p.logits) + (int64_t)r * p.stride;
  // tokens of keys above `edge` are kept, and the first `ties` at it
  uint32_t edge = 0;
  u64 ties = ~0ull;
  const int k = p.top_k ? p.top_k[r] : 0;
  if (k > 0 && k < v) {
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {  // the largest key that at least k tokens reach
      const uint32_t probe = edge | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < v; i += kThreads) n += load_key<T>(row, i) >= probe;
      n = block_sum<kThreads>(n, sc.sum);
      if (n >= (u64)k) edge = probe;
      else above = n;
    }
    ties = (u64)k - above;
  }
  const float tp = p.top_p ? p.top_p[r] : 1.f;
  if (tp < 1.f) {
    const u64 at_edge = ties == ~0ull ? 0 : weigh(logit_of(edge)) * ties;
    u64 total = 0;
    for (int i = tid; i < v; i += kThreads) {
      const uint32_t key = load_key<T>(row, i);
      if (key > edge) total += weigh(logit_of(key));
    }
    total = block_sum<kThreads>(total, sc.sum) + at_edge;
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
      n = block_sum<kThreads>(n, sc.sum);
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
  // index order: each thread a stretch of the row
  const int per = (v + kThreads - 1) / kThreads;
  const int lo = min(v, tid * per), hi = min(v, lo + per);
  u64 n = 0, all;
  for (int i = lo; i < hi; ++i) n += load_key<T>(row, i) == edge;
  const u64 ties_before = scan<kThreads>(n, all, sc.sum);
  auto walk = [&](auto f) {
    u64 seen = ties_before;
    for (int i = lo; i < hi; ++i) {
      const uint32_t key = load_key<T>(row, i);
      bool keep = key > edge;
      if (key == edge) keep = seen++ < ties;
      if (!keep) continue;
      const u64 w = weigh(logit_of(key));
      if (w >= least_w) f(i, w);
    }
  };
  u64 mine = 0;
  walk([&](int, u64 w) { mine += w; });
  u64 run = scan<kThreads>(mine, all, sc.sum);
  u64 want = share_of(p.uniform[r], all);
  if (want >= all) want = all - 1;
  if (run <= want && want < run + mine) {
    walk([&](int i, u64 w) {
      if (run <= want && want < run + w) {
        p.ids[r] = i;
        const float l = load_one<T>(row, i);
        const double d = l == top ? 0. : ((double)l - (double)top) * (1. / (double)t);
        if (p.logp) p.logp[r] = (float)(d - log((double)all / (double)(1ull << p.scale_bits)));
      }
      run += w;
    });
  }
}

// ---------------------------------------------------------------------------------- bins

// `low`: (least biased exponent of the bins' octaves) * 128, at least 128.
// Logits of smaller magnitude share 0's bin (bf16 rows that have such go the slow way); larger ones, infinities and NaN have
// none.
template <typename T>
__device__ __forceinline__ int bin_of(float x, int low) {
  constexpr int kHalf = Bins<T>::kHalf;
  const int b = __float_as_int(x);
  const int off = max(((b >> 16) & 0x7fff) - (low - 1), 0);
  return off <= kHalf ? (b < 0 ? kHalf + off : kHalf - off) : Bins<T>::kNone;
}
// The least magnitude of a bin's logits, signed.
template <typename T>
__device__ __forceinline__ float logit_of_bin(int bin, int low) {
  constexpr int kHalf = Bins<T>::kHalf;
  if (bin == kHalf) return 0.f;
  const int off = bin < kHalf ? kHalf - bin : bin - kHalf;
  const uint32_t mag = (uint32_t)(off - 1 + low) << 16;
  return __uint_as_float(bin < kHalf ? mag : mag | 0x80000000u);
}
// The least of the logits in a bin or above it. (Above all bins, -1: none that a row has.)
template <typename T>
__device__ __forceinline__ float least_of_bin(int bin, int low) {
  constexpr int kHalf = Bins<T>::kHalf;
  if (bin < kHalf) return logit_of_bin<T>(bin, low);
  return __uint_as_float(0x80000000u | (((uint32_t)(bin - kHalf + low) << 16) - 1));
}

struct Shared {
  Scratch sc;
  uint32_t red[2 * kMaxWarps];
  int edge_bin, edge_count;  // the border: of that bin's tokens the first few are kept
  int lo_bin, hi_bin;        // the bins whose tokens are collected
  int list_n, list_over;
  int k_border;              // fp32: top-k ends among the binned tokens
  u64 edge;                  // fp32: the last token kept, as the list has it
  u64 edge_w;                // bf16: the weight of the border's bin
  double inv_t, unit;        // 1 / t and 2^-S
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const Params p) {
  constexpr bool WIDE = sizeof(T) == 4;
  constexpr int N = Row<T>::N, kWarps = kThreads / 32;
  constexpr int kHalf = Bins<T>::kHalf, kBins = Bins<T>::kBins, kNone = Bins<T>::kNone;
  constexpr int kBinsPadded = Bins<T>::template kPadded<kThreads>, kPerThread = kBinsPadded / kThreads;
  constexpr int kWide = kBinsPadded > kList ? kBinsPadded : kList;
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* counts = reinterpret_cast<uint32_t*>(smem);                 // [kBinsPadded + 4]
  u64* weights = reinterpret_cast<u64*>(smem + (kBinsPadded + 4) * 4);  // [kWide + 2]
  u64* list = weights;                                                  // or [kList] {key, ~index}
  uint2* table = reinterpret_cast<uint2*>(smem + (kBinsPadded + 4) * 4 + (kWide + 2) * 8);  // [kTable]
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x;
  for (int i = tid; i < (kBinsPadded + 4) / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < kTable; i += kThreads) table[i] = g_powers.at[i];
  if (tid == 0) sh.unit = 1. / (double)(1ull << p.scale_bits);
  if (tid == 0) {
    sh.edge_bin = kNone, sh.edge_count = 0, sh.lo_bin = kBinsPadded, sh.hi_bin = -1;
    sh.list_n = 0, sh.list_over = 0, sh.k_border = 0;
  }
  pdl_wait();
  const Row<T> row(p, r);
  const float t = p.temperature[r];
  const bool greedy = !(t > 0.f);
  if (tid == 0) sh.inv_t = 1. / (double)t;

  // ---- the largest logit, and the least
  float top = -INFINITY, least = INFINITY;  // (maxima and minima leave NaN out)
#pragma unroll 8
  for (int j = row.full0() + tid; j < row.full1(); j += kThreads) {
    const uint4 w = row.whole(j);
    top = fmaxf(top, Row<T>::largest(w)), least = fminf(least, Row<T>::least(w));
  }
  const int my_edge = row.edge();  // (these threads have that vector too)
  if (my_edge >= 0) row.each(my_edge, [&](int, float x) { top = fmaxf(top, x), least = fminf(least, x); });
  const float my_top = top;
  {
    uint32_t a = key_of(top), b = key_of(least);
    a = __reduce_max_sync(kAll, a);
    b = __reduce_min_sync(kAll, b);
    if (lane == 0) sh.red[warp] = a, sh.red[kWarps + warp] = b;
    __syncthreads();
    a = __reduce_max_sync(kAll, sh.red[lane % kWarps]);
    b = __reduce_min_sync(kAll, sh.red[kWarps + lane % kWarps]);
    top = logit_of(a);
    least = logit_of(b);
  }
  if (top == -INFINITY) {
    if (tid == 0) {
      p.ids[r] = -1;
      if (p.logp) p.logp[r] = NAN;
    }
    return;
  }
  if (greedy) {
    int first = INT32_MAX;
    if (my_top == top) {
      auto find = [&](int i, float x) {
        if (x == top) first = min(first, i);
      };
      for (int j = row.full0() + tid; j < row.full1(); j += kThreads)
        if (Row<T>::largest(row.whole(j)) == top) row.each(j, find);
      if (my_edge >= 0) row.each(my_edge, find);
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
  const int k = p.top_k ? p.top_k[r] : 0;
  const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < p.vocab, by_p = tp < 1.f, by_m = mp > 0.f;
  const u64 least_w = by_m ? share_of(mp, 1ull << p.scale_bits, true) : 0;
  if (isinf(top) || isinf(1.44269502f / t)) {
    const Weigher weigh = {(double)top, 1. / (double)t, (double)(1ull << p.scale_bits)};
    slow_row<T, kThreads>(p, r, top, t, weigh, least_w, sh.sc);
    return;
  }
  FastWeigher weigh;
  {
    constexpr float kLog2e = 1.44269502f, kRest = 1.92596299e-8f;  // their sum is log2(e)
    weigh.top = top;
    weigh.c = kLog2e / t;
    weigh.c_low = isinf(t) ? 0.f : (fmaf(-weigh.c, t, kLog2e) + kRest) / t;
    weigh.down = 63 - p.scale_bits;
    weigh.table = table;
  }
  // the log-probability of a token among kept weights that add up to `all`
  auto log_share = [&](float l, u64 all) {
    return (float)(((double)l - (double)top) * sh.inv_t - log((double)all * sh.unit));
  };
  // below this no weight is left
  const float cutoff = fmaxf(top - t * (0.694f * (float)(p.scale_bits + 2)) - 1e-6f * fabsf(top), -3.4e38f);
  const float widest = fmaxf(fabsf(top), fabsf(fmaxf(least, cutoff)));
  const int low = max((int)(__float_as_uint(widest) >> 23) - (kHalf / 128 - 1), 1) * 128;

  // ---- top-k of a few
  if (by_k && k <= kThreads / 2) {
    // The bin of the k-th largest of the threads' largest: at least k tokens are in it or above. Where fewer threads
    // have any, or theirs weigh nothing, there is none, and every token that weighs is taken.
    const int my_bin = bin_of<T>(my_top, low);
    if (my_bin != kNone) atomicAdd(&counts[my_bin], 1u);
    __syncthreads();
    const int b0 = tid * kPerThread;
    u64 mine = 0, all;
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) mine += counts[b0 + i];
    u64 before = scan<kThreads>(mine, all, sh.sc.sum);
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) {
      if (before < (u64)k && before + counts[b0 + i] >= (u64)k) sh.hi_bin = b0 + i;
      before += counts[b0 + i];
    }
    __syncthreads();
    const int hi = sh.hi_bin;
    const float from = hi < 0 ? fmaxf(least, cutoff) : least_of_bin<T>(hi, low);
    if (my_top >= from) {
      for (int j = row.full0() + tid, e = my_edge; j < row.full1() || e >= 0; j += 4 * kThreads) {
        uint32_t hits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i * kThreads < row.full1()) hits |= (uint32_t)(Row<T>::largest(row.whole(j + i * kThreads)) >= from) << i;
        if (e >= 0) hits |= 16;
        for (; hits != 0; hits &= hits - 1) {
          const int at = hits & 15 ? j + (__ffs(hits) - 1) * kThreads : e;
          float x[N];
          row.load(at, x);
          uint32_t in = 0;
#pragma unroll
          for (int i = 0; i < N; ++i) in |= (uint32_t)(x[i] >= from) << i;
          int to = in != 0 ? atomicAdd(&sh.list_n, __popc(in)) : 0;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if ((in >> i & 1) == 0) continue;
            if (to < kList) list[to] = (u64)key_of(x[i]) << 32 | (uint32_t)~(at * N - row.shift + i);
            ++to;
          }
        }
        e = -1;
      }
    }
    if (my_bin != kNone) counts[my_bin] = 0;  // (only that bin's threads, and for whoever comes next)
    __syncthreads();
    const int n = sh.list_n;
    if (n <= kList) {
      int size = 64;
      while (size < n) size <<= 1;
      for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
      __syncthreads();
      sort<kThreads>(list, size);
      // at most one of the first k to a thread: weights fall along the threads, so what is kept is a beginning of them
      const int m = min(n, k);
      const u64 w = tid < m ? weigh(logit_of((uint32_t)(list[tid] >> 32))) : 0;
      u64 all_w;
      const u64 before_w = scan<kThreads>(w, all_w, sh.sc.sum);
      const u64 want = by_p ? share_of(tp, all_w, true) : ~0ull;
      const bool keep = tid < m && (tid == 0 || (before_w < want && w >= least_w));
      const int kept = __syncthreads_count(keep);
      // in index order
      u64* order = reinterpret_cast<u64*>(counts);  // {~index, place}
      int size2 = 64;
      while (size2 < kept) size2 <<= 1;
      if (tid < size2) order[tid] = tid < kept ? (u64)(uint32_t)list[tid] << 32 | (uint32_t)tid : 0;
      __syncthreads();
      sort<kThreads>(order, size2);
      const bool mine_kept = tid < kept;
      const u64 at = mine_kept ? list[(uint32_t)order[tid]] : 0;
      const float l = logit_of((uint32_t)(at >> 32));
      const u64 w2 = mine_kept ? weigh(l) : 0;
      u64 all2;
      const u64 run = scan<kThreads>(w2, all2, sh.sc.sum);
      u64 target = share_of(p.uniform[r], all2);
      if (target >= all2) target = all2 - 1;
      if (mine_kept && run <= target && target < run + w2) {
        p.ids[r] = (int)~(uint32_t)at;
        if (p.logp) p.logp[r] = log_share(l, all2);
      }
      return;
    }
    __syncthreads();  // (every thread has seen how many there are)
    if (tid == 0) sh.hi_bin = -1, sh.list_n = 0;
    __syncthreads();
  }

  // ---- bins
  const bool bins = by_k || by_p;
  if (bins) {
    bool strange = false;
    // fp32: the mean logit of the bins whose tokens weigh e^-6 or more, of which few may make up the total
    const int heavy = WIDE && by_p ? bin_of<T>(top - 6.f * t, low) : -1;
    const int coarse = max(16 - __clz(p.vocab - 1), 0);  // so that the whole vocabulary's low halves add up to less than 2^32
    if (WIDE && by_p) {
      for (int i = tid; i < kBinsPadded; i += kThreads) weights[i] = 0;
      __syncthreads();
    }
#pragma unroll 2
    for (int j = tid; j < row.vectors; j += kThreads) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of<T>(x[i], low);
        if (!WIDE) strange |= bin == kHalf && x[i] != 0.f;
        if (bin != kNone) atomicAdd(&counts[bin], 1u);
        if (WIDE && bin <= heavy && bin != kNone)
          atomicAdd(reinterpret_cast<uint32_t*>(&weights[bin]), (__float_as_uint(x[i]) & 0xffffu) >> coarse);
      }
    }
    if (__syncthreads_or(strange)) {
      slow_row<T, kThreads>(p, r, top, t, weigh, least_w, sh.sc);
      return;
    }
    // Their weights: neighbouring bins, which tend to be filled together, on different threads. Where fp32 has no mean
    // it takes a bin's middle.
    for (int b = tid; b < kBins; b += kThreads) {
      const uint32_t n = counts[b];
      if (n == 0) continue;
      float l = logit_of_bin<T>(b, low);
      if (WIDE && b != kHalf) {
        const uint32_t in =
            b <= heavy ? (uint32_t)(__fdividef((float)(uint32_t)weights[b], (float)n) * (float)(1 << coarse)) : 0x8000u;
        l = fminf(__uint_as_float(__float_as_uint(l) + in), top);
      }
      weights[b] = weigh(l);
    }
    __syncthreads();
    // Each thread a few neighbouring bins, largest logits first: tokens of each that top-k leaves, and their mass.
    const int b0 = tid * kPerThread;
    u64 mine_n = 0, mine_w = 0, all_n, all_w;
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) mine_n += counts[b0 + i];
    u64 before = scan<kThreads>(mine_n, all_n, sh.sc.sum);
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) {
      const uint32_t had = counts[b0 + i];
      uint32_t n = had;
      if (by_k) {
        n = before >= (u64)k ? 0u : (uint32_t)min((u64)had, (u64)k - before);
        if ((n < had && n > 0) || (before + had == (u64)k && had > 0)) {
          if (!WIDE) sh.edge_bin = b0 + i, sh.edge_count = (int)n;
          else atomicMin(&sh.lo_bin, b0 + i), atomicMax(&sh.hi_bin, b0 + i), sh.k_border = 1;
        }
        counts[b0 + i] = n;
      }
      before += had;
      if (n > 0) mine_w += weights[b0 + i] * n;
    }
    u64 mass = scan<kThreads>(mine_w, all_w, sh.sc.sum);
    const u64 want = by_p ? share_of(tp, all_w, true) : ~0ull;
    // fp32: the border is somewhere near (checked later): within 2^-11 of the total and five deviations of what
    // the others' middles leave out, a token of half a bin's width h being off by up to w h / t, on average 0
    u64 slack = 0;
    if (WIDE && by_p) {
      float off = 0.f;
      const float per_width = 0.0078125f / t;
#pragma unroll 3
      for (int i = 0; i < kPerThread; ++i) {
        const int b = b0 + i;
        if (counts[b] == 0 || b == kHalf || b <= heavy) continue;
        const float width = fabsf(logit_of_bin<T>(b, low)) * per_width;  // at most
        const float one_off = (float)weights[b] * fminf(0.5f * width, 4.f);
        off += (float)counts[b] * one_off * one_off * 0.333f;
      }
      off = warp_sum(off);
      if (lane == 0) sh.red[warp] = __float_as_uint(off);
      __syncthreads();
      off = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) off += __uint_as_float(sh.red[i]);
      slack = (all_w >> 11) + 1 + (u64)fminf(5.f * sqrtf(off), (float)all_w);
    }
    const u64 want_lo = want > slack ? want - slack : 0, want_hi = want + slack;
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) {
      const int b = b0 + i;
      uint32_t n = counts[b];
      if (n == 0) {
        if (!WIDE) weights[b] = 0;
        continue;
      }
      const u64 w = weights[b], here = w * n;
      if (WIDE) {  // bins that the border may fall into
        if (by_p && mass <= want_hi && mass + here >= want_lo) atomicMin(&sh.lo_bin, b), atomicMax(&sh.hi_bin, b);
      } else {
        bool keep = true;
        if (by_p) {
          const uint32_t had = n;
          if (mass >= want) n = mass == 0;  // the first token always stays
          else if (w > 0 && mass + here >= want) n = (uint32_t)min((u64)had, (want - mass + w - 1) / w);
          keep = n > 0;
          if (keep && (n < had || mass + here >= want)) sh.edge_bin = b, sh.edge_count = (int)n;
        }
        if (!keep || w < least_w) weights[b] = 0;
      }
      mass += here;
    }
    __syncthreads();
    if (!WIDE) {
      // the border's bin is counted token by token
      if (tid == 0) {
        weights[kNone] = 0;
        if (sh.edge_bin != kNone) {
          sh.edge_w = weights[sh.edge_bin];
          weights[sh.edge_bin] = 0;
        }
      }
      __syncthreads();
    }
  }

  // ---- kept weights of every warp's stretch
  const int per_warp = (row.vectors + kWarps - 1) / kWarps;
  const int v0 = min(row.vectors, warp * per_warp), v1 = min(row.vectors, v0 + per_warp);
  if (!WIDE && bins) {
    const int edge = sh.edge_bin;
    const u64 edge_w = edge == kNone ? 0 : sh.edge_w;
    const u64 edge_n = (u64)sh.edge_count;
    u64 sum = 0;
    uint32_t ties = 0;
#pragma unroll 2
    for (int j = v0 + lane; j < v1; j += 32) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of<T>(x[i], low);
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
    // a stretch to a lane: ties before it, and the weight with those that stay
    const u64 my_ties = lane < kWarps ? sh.sc.sum2[lane] : 0;
    const u64 seen = lane_scan(my_ties);
    const u64 stay = seen >= edge_n ? 0 : min(my_ties, edge_n - seen);
    const Stretch in = stretch_of((lane < kWarps ? sh.sc.sum[lane] : 0) + stay * edge_w, p.uniform[r]);
    const u64 seen_in = __shfl_sync(kAll, seen, in.at);
    __syncthreads();
    // ---- the stretch with the target, a vector or a few to a thread
    const int s0 = min(row.vectors, in.at * per_warp), s1 = min(row.vectors, s0 + per_warp);
    const int per = (s1 - s0 + kThreads - 1) / kThreads;
    const int j0 = min(s1, s0 + tid * per), j1 = min(s1, j0 + per);
    u64 mine = 0, mine_ties = 0, dummy;
    for (int j = j0; j < j1; ++j) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int bin = bin_of<T>(x[i], low);
        mine += weights[bin];
        mine_ties += bin == edge && edge != kNone;
      }
    }
    u64 my_seen = seen_in + scan<kThreads>(mine_ties, dummy, sh.sc.sum);
    const u64 my_stay = my_seen >= edge_n ? 0 : min(mine_ties, edge_n - my_seen);
    mine += my_stay * edge_w;
    u64 my_run = in.before + scan<kThreads>(mine, dummy, sh.sc.sum);
    if (my_run <= in.target && in.target < my_run + mine) {
      for (int j = j0; j < j1; ++j) {
        float x[N];
        row.load(j, x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int bin = bin_of<T>(x[i], low);
          u64 w = weights[bin];
          if (bin == edge && edge != kNone && my_seen++ < edge_n) w = edge_w;
          if (my_run <= in.target && in.target < my_run + w) {
            p.ids[r] = j * N - row.shift + i;
            if (p.logp) p.logp[r] = log_share(x[i], in.all);
          }
          my_run += w;
        }
      }
    }
    return;
  }

  const bool edged = WIDE && bins && sh.hi_bin >= 0;  // (top-k of more tokens than weigh anything leaves all)
  const int lo = edged ? sh.lo_bin : kNone, hi = edged ? sh.hi_bin : kNone;
  const bool all_rest = by_p && !sh.k_border;  // the total that top-p takes a share of goes on below the list
  u64 sum = 0, total = 0, above_w = 0;
  if (!edged) {
#pragma unroll 2
    for (int j = v0 + lane; j < v1; j += 32) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u64 w = weigh(x[i]);
        sum += by_m && w < least_w ? 0 : w;
      }
    }
  } else {
    const float from_above = least_of_bin<T>(lo - 1, low), from_list = least_of_bin<T>(hi, low);
#pragma unroll 2
    for (int j = v0 + lane; j < v1; j += 32) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u64 w = weigh(x[i]);
        const bool above = x[i] >= from_above;
        total += w;
        above_w += above ? w : 0;
        if (by_m) sum += above && w >= least_w ? w : 0;
        if (!above && x[i] >= from_list) {
          const int at = atomicAdd(&sh.list_n, 1);
          if (at < kList) list[at] = (u64)key_of(x[i]) << 32 | (uint32_t)~(j * N - row.shift + i);
        }
      }
    }
    if (!by_m) sum = above_w;
  }
  u64 edge = 0;  // tokens at or above it (key, then lower indexes) are kept
  if (edged) {
    u64 n_above = 0;  // (these bins have all their tokens)
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i)
      if (tid * kPerThread + i < lo) n_above += counts[tid * kPerThread + i];
    block_sums<kThreads>(above_w, total, n_above, sh.sc);
    const int n = sh.list_n;
    if (n > kList) {
      slow_row<T, kThreads>(p, r, top, t, weigh, least_w, sh.sc);
      return;
    }
    // sort the list, largest first
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    sort<kThreads>(list, size);
    // their weights, and what top-k, then top-p leaves of them
    const int per = (size + kThreads - 1) / kThreads, i0 = min(size, tid * per), i1 = min(size, i0 + per);
    const u64 left_k = by_k ? ((u64)k > n_above ? (u64)k - n_above : 0) : ~0ull;
    u64 mine = 0, all_w;
    for (int i = i0; i < i1; ++i)
      if (i < n && (u64)i < left_k) mine += weigh(logit_of((uint32_t)(list[i] >> 32)));
    u64 mass = above_w + scan<kThreads>(mine, all_w, sh.sc.sum);
    // (where all_rest holds, all_w is the list's whole mass)
    const u64 rest_w = all_rest ? total - above_w - all_w : 0;
    const u64 want = by_p ? share_of(tp, above_w + all_w + rest_w, true) : ~0ull;
    if (tid == 0) sh.edge = 0, sh.list_over = 0;
    __syncthreads();
    // The last token kept; the first of all always is. A top-p border outside the list is a slow row.
    for (int i = i0; i < i1; ++i) {
      if (i >= n || (u64)i >= left_k) break;
      const u64 w = weigh(logit_of((uint32_t)(list[i] >> 32)));
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
      slow_row<T, kThreads>(p, r, top, t, weigh, least_w, sh.sc);
      return;
    }
  }
  auto kept = [&](float l, int i) {
    const u64 w = weigh(l);
    const bool below = edged && ((u64)key_of(l) << 32 | (uint32_t)~i) < edge;
    return below || w < least_w ? 0 : w;
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
      const u64 w = kept(logit_of((uint32_t)(list[i] >> 32)), index);
      if (w) atomicAdd(&sh.sc.sum2[(index + row.shift) / N / per_warp], w);
    }
  }
  if (lane == 0) sh.sc.sum[warp] = sum;
  __syncthreads();
  const Stretch in = stretch_of(lane < kWarps ? sh.sc.sum[lane] + sh.sc.sum2[lane] : 0, p.uniform[r]);
  __syncthreads();
  // ---- the stretch with the target, a vector or a few to a thread
  const int s0 = min(row.vectors, in.at * per_warp), s1 = min(row.vectors, s0 + per_warp);
  const int per = (s1 - s0 + kThreads - 1) / kThreads;
  const int j0 = min(s1, s0 + tid * per), j1 = min(s1, j0 + per);
  u64 mine = 0, dummy;
  for (int j = j0; j < j1; ++j) {
    float x[N];
    row.load(j, x);
#pragma unroll
    for (int i = 0; i < N; ++i) mine += kept(x[i], j * N - row.shift + i);
  }
  u64 my_run = in.before + scan<kThreads>(mine, dummy, sh.sc.sum);
  if (my_run <= in.target && in.target < my_run + mine) {
    for (int j = j0; j < j1; ++j) {
      float x[N];
      row.load(j, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u64 w = kept(x[i], j * N - row.shift + i);
        if (my_run <= in.target && in.target < my_run + w) {
          p.ids[r] = j * N - row.shift + i;
          if (p.logp) p.logp[r] = log_share(x[i], in.all);
        }
        my_run += w;
      }
    }
  }
}

template <typename T, int kThreads>
static int launch(const Params& p, int rows, cudaStream_t st) {
  constexpr int kBinsPadded = Bins<T>::template kPadded<kThreads>, kWide = kBinsPadded > kList ? kBinsPadded : kList;
  constexpr int SMEM = (kBinsPadded + 4) * 4 + (kWide + 2) * 8 + kTable * 8;
  static_assert(kBinsPadded > Bins<T>::kNone, "room for no bin");
  static_assert(1024 / kThreads * (SMEM + 2048) <= 228 * 1024, "CTAs an SM");
  auto kernel = sample_kernel<T, kThreads>;
  if (allow_shared(reinterpret_cast<const void*>(kernel), SMEM) != cudaSuccess) return CDB_ERR_CUDA;
  return launch_pdl(kernel, dim3(rows), dim3(kThreads), SMEM, st, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
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
  // One CTA an SM has the whole SM while there are no more rows than SMs; two share it where there are more.
  if (num_rows <= 148)
    return logits_fp32 ? launch<float, 1024>(p, num_rows, st) : launch<__nv_bfloat16, 1024>(p, num_rows, st);
  return logits_fp32 ? launch<float, 512>(p, num_rows, st) : launch<__nv_bfloat16, 512>(p, num_rows, st);
}
