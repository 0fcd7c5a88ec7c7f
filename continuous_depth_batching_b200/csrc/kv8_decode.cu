// Decode attention over the 8-bit paged cache (layout in kv8.cuh): one query row per item, any
// number of query heads per kv head.
//
// Work. The pages (blocks) of all (row, kv head, group of up to 8 query heads) segments, in that order
// and in pairs, form one stream that is cut into equal shares, one per CTA, and each share into one per
// warp: a long row is spread over the whole GPU and short rows are packed, by the positions that lie on
// the device. Each warp streams its pairs of pages through a ring of its own in shared memory (a page is
// two contiguous tiles, K and V, one copy each), so no warp waits for another until its share ends. Pairs,
// because a page alone leaves the warp with one chain of dependent products and pays for the loop, the
// copies' bookkeeping and the softmax's vote by itself.
//
// Mathematics. Per page, with K the 16 x D tile of codes: S = K q (tensor cores, f16 operands, fp32
// accumulators). Codes convert to f16 exactly, and q is divided by a power of two that brings its
// largest element to [1, 2), so that bf16's 8 significant bits fit f16; what f16 loses lies below
// 2^-24 of the row's largest element. x = S * (scale log2e 2^e s_k) in fp32. The softmax runs online
// in base 2: m is a maximum of x that only moves when x passes it by 8 (then l, the sum of 2^(x-m),
// is rescaled), and the weights of V, 2^(x-m) s_v, are taken relative to their own maximum M of
// x + log2 s_v, so that they fit f16 whatever the blocks' scales are (kLift in kv8.cuh: 2^-11 relative rounding each,
// averaged over the keys, or 2^-32 of the largest). O = V^T P (tensor cores again) in fp32.
//
// Pieces of a segment (m, l, o) meet in two steps: the warps of a CTA through shared memory, CTAs
// through the workspace, where the last one to arrive adds them up in CTA order, head by head. The result
// does not depend on which one that is.
//
// Measured: 8 rows of 30,000 to 65,536 positions, 32 query heads on 8 of 128: 141 us, 5.6 TB/s, bound by HBM; 80 rows
// at 64 to 1300, 16 heads: 47 us, 4.8 TB/s over all, of which 3.6 us go by before the first page and 4 in the joins;
// one row of 700: 9.7 us, a chain of latencies. (Eager calls; one from a captured graph takes 1 to 1.5 us more, 11.2
// there, because a fill in front of it zeroes counters of its own: the graph may run beside others.) 12 warps, because
// 163 registers a thread (a head's q and output stay in them) and rings of two pairs (8 KB each at 128) take the SM's
// registers and shared memory. More than 8 query heads a kv head stream its pages once per 8 of them, the second time
// from L2: 8 rows of 32,768 with 16 heads on 2 43 us (134 MB), 32 heads on 2 57 us.
#include <cuda.h>

#include "kv8.cuh"

namespace cdb {
namespace kv8 {

constexpr int kWarps = 12;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxStages = 4;
constexpr int kGroup = 8;  // query heads of one segment (the n of an m16n8k16 product)
constexpr uint32_t kFull = 0xffffffffu;

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const uint8_t* codes;  // this cache layer's K; V follows num_blocks * kv_heads tiles later
  const float* scales;
  int num_blocks, kv_heads, heads_per_kv, groups;  // groups of kGroup query heads per kv head
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int32_t* item_slot;
  const int32_t* item_pos;
  int num_items;
  float scale_log2;
  int min_share;     // pairs of one CTA's share, at least
  int whole_pairs;   // the longest segments that are kept in one CTA, where there are few
  int stages;        // pairs in a warp's ring
  int stored_heads;  // heads of a stored piece: min(heads_per_kv, kGroup)
  float* parts;      // [CTAs][2][stored_heads][D + 2], then, unless they fit shared memory, each CTA's
  float* first;      // [CTAs][kWarps][stored_heads][D + 2] first pieces of the warps; null: shared memory
  int32_t* counters;
  int32_t* status;
};

// a / b for a, b >= 0: a 64-bit division takes some 400 cycles, and the numbers nearly always fit 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Pairs of cached pages of row b; 0 for a padding row and for one whose indexes do not fit the table.
__device__ __forceinline__ int row_pairs(const DecodeParams& p, int b, bool& bad) {
  const int pos = p.item_pos[b], slot = p.item_slot[b];
  if (pos < 0) return 0;
  if (slot < 0 || slot >= p.bt_rows || pos / kBlock >= p.bt_width) {
    bad = true;
    return 0;
  }
  return pos / (2 * kBlock) + 1;
}

// A place in the stream: pair `pair` of row `row`, query-head group `grp` of kv head `kvh`.
struct Cursor {
  int row, kvh, grp, pair, pairs, pos, slot;
};

// Its row's position, slot and pairs. `rows`: {position, slot} of every row in shared memory (a row that does
// not count has position -1), or null where there are more rows than threads.
__device__ __forceinline__ void load_row(const DecodeParams& p, const int2* rows, Cursor& c) {
  if (rows != nullptr) {
    c.pos = rows[c.row].x;
    c.slot = rows[c.row].y;
    c.pairs = c.pos < 0 ? 0 : c.pos / (2 * kBlock) + 1;
  } else {
    bool bad = false;
    c.pairs = row_pairs(p, c.row, bad);
    c.pos = p.item_pos[c.row];
    c.slot = p.item_slot[c.row];
  }
}

// To the next pair.
__device__ __forceinline__ void advance(const DecodeParams& p, const int2* rows, Cursor& c) {
  if (++c.pair < c.pairs) return;
  c.pair = 0;
  if (++c.grp < p.groups) return;
  c.grp = 0;
  if (++c.kvh < p.kv_heads) return;
  c.kvh = 0;
  do {
    if (++c.row >= p.num_items) return;  // the stream's end
    load_row(p, rows, c);
  } while (c.pairs == 0);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void tensor_load(uint32_t dst, const CUtensorMap* map, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(bar)
      : "memory");
}

// 4 bytes to shared memory, asynchronously; async_arrive lets `bar` count their completion.
__device__ __forceinline__ void async_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Where a piece lies in its segment, for the joins.
struct PieceTag {
  int row, kvh, grp;
  int first, last, pairs;  // pairs [first, last) of `pairs`
};

template <int D>
struct Shape {
  static constexpr int KD = D / 4;         // dims of K that a lane multiplies: [t * KD, t * KD + KD) of rows g, g + 8
  static constexpr int VD = D / 8;         // dims of V that a lane multiplies: [g * VD, g * VD + VD) of 4 tokens
  static constexpr int KS = D / 16;        // k-steps of K q
  static constexpr int MT = D / 16;        // m-tiles of V^T P
  static constexpr int TILE = kBlock * D;  // bytes of a K or V tile
  // Rows of 128 and 64 bytes come through a tensor map with the swizzle of that width, which spreads
  // the fragment loads below over the banks (unswizzled, a V load hits each bank four times); rows of 96
  // bytes spread by themselves and come as one untiled copy.
  static constexpr bool SWIZZLED = D != 96;
};

// Byte offset of byte c (16-byte aligned) of row r in a tile.
template <int D>
__device__ __forceinline__ int tile_at(int r, int c) {
  if (D == 128) return r * 128 + (c ^ ((r & 7) << 4));
  if (D == 64) return r * 64 + (c ^ (((r >> 1) & 3) << 4));
  return r * D + c;
}

// The running softmax of one segment piece and what a lane holds of V^T P: dims g * VD + 4 i + {0, 1, 2,
// 3} of head 2t (h = 0) and 2t + 1 (h = 1) in acc[2i][h], acc[2i][2 + h], acc[2i + 1][h], acc[2i + 1][2 + h].
// HN: heads a lane keeps (1 where a kv head has one query head: only h = 0 of t = 0 means anything then).
template <int D, int HN>
struct Running {
  float acc[Shape<D>::MT][4];
  float m[HN], mw[HN], l[HN];  // mw: M - kLift
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < Shape<D>::MT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      m[h] = mw[h] = -INFINITY;
      l[h] = 0.f;
    }
  }
};

// q's rows of one segment as the B operand: head g of the group, dims [t * KD, (t + 1) * KD). e is the
// power of two that was divided out (for heads 2t and 2t + 1).
template <int D>
__device__ __forceinline__ void fetch_q(const DecodeParams& p, const Cursor& c, uint32_t (&w)[D / 8]) {
  constexpr int KD = Shape<D>::KD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int in_kv = c.grp * kGroup + g;
  const bool on = in_kv < p.heads_per_kv;
  const __nv_bfloat16* src =
      p.q + (int64_t)c.row * p.q_stride + (int64_t)(c.kvh * p.heads_per_kv + (on ? in_kv : 0)) * D + t * KD;
#pragma unroll
  for (int i = 0; i < KD / 8; ++i) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (on) v = *reinterpret_cast<const uint4*>(src + i * 8);
    w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
  }
}

template <int D, int HN>
__device__ __forceinline__ void convert_q(const DecodeParams& p, const uint32_t (&w)[D / 8],
                                          uint32_t (&qf)[Shape<D>::KS][2], float (&factor)[HN]) {
  constexpr int KD = Shape<D>::KD;
  const int t = threadIdx.x & 3;
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < KD / 2; ++i) amax = fmaxf(amax, fmaxf(fabsf(bf16lo(w[i])), fabsf(bf16hi(w[i]))));
  amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
  int e = (int)(__float_as_uint(amax) >> 23) - 127;
  e = amax == 0.f ? 0 : max(-126, min(126, e));
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int i = 0; i < KD / 2; ++i) qf[i >> 1][i & 1] = pack_f16x2(bf16lo(w[i]) * down, bf16hi(w[i]) * down);
  const float f = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
#pragma unroll
  for (int h = 0; h < HN; ++h) factor[h] = __shfl_sync(kFull, f, t * 8 + h * 4);  // the lanes of head 2t + h
}

// The fragments of one page's K: rows g and g + 8, dims [t * KD, (t + 1) * KD).
template <int D>
__device__ __forceinline__ void load_k(const uint8_t* k, uint32_t (&ka)[D / 16], uint32_t (&kb)[D / 16]) {
  constexpr int KD = Shape<D>::KD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if constexpr (KD % 16 == 0) {
#pragma unroll
    for (int i = 0; i < KD / 16; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(k + tile_at<D>(g, t * KD + i * 16));
      const uint4 y = *reinterpret_cast<const uint4*>(k + tile_at<D>(g + 8, t * KD + i * 16));
      ka[4 * i] = x.x, ka[4 * i + 1] = x.y, ka[4 * i + 2] = x.z, ka[4 * i + 3] = x.w;
      kb[4 * i] = y.x, kb[4 * i + 1] = y.y, kb[4 * i + 2] = y.z, kb[4 * i + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < KD / 8; ++i) {
      const uint2 x = *reinterpret_cast<const uint2*>(k + g * D + t * KD + i * 8);
      const uint2 y = *reinterpret_cast<const uint2*>(k + (g + 8) * D + t * KD + i * 8);
      ka[2 * i] = x.x, ka[2 * i + 1] = x.y, kb[2 * i] = y.x, kb[2 * i + 1] = y.y;
    }
  }
}

// The fragments of one page's V: tokens 2t, 2t + 1, 2t + 8, 2t + 9, dims [g * VD, (g + 1) * VD).
template <int D>
__device__ __forceinline__ void load_v(const uint8_t* v, uint32_t (&vw)[4][D / 32]) {
  constexpr int VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
    if constexpr (VD == 16) {
      const uint4 x = *reinterpret_cast<const uint4*>(v + tile_at<D>(tok, g * 16));
      vw[j][0] = x.x, vw[j][1] = x.y, vw[j][2] = x.z, vw[j][3] = x.w;
    } else if constexpr (VD == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(v + tile_at<D>(tok, (g >> 1) * 16) + (g & 1) * 8);
      vw[j][0] = x.x, vw[j][1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < VD / 4; ++i) vw[j][i] = *reinterpret_cast<const uint32_t*>(v + tok * D + g * VD + i * 4);
    }
  }
}

// One pair of pages at `at` (K, V of the first, K, V of the second). scale: K's and V's of the first, then
// of the second; K's < 0 where the page does not exist. `live` tokens of the pair count.
template <int D, int HN>
__device__ __forceinline__ void pair_step(const uint8_t* at, const float4 scale, int live,
                                          const uint32_t (&qf)[Shape<D>::KS][2], const float (&factor)[HN],
                                          Running<D, HN>& r) {
  constexpr int KD = Shape<D>::KD, VD = Shape<D>::VD, TILE = Shape<D>::TILE;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[2][4];
#pragma unroll
  for (int pg = 0; pg < 2; ++pg) {
    uint32_t ka[KD / 4], kb[KD / 4];
    load_k<D>(at + pg * 2 * TILE, ka, kb);
    s[pg][0] = s[pg][1] = s[pg][2] = s[pg][3] = 0.f;
#pragma unroll
    for (int i = 0; i < KD / 4; ++i)
      mma_f16(s[pg], cvt_e4m3x2_f16x2(ka[i] & 0xffffu), cvt_e4m3x2_f16x2(kb[i] & 0xffffu),
              cvt_e4m3x2_f16x2(ka[i] >> 16), cvt_e4m3x2_f16x2(kb[i] >> 16), qf[i][0], qf[i][1]);
  }
  uint32_t vw[2][4][VD / 4];
  load_v<D>(at + TILE, vw[0]);
  load_v<D>(at + 3 * TILE, vw[1]);
  // s[pg][h]: token g, head 2t + h; s[pg][2 + h]: token g + 8
  const float ks[2] = {scale.x, scale.z};
  const float ev[2] = {scale.y > 0.f ? __log2f(scale.y) : -126.f, scale.w > 0.f ? __log2f(scale.w) : -126.f};
  float x[HN][4];
#pragma unroll
  for (int h = 0; h < HN; ++h) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const float f = factor[h] * ks[pg];
      x[h][2 * pg] = s[pg][h] * f;
      x[h][2 * pg + 1] = s[pg][2 + h] * f;
    }
  }
  if (live < 2 * kBlock || ks[0] < 0.f || ks[1] < 0.f) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const int end = ks[pg] < 0.f ? 0 : live - pg * kBlock;
#pragma unroll
      for (int h = 0; h < HN; ++h) {
        if (g >= end) x[h][2 * pg] = -INFINITY;
        if (g + 8 >= end) x[h][2 * pg + 1] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // codes behind the row's end may be anything, NaN too
        if (2 * t + (j & 1) + 8 * (j >> 1) >= end) {
#pragma unroll
          for (int i = 0; i < VD / 4; ++i) vw[pg][j][i] = 0u;
        }
      }
    }
  }
  // m and M only move when a logit passes them by 8 (the weights stay within 2^8 of 2^kLift): a vote a pair
  bool up = false;
#pragma unroll
  for (int h = 0; h < HN; ++h) {
    const float a = fmaxf(x[h][0], x[h][1]), b = fmaxf(x[h][2], x[h][3]);
    up = up || fmaxf(a, b) > r.m[h] + 8.f || fmaxf(a + ev[0], b + ev[1]) > r.mw[h] + (8.f + kLift);
  }
  if (__any_sync(kFull, up)) {
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      const float a = fmaxf(x[h][0], x[h][1]), b = fmaxf(x[h][2], x[h][3]);
      float mx = fmaxf(a, b), mz = fmaxf(a + ev[0], b + ev[1]);
#pragma unroll
      for (int d = 4; d <= 16; d <<= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
        mz = fmaxf(mz, __shfl_xor_sync(kFull, mz, d));
      }
      const float m = fmaxf(r.m[h], mx), mw = fmaxf(r.mw[h], mz - kLift);
      r.l[h] *= m == -INFINITY ? 1.f : ex2(r.m[h] - m);
      const float down = mw == -INFINITY ? 1.f : ex2(r.mw[h] - mw);
      r.m[h] = m;
      r.mw[h] = mw;
#pragma unroll
      for (int i = 0; i < Shape<D>::MT; ++i) r.acc[i][h] *= down, r.acc[i][2 + h] *= down;
    }
  }
  float pw[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    pw[j][1] = 0.f;
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      const bool off = x[h][j] == -INFINITY;  // also where m is still -inf
      r.l[h] += off ? 0.f : ex2(x[h][j] - r.m[h]);
      pw[j][h] = off ? 0.f : ex2(x[h][j] + ev[j >> 1] - r.mw[h]);
    }
  }
#pragma unroll
  for (int pg = 0; pg < 2; ++pg) {
    const uint32_t b0 = transpose8(pack_f16x2(pw[2 * pg][0], pw[2 * pg][1]));
    const uint32_t b1 = transpose8(pack_f16x2(pw[2 * pg + 1][0], pw[2 * pg + 1][1]));
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) {
      const uint32_t lo0 = __byte_perm(vw[pg][0][i], vw[pg][1][i], 0x5140);
      const uint32_t hi0 = __byte_perm(vw[pg][0][i], vw[pg][1][i], 0x7362);
      const uint32_t lo1 = __byte_perm(vw[pg][2][i], vw[pg][3][i], 0x5140);
      const uint32_t hi1 = __byte_perm(vw[pg][2][i], vw[pg][3][i], 0x7362);
      mma_f16(r.acc[2 * i], cvt_e4m3x2_f16x2(lo0 & 0xffffu), cvt_e4m3x2_f16x2(lo0 >> 16),
              cvt_e4m3x2_f16x2(lo1 & 0xffffu), cvt_e4m3x2_f16x2(lo1 >> 16), b0, b1);
      mma_f16(r.acc[2 * i + 1], cvt_e4m3x2_f16x2(hi0 & 0xffffu), cvt_e4m3x2_f16x2(hi0 >> 16),
              cvt_e4m3x2_f16x2(hi1 & 0xffffu), cvt_e4m3x2_f16x2(hi1 >> 16), b0, b1);
    }
  }
}

// A finished segment's output, straight from a warp's registers (l already summed over the warp).
template <int D, int HN>
__device__ __forceinline__ void write_out(const DecodeParams& p, const Cursor& c, const Running<D, HN>& r) {
  constexpr int VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int h = 0; h < HN; ++h) {
    const int in_kv = c.grp * kGroup + 2 * t + h;
    if (in_kv >= p.heads_per_kv) continue;
    const float f = r.l[h] > 0.f ? ex2(r.mw[h] + kLift - r.m[h]) * kUnlift / r.l[h] : (r.l[h] == 0.f ? 0.f : r.l[h]);
    __nv_bfloat16* dst =
        p.out + (int64_t)c.row * p.out_stride + (int64_t)(c.kvh * p.heads_per_kv + in_kv) * D + g * VD;
#pragma unroll
    for (int i = 0; i < VD / 4; ++i)
      *reinterpret_cast<uint2*>(dst + i * 4) =
          make_uint2(pack_bf16x2(r.acc[2 * i][h] * f, r.acc[2 * i][2 + h] * f),
                     pack_bf16x2(r.acc[2 * i + 1][h] * f, r.acc[2 * i + 1][2 + h] * f));
  }
}

// A piece: per stored head D values of o = sum 2^(x-m) v, then m and l.
template <int D, int HN>
__device__ __forceinline__ void store_piece(float* dst, int heads, const Running<D, HN>& r) {
  constexpr int VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int h = 0; h < HN; ++h) {
    const int head = 2 * t + h;
    if (head >= heads) continue;
    float* o = dst + head * (D + 2);
    const float f = r.mw[h] == -INFINITY ? 0.f : ex2(r.mw[h] + kLift - r.m[h]) * kUnlift;
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) {
      float2* at = reinterpret_cast<float2*>(o + g * VD + 4 * i);
      at[0] = make_float2(r.acc[2 * i][h] * f, r.acc[2 * i][2 + h] * f);
      at[1] = make_float2(r.acc[2 * i + 1][h] * f, r.acc[2 * i + 1][2 + h] * f);
    }
    if (g == 0) {
      o[D] = r.m[h];
      o[D + 1] = r.l[h];
    }
  }
}

template <int D, int HN>
__global__ void __launch_bounds__(kThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap map, const DecodeParams p) {
  pdl_trigger();
  constexpr int TILE = Shape<D>::TILE, PAIR = 4 * TILE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int64_t s_before[kThreads + 1];  // pairs before each thread's rows
  __shared__ int64_t s_warp[kWarps];
  __shared__ int s_most[kWarps];
  __shared__ int2 s_row[kThreads];
  __shared__ PieceTag s_tag[kWarps][2];
  __shared__ __align__(8) uint64_t s_bar[kWarps][kMaxStages];
  __shared__ __align__(16) float s_scale[kWarps][kMaxStages][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vheads = p.kv_heads * p.groups;
  const int piece_floats = p.stored_heads * (D + 2);
  const int ring_bytes = p.stages * PAIR;
  uint8_t* ring = smem + (size_t)warp * ring_bytes;
  // Places of the CTA's pieces. A piece that ends inside its segment's share (slot 0) has one of its own, in
  // shared memory or in the workspace; one that ends the warp's share (slot 1) lies over the warp's ring,
  // which is empty by then.
  float* first_pieces = p.first != nullptr ? p.first + (int64_t)blockIdx.x * kWarps * piece_floats
                                           : reinterpret_cast<float*>(smem + (size_t)kWarps * ring_bytes);
  auto place = [&](int w, int slot) {
    return slot ? reinterpret_cast<float*>(smem + (size_t)w * ring_bytes) : first_pieces + w * piece_floats;
  };
  if (lane == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&s_bar[warp][i], 5);  // expected bytes, and four lanes' scales
    fence_barrier_init();
    s_tag[warp][0].row = s_tag[warp][1].row = -1;
  }
  pdl_wait();

  // ---- the stream: pairs before every thread's rows
  const int per = (p.num_items + kThreads - 1) / kThreads;
  const int2* rows = per == 1 ? s_row : nullptr;
  int longest;
  {
    int64_t mine = 0;
    int most = 0;
    bool bad = false;
    for (int b = threadIdx.x * per; b < min(p.num_items, (int)(threadIdx.x + 1) * per); ++b) {
      const int n = row_pairs(p, b, bad);
      mine += n;
      most = max(most, n);
      if (per == 1) s_row[b] = make_int2(n > 0 ? p.item_pos[b] : -1, p.item_slot[b]);
    }
    if (bad && blockIdx.x == 0) set_error(p.status, CDB_ERR_INDEX);
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    most = __reduce_max_sync(kFull, most);
    if (lane == 31) s_warp[warp] = x, s_most[warp] = most;
    __syncthreads();
    int64_t base = 0, all = 0;
    longest = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) base += s_warp[i];
      all += s_warp[i];
      longest = max(longest, s_most[i]);
    }
    s_before[threadIdx.x] = base + x - mine;
    if (threadIdx.x == 0) s_before[kThreads] = all;
    __syncthreads();
  }
  const int64_t total = s_before[kThreads] * vheads;
  const int64_t even = quotient(total + gridDim.x - 1, gridDim.x);
  const int64_t share = even > p.min_share ? even : p.min_share;
  int64_t begin = share * blockIdx.x, end = begin + share < total ? begin + share : total;
  if (rows != nullptr && (int64_t)p.num_items * vheads <= gridDim.x && longest <= p.whole_pairs &&
      (longest <= 2 * kWarps || 2 * even >= longest)) {
    // Few short segments: a CTA for each, so that none has to meet another's piece in the workspace, unless
    // cutting them would leave a CTA less than half of one. Measured (16 heads of 128, from a graph), whole against
    // cut: 1 row of 700 positions 11.2 us (12.7), 8 of 700 11.3 (13.9), 9 of 1400 14.6 (19.1); 1 of 1400 14.4 (12.3),
    // 2 of 1400 14.4 (12.1), 1 of 3000 21.1 (13.7).
    const int row = blockIdx.x / vheads, vh = blockIdx.x - row * vheads;
    if (row >= p.num_items) return;
    const int n = s_row[row].x < 0 ? 0 : s_row[row].x / (2 * kBlock) + 1;
    begin = s_before[row] * vheads + (int64_t)vh * n;
    end = begin + n;
  }
  if (begin >= end) return;  // uniform over the CTA
  const int64_t wshare = quotient(end - begin + kWarps - 1, kWarps);
  const int64_t wbegin = begin + wshare * warp;
  const int count = (int)((wbegin + wshare < end ? wbegin + wshare : end) - wbegin);  // this warp's pairs, if > 0

  if (count > 0) {
    // the row that holds pair wbegin
    Cursor c;
    // the last of the threads whose rows begin at or before it, found by two looks of the warp
    static_assert(kThreads % 32 == 0 && kThreads / 32 <= 32, "32 samples, then the stretch between two");
    constexpr int STRETCH = kThreads / 32;
    const unsigned far = __ballot_sync(kFull, s_before[lane * STRETCH] * vheads <= wbegin);
    const int near = (31 - __clz(far)) * STRETCH;
    const unsigned in = __ballot_sync(kFull, lane < STRETCH && s_before[near + lane] * vheads <= wbegin);
    const int lo = near + 31 - __clz(in);
    int64_t at = wbegin - s_before[lo] * vheads;
    c.row = lo * per;
    load_row(p, rows, c);
    while (at >= (int64_t)c.pairs * vheads) {
      at -= (int64_t)c.pairs * vheads;
      ++c.row;
      load_row(p, rows, c);
    }
    const int vh = (int)quotient(at, c.pairs);
    c.pair = (int)(at - (int64_t)vh * c.pairs);
    c.kvh = p.groups == 1 ? vh : vh / p.groups;
    c.grp = vh - c.kvh * p.groups;

    uint32_t qraw[D / 8];
    fetch_q<D>(p, c, qraw);  // before the pages, which would keep it waiting
    const int v_tiles = p.num_blocks * p.kv_heads;
    const uint32_t ring_u = smem_u32(ring), bar_u = smem_u32(&s_bar[warp][0]), scale_u = smem_u32(&s_scale[warp][0][0]);
    Cursor ahead = c;
    int issued = 0, put = 0;
    // Lane i holds the block id of page i of a window of 32 pages of the issuing cursor's row.
    int win_row = -1, win_first = 0, win_id = -1;
    auto issue = [&]() {
      const int page = 2 * ahead.pair, first = page & ~31;
      if (ahead.row != win_row || first != win_first) {
        win_row = ahead.row;
        win_first = first;
        win_id = first + lane <= ahead.pos / kBlock ? p.block_table[(int64_t)ahead.slot * p.bt_stride + first + lane]
                                                     : INT32_MIN;  // behind the row's last page
      }
      // lane 0: K of the first page, 1: its V, 2 and 3: the second's
      const int id = __shfl_sync(kFull, win_id, (page & 31) + ((lane >> 1) & 1));
      const bool ok = id >= 0 && id < p.num_blocks;
      const int known = __popc(__ballot_sync(kFull, ok && lane < 4));
      const uint32_t bar = bar_u + put * 8;
      if (lane == 0) mbar_arrive_expect_tx(&s_bar[warp][put], known * TILE);
      __syncwarp();
      if (lane < 4) {
        const int tile = (lane & 1 ? v_tiles : 0) + id * p.kv_heads + ahead.kvh;
        if (ok) {
          const uint32_t dst = ring_u + put * PAIR + lane * TILE;
          if (Shape<D>::SWIZZLED) tensor_load(dst, &map, tile * kBlock, bar);
          else bulk_load(dst, p.codes + (int64_t)tile * TILE, TILE, bar);
          async_copy4(scale_u + put * 16 + lane * 4, p.scales + tile);
          async_arrive(bar);
        } else {
          if (id != INT32_MIN) set_error(p.status, CDB_ERR_INDEX);
          s_scale[warp][put][lane] = -1.f;
          mbar_arrive(&s_bar[warp][put]);
        }
      }
      put = put + 1 == p.stages ? 0 : put + 1;
      if (++issued < count) advance(p, rows, ahead);
    };
    for (int i = 0; i < p.stages && issued < count; ++i) issue();

    Running<D, HN> r;
    uint32_t qf[Shape<D>::KS][2];
    float factor[HN];
    int first = 0, get = 0;
    uint32_t phase = 0;
    bool fresh = true;
    for (int i = 0; i < count; ++i) {
      if (fresh) {
        first = c.pair;
        if (i > 0) fetch_q<D>(p, c, qraw);
        convert_q<D, HN>(p, qraw, qf, factor);
        r.clear();
      }
      if (!__all_sync(kFull, mbar_wait(&s_bar[warp][get], phase, p.status))) {
        for (int j = i + 1; j < issued; ++j) {  // a copy that never came: the error is recorded; wait for the others
          get = get + 1 == p.stages ? (phase ^= 1u, 0) : get + 1;
          mbar_wait(&s_bar[warp][get], phase, p.status);
        }
        break;
      }
      const float4 sc = *reinterpret_cast<const float4*>(&s_scale[warp][get][0]);
      const bool seg_end = c.pair + 1 == c.pairs;
      pair_step<D, HN>(ring + get * PAIR, sc, seg_end ? (c.pos & (2 * kBlock - 1)) + 1 : 2 * kBlock, qf, factor, r);
      get = get + 1 == p.stages ? (phase ^= 1u, 0) : get + 1;
      __syncwarp();
      if (issued < count) issue();
      fresh = seg_end;
      if (seg_end || i + 1 == count) {
#pragma unroll
        for (int h = 0; h < HN; ++h) {
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 4);
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 8);
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 16);
        }
        if (seg_end && first == 0) {
          write_out<D, HN>(p, c, r);
        } else {
          const int slot = first == 0 ? 1 : 0;  // a piece that begins its segment is this warp's last
          store_piece<D, HN>(place(warp, slot), p.stored_heads, r);
          if (lane == 0) {
            PieceTag tag;
            tag.row = c.row, tag.kvh = c.kvh, tag.grp = c.grp;
            tag.first = first, tag.last = c.pair + 1, tag.pairs = c.pairs;
            s_tag[warp][slot] = tag;
          }
        }
      }
      if (i + 1 < count) advance(p, rows, c);
    }
  }
  __syncthreads();

  // ---- join the pieces. Every warp sees which pieces belong together (lane j holds the tag of piece j); head h
  // of a segment falls to the warp h places after the one that its first piece comes from.
  static_assert(2 * kWarps <= 32, "a lane per piece");
  const PieceTag tag = s_tag[lane < 2 * kWarps ? lane >> 1 : 0][lane & 1];
  const bool used = lane < 2 * kWarps && tag.row >= 0;
  const int64_t key = used ? ((int64_t)tag.row * p.kv_heads + tag.kvh) * p.groups + tag.grp : -1 - lane;
  const unsigned group = __match_any_sync(kFull, key);
  unsigned leaders = __ballot_sync(kFull, used && (group & ((1u << lane) - 1u)) == 0u);
  if (p.stored_heads == 1) leaders &= 3u << (2 * warp);
  for (; leaders; leaders &= leaders - 1) {
    const int lead = __ffs(leaders) - 1;
    int h = warp - (lead >> 1);
    if (h < 0) h += kWarps;
    if (h >= p.stored_heads) continue;
    const unsigned members = __shfl_sync(kFull, group, lead);
    const int row = __shfl_sync(kFull, tag.row, lead), kvh = __shfl_sync(kFull, tag.kvh, lead);
    const int grp = __shfl_sync(kFull, tag.grp, lead), pairs = __shfl_sync(kFull, tag.pairs, lead);
    const int first = __shfl_sync(kFull, tag.first, lead), last = __shfl_sync(kFull, tag.last, 31 - __clz(members));
    if (grp * kGroup + h >= p.heads_per_kv) continue;
    const bool mine = (members >> lane) & 1u;
    const float* piece = mine ? place(lane >> 1, lane & 1) + h * (D + 2) : nullptr;
    const float pm = mine ? piece[D] : -INFINITY;
    float m = warp_max(pm);
    const float pf = pm == -INFINITY ? 0.f : ex2(pm - m);
    float l = warp_sum(mine ? piece[D + 1] * pf : 0.f);
    float o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
    const int end = 32 - __clz(members);
#pragma unroll 2
    for (int j = lead; j < end; ++j) {
      const float f = __shfl_sync(kFull, pf, j);
      if (!((members >> j) & 1u)) continue;
      const float* src = place(j >> 1, j & 1) + h * (D + 2) + lane;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] += src[i * 32] * f;
    }
    if (first != 0 || last != pairs) {
      // The segment goes on in other CTAs, which follow from its first pair's place in the stream. This CTA's
      // piece goes to the workspace; whoever is last adds all of them up, in CTA order.
      int64_t before = s_before[row / per];
      for (int b = row / per * per; b < row; ++b) {
        bool bad = false;
        before += row_pairs(p, b, bad);
      }
      const int64_t seg0 = before * vheads + (int64_t)(kvh * p.groups + grp) * pairs;
      const int c0 = (int)quotient(seg0, share), c1 = (int)quotient(seg0 + pairs - 1, share);
      const int64_t head_floats = D + 2;
      float* dst = p.parts + ((int64_t)blockIdx.x * 2 + (first > 0 ? 0 : 1)) * piece_floats + h * head_floats;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) __stcg(dst + i * 32 + lane, o[i]);
      if (lane == 0) {
        __stcg(dst + D, m);
        __stcg(dst + D + 1, l);
      }
      __threadfence();
      __syncwarp();
      int arrived = 0;
      if (lane == 0) arrived = atomicAdd(p.counters + c0 * kGroup + h, 1);
      arrived = __shfl_sync(kFull, arrived, 0);
      if (arrived != c1 - c0) continue;
      __threadfence();
      if (lane == 0) p.counters[c0 * kGroup + h] = 0;  // as the next launch expects it
      // the segment begins in c0's second place and goes on in the others' first
      auto part_of = [&](int cta) {
        return p.parts + ((int64_t)cta * 2 + (cta == c0 ? 1 : 0)) * piece_floats + h * head_floats;
      };
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
#pragma unroll 1
      for (int c = c0; c <= c1; c += 32) {  // 32 pieces at a time
        const bool on = c + lane <= c1;
        const float qm = on ? __ldcg(part_of(c + lane) + D) : -INFINITY;
        const float ql = on ? __ldcg(part_of(c + lane) + D + 1) : 0.f;
        const float nm = fmaxf(m, warp_max(qm));
        const float down = m == -INFINITY ? 0.f : ex2(m - nm), qf2 = qm == -INFINITY ? 0.f : ex2(qm - nm);
        l = l * down + warp_sum(ql * qf2);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= down;
        m = nm;
        const int n = min(32, c1 - c + 1);
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
          const float f = __shfl_sync(kFull, qf2, j);
          const float* src = part_of(c + j) + lane;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) o[i] += __ldcg(src + i * 32) * f;
        }
      }
    }
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    __nv_bfloat16* dst = p.out + (int64_t)row * p.out_stride + (int64_t)(kvh * p.heads_per_kv + grp * kGroup + h) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dst[i * 32 + lane] = f_to_bf16(o[i] * f);
  }
}

constexpr int kSmemLimit = 218 * 1024;  // dynamic, beside 8 KB of static shared memory

template <int D, int HN>
static int launch_decode(DecodeParams p, int num_ctas, cudaStream_t st) {
  CUtensorMap map = {};
  if (Shape<D>::SWIZZLED) {  // this layer's tiles, K then V, as rows of D bytes
    EncodeFn encode = tensor_map_encoder();
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)2 * p.num_blocks * p.kv_heads * kBlock};
    const cuuint64_t strides[1] = {(cuuint64_t)D};
    const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)kBlock}, ones[2] = {1, 1};
    if (encode == nullptr ||
        encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p.codes), dims, strides, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return CDB_ERR_TMA_ENCODE;
  }
  // Two pairs a warp in flight at least; first pieces that do not fit beside them go to the workspace.
  constexpr int RING = kWarps * 4 * Shape<D>::TILE;
  const int pieces = kWarps * p.stored_heads * (D + 2) * 4;
  const bool inside = 1024 + 2 * RING + pieces <= kSmemLimit;
  if (inside) p.first = nullptr;
  p.stages = (kSmemLimit - 1024 - (inside ? pieces : 0)) / RING;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int smem = 1024 + p.stages * RING + (inside ? pieces : 0);
  auto kernel = decode_kernel<D, HN>;
  if (allow_shared(reinterpret_cast<const void*>(kernel), kSmemLimit) != cudaSuccess) return CDB_ERR_CUDA;
  return launch_pdl(kernel, dim3(num_ctas), dim3(kThreads), smem, st, map, p) == cudaSuccess ? CDB_OK
                                                                                                : CDB_ERR_CUDA;
}

}  // namespace kv8
}  // namespace cdb

extern "C" int cdb_kv8_decode_counters(int num_ctas) { return num_ctas > 0 ? num_ctas * cdb::kv8::kGroup : 0; }

extern "C" int64_t cdb_kv8_decode_workspace_floats(int num_ctas, int head_dim) {
  if (num_ctas <= 0 || head_dim <= 0) return 0;
  return (int64_t)num_ctas * (2 + cdb::kv8::kWarps) * cdb::kv8::kGroup * (head_dim + 2);
}

extern "C" int cdb_kv8_decode_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                        const void* codes, const float* scales, int num_cache_layers, int cache_layer,
                                        int num_blocks, const int32_t* block_table, int64_t block_table_stride,
                                        int table_rows, int table_width, const int32_t* item_slot,
                                        const int32_t* item_pos, int num_items, int num_heads, int num_kv_heads,
                                        int head_dim, float scale, int num_ctas, float* workspace,
                                        int64_t workspace_floats, int32_t* counters, int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::kv8;
  if (codes == nullptr || scales == nullptr || (reinterpret_cast<uintptr_t>(codes) & 15) || cache_layer < 0 ||
      cache_layer >= num_cache_layers || num_blocks <= 0 || num_items < 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0 || num_ctas <= 0 || !(scale > 0.f) ||
      scale > 1e30f)
    return CDB_ERR_INVALID_ARGUMENT;
  if ((int64_t)num_blocks * num_kv_heads * 2 * kBlock > 0x7fffffff) return CDB_ERR_UNSUPPORTED;  // tile rows are int32
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_stride & 7) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (out_stride & 7))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_items == 0) return CDB_OK;
  if (q == nullptr || out == nullptr || block_table == nullptr || item_slot == nullptr || item_pos == nullptr ||
      workspace == nullptr || counters == nullptr ||
      workspace_floats < cdb_kv8_decode_workspace_floats(num_ctas, head_dim))
    return CDB_ERR_INVALID_ARGUMENT;
  DecodeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  const int64_t tiles = (int64_t)num_blocks * num_kv_heads * 2 * cache_layer;
  p.codes = static_cast<const uint8_t*>(codes) + tiles * kBlock * head_dim;
  p.scales = scales + tiles;
  p.num_blocks = num_blocks;
  p.kv_heads = num_kv_heads;
  p.heads_per_kv = num_heads / num_kv_heads;
  p.groups = (p.heads_per_kv + kGroup - 1) / kGroup;
  p.stored_heads = p.heads_per_kv < kGroup ? p.heads_per_kv : kGroup;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.num_items = num_items;
  p.scale_log2 = scale * kLog2e;
  p.min_share = kWarps / 2;  // 1, 6, 12, 24 pairs: 12.4, 12.3, 12.9, 14.2 us for one row of 1400 positions
  p.whole_pairs = 4 * kWarps;
  p.stages = 0;
  p.parts = workspace;
  p.first = workspace + (int64_t)num_ctas * 2 * p.stored_heads * (head_dim + 2);
  p.counters = counters;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.heads_per_kv == 1) {
    if (head_dim == 128) return launch_decode<128, 1>(p, num_ctas, st);
    if (head_dim == 96) return launch_decode<96, 1>(p, num_ctas, st);
    return launch_decode<64, 1>(p, num_ctas, st);
  }
  if (head_dim == 128) return launch_decode<128, 2>(p, num_ctas, st);
  if (head_dim == 96) return launch_decode<96, 2>(p, num_ctas, st);
  return launch_decode<64, 2>(p, num_ctas, st);
}
