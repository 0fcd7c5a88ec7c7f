// Decode attention over the 8-bit paged cache (layout in kv8.cuh): one query row per item, any
// number of query heads per kv head.
//
// Work. The pages of all (row, kv head, group of up to 8 query heads) segments, in that order, form
// one stream that is cut into equal shares, one per CTA, and each share into eight, one per warp: a
// long row is spread over the whole GPU and short rows are packed, by the positions that lie on the
// device. Each warp streams its pages through a ring of its own in shared memory (a page is two
// contiguous tiles, K and V, one bulk copy each), so no warp waits for another until its share ends.
//
// Mathematics. Per page, with K the 16 x D tile of codes: S = K q (tensor cores, f16 operands, fp32
// accumulators). Codes convert to f16 exactly, and q is divided by a power of two that brings its
// largest element to [1, 2), so that bf16's 8 significant bits fit f16; what f16 loses lies below
// 2^-24 of the row's largest element. x = S * (scale log2e 2^e s_k) in fp32. The softmax runs online
// in base 2: m is a maximum of x that only moves when x passes it by 8 (then l, the sum of 2^(x-m),
// is rescaled), and the weights of V, 2^(x-m) s_v, are taken relative to their own maximum M of
// x + log2 s_v, so that they fit f16 (at most 2^8; 2^-11 relative rounding each, averaged over the
// keys) whatever the blocks' scales are. O = V^T P (tensor cores again) in fp32.
//
// Pieces of a segment (m, l, o) meet in two steps: the warps of a CTA through shared memory, CTAs
// through the workspace, where the last one to arrive adds them up in CTA order. The result does not
// depend on which one that is.
#include "kv8.cuh"

namespace cdb {
namespace kv8 {

constexpr int kWarps = 8;
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
  int min_share;     // pages of one CTA's share, at least
  int stages;        // pages of a warp's ring
  int stored_heads;  // heads of a stored piece: min(heads_per_kv, kGroup)
  float* parts;      // [CTAs][2][stored_heads][D + 2]
  int32_t* counters;
  int32_t* status;
};

// Cached pages of row b; 0 for a padding row and for one whose indexes do not fit the table.
__device__ __forceinline__ int row_pages(const DecodeParams& p, int b, bool& bad) {
  const int pos = p.item_pos[b], slot = p.item_slot[b];
  if (pos < 0) return 0;
  if (slot < 0 || slot >= p.bt_rows || pos / kBlock >= p.bt_width) {
    bad = true;
    return 0;
  }
  return pos / kBlock + 1;
}

// A place in the page stream: page `page` of row `row`, virtual head `vh` (kv head * groups + group).
struct Cursor {
  int row, vh, page, pages, pos, slot;
};

__device__ __forceinline__ void load_row(const DecodeParams& p, Cursor& c) {
  bool bad = false;
  c.pages = row_pages(p, c.row, bad);
  c.pos = p.item_pos[c.row];
  c.slot = p.item_slot[c.row];
}

__device__ __forceinline__ void advance(const DecodeParams& p, Cursor& c, int vheads) {
  if (++c.page < c.pages) return;
  c.page = 0;
  if (++c.vh < vheads) return;
  c.vh = 0;
  do {
    if (++c.row >= p.num_items) return;  // the stream's end
    load_row(p, c);
  } while (c.pages == 0);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Where a piece lies in its segment, for the joins.
struct PieceTag {
  int row, vh;
  int first, last, pages;  // pages [first, last) of `pages`
};

template <int D>
struct Shape {
  static constexpr int KD = D / 4;        // dims of K that a lane multiplies: [t * KD, t * KD + KD) of rows g, g + 8
  static constexpr int VD = D / 8;        // dims of V that a lane multiplies: [g * VD, g * VD + VD) of 4 tokens
  static constexpr int KS = D / 16;       // k-steps of K q
  static constexpr int MT = D / 16;       // m-tiles of V^T P
  static constexpr int TILE = kBlock * D; // bytes of a K or V tile
};

// The running softmax of one segment piece and what a lane holds of V^T P: dims g * VD + 4 i + {0, 1, 2,
// 3} of heads 2t, 2t + 1 in acc[2i][0, 2], acc[2i + 1][0, 2] (head 2t) and [1, 3] (head 2t + 1).
template <int D>
struct Running {
  float acc[Shape<D>::MT][4];
  float m[2], mw[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < Shape<D>::MT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    m[0] = m[1] = mw[0] = mw[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
};

// q's rows of one segment as the B operand: head g of the group, dims [t * KD, (t + 1) * KD). e is the
// power of two that was divided out (for heads 2t and 2t + 1).
template <int D>
__device__ __forceinline__ void load_q(const DecodeParams& p, int row, int vh, uint32_t (&qf)[Shape<D>::KS][2],
                                       float (&factor)[2]) {
  constexpr int KD = Shape<D>::KD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = vh / p.groups, grp = vh - kvh * p.groups;
  const int in_kv = grp * kGroup + g;
  const bool on = in_kv < p.heads_per_kv;
  const __nv_bfloat16* src =
      p.q + (int64_t)row * p.q_stride + (int64_t)(kvh * p.heads_per_kv + (on ? in_kv : 0)) * D + t * KD;
  uint32_t w[KD / 2];
#pragma unroll
  for (int i = 0; i < KD / 8; ++i) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (on) v = *reinterpret_cast<const uint4*>(src + i * 8);
    w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
  }
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
  factor[0] = __shfl_sync(kFull, f, t * 8);  // lanes of head 2t, then 2t + 1
  factor[1] = __shfl_sync(kFull, f, t * 8 + 4);
}

// One page: `live` tokens of it count.
template <int D>
__device__ __forceinline__ void page_step(const uint8_t* k, const uint8_t* v, float sk, float sv, int live,
                                          const uint32_t (&qf)[Shape<D>::KS][2], const float (&factor)[2],
                                          Running<D>& r) {
  constexpr int KD = Shape<D>::KD, VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  {
    uint32_t ka[KD / 4], kb[KD / 4];
    const uint8_t* r0 = k + g * D + t * KD;
    const uint8_t* r1 = r0 + 8 * D;
#pragma unroll
    for (int i = 0; i < KD / 8; ++i) {
      const uint2 x = *reinterpret_cast<const uint2*>(r0 + i * 8), y = *reinterpret_cast<const uint2*>(r1 + i * 8);
      ka[2 * i] = x.x, ka[2 * i + 1] = x.y, kb[2 * i] = y.x, kb[2 * i + 1] = y.y;
    }
#pragma unroll
    for (int i = 0; i < KD / 4; ++i)
      mma_f16(s, cvt_e4m3x2_f16x2(ka[i] & 0xffffu), cvt_e4m3x2_f16x2(kb[i] & 0xffffu), cvt_e4m3x2_f16x2(ka[i] >> 16),
              cvt_e4m3x2_f16x2(kb[i] >> 16), qf[i][0], qf[i][1]);
  }
  // s[0], s[1]: token g, heads 2t, 2t + 1; s[2], s[3]: token g + 8
  const float ev = sv > 0.f ? __log2f(sv) : -126.f;
  float pw[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float f = factor[h] * sk;
    const float x0 = g < live ? s[h] * f : -INFINITY;
    const float x1 = g + 8 < live ? s[2 + h] * f : -INFINITY;
    float mx = fmaxf(x0, x1);
    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
    // m and M move only when passed by 8: the weights stay within 2^8
    if (mx > r.m[h] + 8.f) {
      r.l[h] *= ex2(r.m[h] - mx);
      r.m[h] = mx;
    }
    const bool up = mx + ev > r.mw[h] + 8.f;
    if (__any_sync(kFull, up)) {
      const float to = up ? mx + ev : r.mw[h];
      const float down = up ? ex2(r.mw[h] - to) : 1.f;
#pragma unroll
      for (int i = 0; i < Shape<D>::MT; ++i) r.acc[i][h] *= down, r.acc[i][2 + h] *= down;
      r.mw[h] = to;
    }
    const float p0 = x0 == -INFINITY ? 0.f : ex2(x0 - r.m[h]);
    const float p1 = x1 == -INFINITY ? 0.f : ex2(x1 - r.m[h]);
    r.l[h] += p0 + p1;
    pw[0][h] = x0 == -INFINITY ? 0.f : ex2(x0 + ev - r.mw[h]);
    pw[1][h] = x1 == -INFINITY ? 0.f : ex2(x1 + ev - r.mw[h]);
  }
  const uint32_t b0 = transpose8(pack_f16x2(pw[0][0], pw[0][1]));
  const uint32_t b1 = transpose8(pack_f16x2(pw[1][0], pw[1][1]));
  // V: tokens 2t, 2t + 1, 2t + 8, 2t + 9, dims [g * VD, (g + 1) * VD)
  uint32_t vw[4][VD / 4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
    const uint8_t* src = v + tok * D + g * VD;
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) vw[j][i] = *reinterpret_cast<const uint32_t*>(src + i * 4);
    if (tok >= live) {  // codes behind the row's end may be anything, NaN too
#pragma unroll
      for (int i = 0; i < VD / 4; ++i) vw[j][i] = 0u;
    }
  }
#pragma unroll
  for (int i = 0; i < VD / 4; ++i) {
    const uint32_t lo0 = __byte_perm(vw[0][i], vw[1][i], 0x5140), hi0 = __byte_perm(vw[0][i], vw[1][i], 0x7362);
    const uint32_t lo1 = __byte_perm(vw[2][i], vw[3][i], 0x5140), hi1 = __byte_perm(vw[2][i], vw[3][i], 0x7362);
    mma_f16(r.acc[2 * i], cvt_e4m3x2_f16x2(lo0 & 0xffffu), cvt_e4m3x2_f16x2(lo0 >> 16),
            cvt_e4m3x2_f16x2(lo1 & 0xffffu), cvt_e4m3x2_f16x2(lo1 >> 16), b0, b1);
    mma_f16(r.acc[2 * i + 1], cvt_e4m3x2_f16x2(hi0 & 0xffffu), cvt_e4m3x2_f16x2(hi0 >> 16),
            cvt_e4m3x2_f16x2(hi1 & 0xffffu), cvt_e4m3x2_f16x2(hi1 >> 16), b0, b1);
  }
}

// A finished segment's output, straight from a warp's registers (l already summed over the warp).
template <int D>
__device__ __forceinline__ void write_out(const DecodeParams& p, int row, int vh, const Running<D>& r) {
  constexpr int VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = vh / p.groups, grp = vh - kvh * p.groups;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int in_kv = grp * kGroup + 2 * t + h;
    if (in_kv >= p.heads_per_kv) continue;
    const float f = r.l[h] > 0.f ? ex2(r.mw[h] - r.m[h]) / r.l[h] : (r.l[h] == 0.f ? 0.f : r.l[h]);
    __nv_bfloat16* dst = p.out + (int64_t)row * p.out_stride + (int64_t)(kvh * p.heads_per_kv + in_kv) * D + g * VD;
#pragma unroll
    for (int i = 0; i < VD / 4; ++i)
      *reinterpret_cast<uint2*>(dst + i * 4) =
          make_uint2(pack_bf16x2(r.acc[2 * i][h] * f, r.acc[2 * i][2 + h] * f),
                     pack_bf16x2(r.acc[2 * i + 1][h] * f, r.acc[2 * i + 1][2 + h] * f));
  }
}

// A piece: per stored head D values of o = sum 2^(x-m) v, then m and l.
template <int D>
__device__ __forceinline__ void store_piece(float* dst, int heads, const Running<D>& r) {
  constexpr int VD = Shape<D>::VD;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int head = 2 * t + h;
    if (head >= heads) continue;
    float* o = dst + head * (D + 2);
    const float f = r.mw[h] == -INFINITY ? 0.f : ex2(r.mw[h] - r.m[h]);
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

template <int D>
__global__ void __launch_bounds__(kWarps * 32, 2) decode_kernel(const DecodeParams p) {
  pdl_trigger();
  constexpr int TILE = Shape<D>::TILE;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_before[kWarps * 32 + 1];  // pages before each thread's rows
  __shared__ int64_t s_warp[kWarps];
  __shared__ PieceTag s_tag[kWarps][2];
  __shared__ __align__(8) uint64_t s_bar[kWarps][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vheads = p.kv_heads * p.groups;
  const int piece_floats = p.stored_heads * (D + 2);
  uint8_t* ring = smem + (size_t)warp * p.stages * 2 * TILE;
  float* s_piece = reinterpret_cast<float*>(smem + (size_t)kWarps * p.stages * 2 * TILE);
  if (lane == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&s_bar[warp][i], 1);
    fence_barrier_init();
    s_tag[warp][0].row = s_tag[warp][1].row = -1;
  }
  pdl_wait();

  // ---- the page stream: pages before every thread's rows
  const int per = (p.num_items + kWarps * 32 - 1) / (kWarps * 32);
  {
    int64_t mine = 0;
    bool bad = false;
    for (int b = threadIdx.x * per; b < min(p.num_items, (int)(threadIdx.x + 1) * per); ++b) mine += row_pages(p, b, bad);
    if (bad && blockIdx.x == 0) set_error(p.status, CDB_ERR_INDEX);
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int64_t base = 0, all = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) base += s_warp[i];
      all += s_warp[i];
    }
    s_before[threadIdx.x] = base + x - mine;
    if (threadIdx.x == 0) s_before[kWarps * 32] = all;
    __syncthreads();
  }
  const int64_t total = s_before[kWarps * 32] * vheads;
  const int64_t even = (total + gridDim.x - 1) / gridDim.x;
  const int64_t share = even > p.min_share ? even : p.min_share;
  const int64_t begin = share * blockIdx.x, end = begin + share < total ? begin + share : total;
  const int64_t wshare = (end - begin + kWarps - 1) / kWarps;
  const int64_t wbegin = begin + wshare * warp;
  const int count = (int)((wbegin + wshare < end ? wbegin + wshare : end) - wbegin);  // this warp's pages, if > 0
  if (begin >= end) return;  // uniform over the CTA

  if (count > 0) {
    // the row that holds page wbegin
    Cursor c;
    int lo = 0, hi = kWarps * 32;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_before[mid] * vheads <= wbegin) lo = mid; else hi = mid;
    }
    int64_t at = wbegin - s_before[lo] * vheads;
    c.row = lo * per;
    load_row(p, c);
    while (at >= (int64_t)c.pages * vheads) {
      at -= (int64_t)c.pages * vheads;
      ++c.row;
      load_row(p, c);
    }
    c.vh = (int)(at / c.pages);
    c.page = (int)(at - (int64_t)c.vh * c.pages);

    const int64_t v_tiles = (int64_t)p.num_blocks * p.kv_heads;
    const uint32_t ring_u = smem_u32(ring);
    Cursor ahead = c;
    int issued = 0;
    // Lane i of the issuing window holds block ids of 32 pages of the cursor's row.
    int win_row = -1, win_first = 0, win_id = -1;
    auto issue = [&]() {
      const int first = ahead.page & ~31;
      if (ahead.row != win_row || first != win_first) {
        win_row = ahead.row;
        win_first = first;
        win_id = first + lane < ahead.pages ? p.block_table[(int64_t)ahead.slot * p.bt_stride + first + lane] : -1;
      }
      const int blk = __shfl_sync(kFull, win_id, ahead.page & 31);
      const int st = issued % p.stages;
      if (lane == 0) {
        if (blk >= 0 && blk < p.num_blocks) {
          const int64_t tile = (int64_t)blk * p.kv_heads + ahead.vh / p.groups;
          const uint32_t bar = smem_u32(&s_bar[warp][st]);
          mbar_arrive_expect_tx(&s_bar[warp][st], 2 * TILE);
          bulk_load(ring_u + st * 2 * TILE, p.codes + tile * TILE, TILE, bar);
          bulk_load(ring_u + st * 2 * TILE + TILE, p.codes + (v_tiles + tile) * TILE, TILE, bar);
        } else {
          set_error(p.status, CDB_ERR_INDEX);
          mbar_arrive(&s_bar[warp][st]);
        }
      }
      ++issued;
      if (issued < count) advance(p, ahead, vheads);
    };
    for (int i = 0; i < p.stages && issued < count; ++i) issue();

    Running<D> r;
    uint32_t qf[Shape<D>::KS][2];
    float factor[2];
    int first = c.page, seg_row = -1, seg_vh = -1;
    int own_row = -1, own_first = 0, own_id = -1;
    for (int i = 0; i < count; ++i) {
      if (c.row != seg_row || c.vh != seg_vh) {
        seg_row = c.row;
        seg_vh = c.vh;
        first = c.page;
        load_q<D>(p, c.row, c.vh, qf, factor);
        r.clear();
      }
      const int wf = c.page & ~31;
      if (c.row != own_row || wf != own_first) {
        own_row = c.row;
        own_first = wf;
        own_id = wf + lane < c.pages ? p.block_table[(int64_t)c.slot * p.bt_stride + wf + lane] : -1;
      }
      const int blk = __shfl_sync(kFull, own_id, c.page & 31);
      const int st = i % p.stages;
      const bool known = blk >= 0 && blk < p.num_blocks;
      float sk = 0.f, sv = 1.f;
      if (known) {
        const int64_t tile = (int64_t)blk * p.kv_heads + c.vh / p.groups;
        sk = p.scales[tile];
        sv = p.scales[v_tiles + tile];
      }
      if (!__all_sync(kFull, mbar_wait(&s_bar[warp][st], (i / p.stages) & 1, p.status))) {
        for (int j = i + 1; j < issued; ++j) mbar_wait(&s_bar[warp][j % p.stages], (j / p.stages) & 1, p.status);
        break;  // a copy that never came: the error is recorded, the copies in flight have been waited for
      }
      if (known) {
        const int live = c.page + 1 == c.pages ? (c.pos & (kBlock - 1)) + 1 : kBlock;
        page_step<D>(ring + st * 2 * TILE, ring + st * 2 * TILE + TILE, sk, sv, live, qf, factor, r);
      }
      __syncwarp();
      if (issued < count) issue();
      const bool seg_end = c.page + 1 == c.pages;
      if (seg_end || i + 1 == count) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 4);
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 8);
          r.l[h] += __shfl_xor_sync(kFull, r.l[h], 16);
        }
        if (seg_end && first == 0) {
          write_out<D>(p, c.row, c.vh, r);
        } else {
          const int slot = first == 0 ? 1 : 0;  // a piece that begins its segment is this warp's last
          store_piece<D>(s_piece + (warp * 2 + slot) * piece_floats, p.stored_heads, r);
          if (lane == 0) {
            PieceTag tag;
            tag.row = c.row, tag.vh = c.vh, tag.first = first, tag.last = c.page + 1, tag.pages = c.pages;
            s_tag[warp][slot] = tag;
          }
        }
      }
      if (i + 1 < count) advance(p, c, vheads);
    }
  }
  __syncthreads();

  // ---- join the pieces: warp w leads those segments whose first piece of this CTA is its own
  for (int slot = 0; slot < 2; ++slot) {
    const PieceTag lead = s_tag[warp][slot];
    if (lead.row < 0) continue;
    bool leads = true;
    for (int j = 0; j < warp * 2 + slot; ++j) {
      const PieceTag& o = s_tag[j >> 1][j & 1];
      leads = leads && !(o.row == lead.row && o.vh == lead.vh);
    }
    if (!leads) continue;
    int last = lead.last;
    unsigned members = 0;  // bit j: piece j belongs here
    for (int j = warp * 2 + slot; j < kWarps * 2; ++j) {
      const PieceTag& o = s_tag[j >> 1][j & 1];
      if (o.row == lead.row && o.vh == lead.vh) {
        members |= 1u << j;
        last = o.last;
      }
    }
    const bool whole = lead.first == 0 && last == lead.pages;
    const int kvh = lead.vh / p.groups, grp = lead.vh - kvh * p.groups;
    const int heads = min(kGroup, p.heads_per_kv - grp * kGroup);
    // stream places of the segment, to know the CTAs that share it
    const int pslot = lead.first > 0 ? 0 : 1;
    float* mine = p.parts + ((int64_t)blockIdx.x * 2 + pslot) * piece_floats;
    for (int h = 0; h < heads; ++h) {
      float m = -INFINITY;
      for (unsigned b = members; b; b &= b - 1) m = fmaxf(m, s_piece[(__ffs(b) - 1) * piece_floats + h * (D + 2) + D]);
      float l = 0.f, o[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
      for (unsigned b = members; b; b &= b - 1) {
        const float* src = s_piece + (__ffs(b) - 1) * piece_floats + h * (D + 2);
        const float f = src[D] == -INFINITY ? 0.f : ex2(src[D] - m);
        l += src[D + 1] * f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] += src[i * 32 + lane] * f;
      }
      if (whole) {
        const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        __nv_bfloat16* dst =
            p.out + (int64_t)lead.row * p.out_stride + (int64_t)(kvh * p.heads_per_kv + grp * kGroup + h) * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dst[i * 32 + lane] = f_to_bf16(o[i] * f);
      } else {
        float* dst = mine + h * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) __stcg(dst + i * 32 + lane, o[i]);
        if (lane == 0) {
          __stcg(dst + D, m);
          __stcg(dst + D + 1, l);
        }
      }
    }
    if (whole) continue;
    // The segment's first page in the stream, from this CTA's own place in it.
    int64_t before = s_before[lead.row / per];
    for (int b = lead.row / per * per; b < lead.row; ++b) {
      bool bad = false;
      before += row_pages(p, b, bad);
    }
    const int64_t seg0 = before * vheads + (int64_t)lead.vh * lead.pages;
    const int c0 = (int)(seg0 / share), c1 = (int)((seg0 + lead.pages - 1) / share);
    __threadfence();
    __syncwarp();
    int arrived = 0;
    if (lane == 0) arrived = atomicAdd(p.counters + c0, 1);
    arrived = __shfl_sync(kFull, arrived, 0);
    if (arrived != c1 - c0) continue;
    __threadfence();
    if (lane == 0) p.counters[c0] = 0;  // as the next launch expects it
    for (int h = 0; h < heads; ++h) {
      float m = -INFINITY;
      for (int cta = c0; cta <= c1; ++cta)
        m = fmaxf(m, __ldcg(p.parts + ((int64_t)cta * 2 + (cta == c0 ? 1 : 0)) * piece_floats + h * (D + 2) + D));
      float l = 0.f, o[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
      for (int cta = c0; cta <= c1; ++cta) {
        const float* src = p.parts + ((int64_t)cta * 2 + (cta == c0 ? 1 : 0)) * piece_floats + h * (D + 2);
        const float pm = __ldcg(src + D), pl = __ldcg(src + D + 1);
        const float f = pm == -INFINITY ? 0.f : ex2(pm - m);
        l += pl * f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] += __ldcg(src + i * 32 + lane) * f;
      }
      const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      __nv_bfloat16* dst =
          p.out + (int64_t)lead.row * p.out_stride + (int64_t)(kvh * p.heads_per_kv + grp * kGroup + h) * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) dst[i * 32 + lane] = f_to_bf16(o[i] * f);
    }
  }
}

constexpr int kSmemLimit = 113 * 1024;  // two CTAs share an SM's 228 KB

template <int D>
static int launch_decode(DecodeParams p, int num_ctas, cudaStream_t st) {
  const int pieces = kWarps * 2 * p.stored_heads * (D + 2) * 4;
  p.stages = 4;
  while (p.stages > 2 && kWarps * p.stages * 2 * Shape<D>::TILE + pieces > kSmemLimit - 4096) --p.stages;
  const int smem = kWarps * p.stages * 2 * Shape<D>::TILE + pieces;
  if (cudaFuncSetAttribute(decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return CDB_ERR_CUDA;
  launch_pdl(decode_kernel<D>, dim3(num_ctas), dim3(kWarps * 32), smem, st, p);
  return cudaPeekAtLastError() == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

}  // namespace kv8
}  // namespace cdb

extern "C" int64_t cdb_kv8_decode_workspace_floats(int num_ctas, int head_dim) {
  if (num_ctas <= 0 || head_dim <= 0) return 0;
  return (int64_t)num_ctas * 2 * cdb::kv8::kGroup * (head_dim + 2);
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
      num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0 || num_ctas <= 0)
    return CDB_ERR_INVALID_ARGUMENT;
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
  p.min_share = 8;
  p.stages = 0;
  p.parts = workspace;
  p.counters = counters;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_decode<128>(p, num_ctas, st);
  if (head_dim == 96) return launch_decode<96>(p, num_ctas, st);
  return launch_decode<64>(p, num_ctas, st);
}
