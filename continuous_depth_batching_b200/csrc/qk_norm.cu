// RMS norms of each head's query and key, the position rotation and the append to the bf16 paged cache, in
// one pass over the projection's rows.
//
// y = x * rsqrt(mean(x^2) + eps) * w over a head's D values, then the rotation of a pair (a, b) of y by its
// position's angle: (a c - b s, b c + a s). All of it in fp32, rounded once, to bf16, as it is stored; values
// are copied.
//
// A head is a group of 8 or 16 lanes with 16 bytes each, so its sum of squares takes three or four shuffles
// and a pair's other half (D / 2 further on, another lane's) four of packed values. A warp takes one row's heads, or a
// slice of them where there are few rows: position, block id, angles and weights are the same for all of a row's
// heads, so a lane loads its part of them once and multiplies the last two: a value costs a product with w c, one of
// its partner with the partner's w s, and one with the norm. Heads of q come first, then k's, then the values, which
// are only copied; four heads of a group are in flight at a time.
//
// Everything is read and written once: bound by HBM over many rows, and by how well their warps fill it. 5411 rows of 32 +
// 2 x 8 heads of 128 take 29.1 us from a graph for 118 MB, 18 of them at 6.6 TB/s: a warp a row is 1353 CTAs on 888 places
// (80 registers leave 24 warps an SM), one wave and a half, and a warp's next heads are loaded when the last are stored. 1643
// rows of 55 + 2 x 55 heads of 96, interleaved pairs: 9.4 us for 48 MB, 7.3 at that rate. Over few rows it is a
// chain of three latencies (position, block id and angles, stores): 80 rows of 16 + 2 x 16 heads, 3.1 us.
#include "cdb_common.cuh"

namespace cdb {
namespace qknorm {

constexpr int kThreads = 128;
constexpr int kBlock = 16;  // tokens of one cache block
constexpr int kDepth = 4;   // heads of a group in flight

struct Params {
  const __nv_bfloat16* qkv;
  int64_t qkv_stride;
  __nv_bfloat16* q_out;  // null: q is left alone
  int64_t q_out_stride;
  __nv_bfloat16* keys;  // this cache layer's; values follow kv_rows rows later
  int64_t kv_rows;
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int32_t* item_slot;
  const int32_t* item_pos;
  const __nv_bfloat16* q_weight;
  const __nv_bfloat16* k_weight;
  const void* rope_cos;
  const void* rope_sin;
  int rope_rows;
  float eps;
  int num_items, heads, kv_heads;
  int slices;  // warps of a row
  int32_t* status;
};

__device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
  v[0] = bf16lo(w.x), v[1] = bf16hi(w.x), v[2] = bf16lo(w.y), v[3] = bf16hi(w.y);
  v[4] = bf16lo(w.z), v[5] = bf16hi(w.z), v[6] = bf16lo(w.w), v[7] = bf16hi(w.w);
}

template <int D, int MODE>
__global__ void __launch_bounds__(kThreads, 6) qk_norm_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  constexpr int LANES = D / 8;                // lanes that hold a head
  constexpr int GROUP = LANES <= 8 ? 8 : 16;  // lanes of a group (4 of 16 idle at 96)
  constexpr int GROUPS = 32 / GROUP;          // heads of a warp at a time
  const int lane = threadIdx.x & 31, c = lane % GROUP, group = lane / GROUP;
  const bool lane_on = c < LANES;
  const int at = lane_on ? c * 8 : 0;
  const bool lower = c < LANES / 2;
  const int other = lower ? c + LANES / 2 : c - LANES / 2;  // the lane with the pair's other half
  const int64_t task = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int row = (int)(task / p.slices), slice = (int)(task - (int64_t)row * p.slices);
  if (row >= p.num_items) return;
  const int pos = p.item_pos[row], slot = p.item_slot[row];
  if (pos < 0) return;
  if (slot < 0 || slot >= p.bt_rows || pos / kBlock >= p.bt_width || (MODE != 0 && pos >= p.rope_rows)) {
    if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
    return;
  }
  const int64_t id = p.block_table[(int64_t)slot * p.bt_stride + pos / kBlock];
  float cv[8], sv[8];  // cosines, and sines with the partner's sign
  if (MODE == 1) {     // bf16 [positions][D]
    unpack(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.rope_cos) + (int64_t)pos * D + at), cv);
    unpack(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.rope_sin) + (int64_t)pos * D + at), sv);
#pragma unroll
    for (int k = 0; k < 8; ++k) sv[k] = lower ? -sv[k] : sv[k];
  } else if (MODE == 2) {  // fp32 [positions][D / 2]
    const float4 cw = *reinterpret_cast<const float4*>(static_cast<const float*>(p.rope_cos) + (int64_t)pos * (D / 2) + at / 2);
    const float4 sw = *reinterpret_cast<const float4*>(static_cast<const float*>(p.rope_sin) + (int64_t)pos * (D / 2) + at / 2);
    cv[0] = cv[1] = cw.x, cv[2] = cv[3] = cw.y, cv[4] = cv[5] = cw.z, cv[6] = cv[7] = cw.w;
    sv[0] = -sw.x, sv[1] = sw.x, sv[2] = -sw.y, sv[3] = sw.y, sv[4] = -sw.z, sv[5] = sw.z, sv[6] = -sw.w, sv[7] = sw.w;
  }
  if (id < 0 || (id + 1) * kBlock > p.kv_rows) {
    if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
    return;
  }
  const __nv_bfloat16* src = p.qkv + (int64_t)row * p.qkv_stride + at;
  const int64_t kv_cols = (int64_t)p.kv_heads * D;
  __nv_bfloat16* keys = p.keys + (id * kBlock + pos % kBlock) * kv_cols + at;
  const int q_steps = (p.heads + GROUPS - 1) / GROUPS, k_steps = (p.kv_heads + GROUPS - 1) / GROUPS;
  const int per = (q_steps + 2 * k_steps + p.slices - 1) / p.slices;

  // `heads` heads from `from` on to `to`, of which this slice takes steps [a, b)
  auto rotate = [&](const __nv_bfloat16* weight, const __nv_bfloat16* from, __nv_bfloat16* to, int heads, int a, int b) {
    if (a >= b) return;
    float wc[8], ws[8];
    unpack(*reinterpret_cast<const uint4*>(weight + at), wc);
    if (MODE == 1) unpack(*reinterpret_cast<const uint4*>(weight + (lane_on ? other * 8 : 0)), ws);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (MODE == 1) ws[k] *= sv[k];
      if (MODE == 2) ws[k] = wc[k ^ 1] * sv[k];
    }
    if (MODE != 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) wc[k] *= cv[k];
    }
    for (int s = a; s < b; s += kDepth) {
      uint4 x[kDepth];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        const int h = (s + i) * GROUPS + group;
        x[i] = s + i < b && h < heads && lane_on ? __ldcg(reinterpret_cast<const uint4*>(from + (int64_t)h * D))
                                                 : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        if (s + i >= b) break;  // (the same for the whole warp)
        const int h = (s + i) * GROUPS + group;
        float y[8], z[8];
        unpack(x[i], y);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = fmaf(y[k], y[k], sum);
#pragma unroll
        for (int o = GROUP / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = rsqrtf(sum * (1.f / D) + p.eps);
        if (MODE == 1)
          unpack(make_uint4(__shfl_sync(0xffffffffu, x[i].x, other, GROUP), __shfl_sync(0xffffffffu, x[i].y, other, GROUP),
                            __shfl_sync(0xffffffffu, x[i].z, other, GROUP), __shfl_sync(0xffffffffu, x[i].w, other, GROUP)),
                 z);
        // (scaled first: a product of large values and weights need not overflow before the norm)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          y[k] *= inv;
          if (MODE == 1) z[k] *= inv;
        }
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          float lo = y[k] * wc[k], hi = y[k + 1] * wc[k + 1];
          if (MODE != 0) {
            lo = fmaf(MODE == 1 ? z[k] : y[k + 1], ws[k], lo);
            hi = fmaf(MODE == 1 ? z[k + 1] : y[k], ws[k + 1], hi);
          }
          w[k / 2] = pack_bf16x2(lo, hi);
        }
        if (h < heads && lane_on)
          *reinterpret_cast<uint4*>(to + (int64_t)h * D) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };
  const int s0 = slice * per, s1 = s0 + per, k_end = q_steps + k_steps, v_end = k_end + k_steps;
  if (p.q_out != nullptr)
    rotate(p.q_weight, src, p.q_out + (int64_t)row * p.q_out_stride + at, p.heads, min(s0, q_steps), min(s1, q_steps));
  rotate(p.k_weight, src + (int64_t)p.heads * D, keys, p.kv_heads, min(max(s0, q_steps), k_end) - q_steps,
         min(max(s1, q_steps), k_end) - q_steps);
  const __nv_bfloat16* values = src + (int64_t)(p.heads + p.kv_heads) * D;
  __nv_bfloat16* to = keys + p.kv_rows * kv_cols;
  const int v1 = min(s1, v_end) - k_end;
  for (int s = max(s0, k_end) - k_end; s < v1; s += kDepth) {
    uint4 x[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int h = (s + i) * GROUPS + group;
      if (s + i < v1 && h < p.kv_heads && lane_on) x[i] = __ldcg(reinterpret_cast<const uint4*>(values + (int64_t)h * D));
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int h = (s + i) * GROUPS + group;
      if (s + i < v1 && h < p.kv_heads && lane_on) *reinterpret_cast<uint4*>(to + (int64_t)h * D) = x[i];
    }
  }
}

template <int D>
static int launch(const Params& p, int mode, cudaStream_t st) {
  const int64_t warps = (int64_t)p.num_items * p.slices;
  const dim3 grid((unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)));
  auto* kernel = mode == 0 ? qk_norm_kernel<D, 0> : mode == 1 ? qk_norm_kernel<D, 1> : qk_norm_kernel<D, 2>;
  return launch_pdl(kernel, grid, dim3(kThreads), 0, st, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

}  // namespace qknorm
}  // namespace cdb

extern "C" int cdb_qk_norm_rope_append(const void* qkv, int64_t qkv_stride, void* q_out, int64_t q_out_stride,
                                       void* kv_base, int num_cache_layers, int64_t kv_rows, int cache_layer,
                                       const int32_t* block_table, int64_t block_table_stride, int table_rows,
                                       int table_width, const int32_t* item_slot, const int32_t* item_pos,
                                       const void* q_weight, const void* k_weight, int rope_mode, const void* rope_cos,
                                       const void* rope_sin, int rope_rows, float eps, int num_items, int num_heads,
                                       int num_kv_heads, int head_dim, int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::qknorm;
  auto off16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  if (cache_layer < 0 || cache_layer >= num_cache_layers || kv_rows < kBlock || num_items < 0 || num_heads <= 0 ||
      num_kv_heads <= 0 || table_rows < 0 || table_width < 0 || rope_mode < 0 || rope_mode > 2 || rope_rows < 0 ||
      !(eps >= 0.f) || eps > 3e38f)
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  // (places within a row and a CTA's heads are counted in 32 bits)
  if ((int64_t)num_heads + 2 * (int64_t)num_kv_heads > (1 << 20)) return CDB_ERR_UNSUPPORTED;
  if (off16(qkv) || (qkv_stride & 7) || off16(q_out) || (q_out_stride & 7) || off16(kv_base) || off16(q_weight) ||
      off16(k_weight) || off16(rope_cos) || off16(rope_sin))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_items == 0) return CDB_OK;
  if (qkv == nullptr || kv_base == nullptr || block_table == nullptr || item_slot == nullptr || item_pos == nullptr ||
      q_weight == nullptr || k_weight == nullptr || (rope_mode != 0 && (rope_cos == nullptr || rope_sin == nullptr)))
    return CDB_ERR_INVALID_ARGUMENT;
  Params p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.qkv_stride = qkv_stride;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_out_stride = q_out_stride;
  p.keys = static_cast<__nv_bfloat16*>(kv_base) + 2 * (int64_t)cache_layer * kv_rows * num_kv_heads * head_dim;
  p.kv_rows = kv_rows;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
  p.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
  p.rope_cos = rope_cos;
  p.rope_sin = rope_sin;
  p.rope_rows = rope_rows;
  p.eps = eps;
  p.num_items = num_items;
  p.heads = num_heads;
  p.kv_heads = num_kv_heads;
  // A warp's heads take a round of memory latency each kDepth steps, so few rows are cut into as many slices as leave each
  // one round; many rows fill the GPU by themselves.
  const int groups = head_dim == 64 ? 4 : 2;
  const int steps = (num_heads + groups - 1) / groups + 2 * ((num_kv_heads + groups - 1) / groups);
  const int most = (steps + kDepth - 1) / kDepth, want = 148 * 24 / num_items;
  p.slices = want < 1 ? 1 : want < most ? want : most;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch<128>(p, rope_mode, st);
  if (head_dim == 96) return launch<96>(p, rope_mode, st);
  return launch<64>(p, rope_mode, st);
}
