// RMS norms of each head's query and key, the position rotation and the append to the bf16 paged cache, in
// one pass over the projection's rows.
//
// y = x * rsqrt(mean(x^2) + eps) * w over a head's D values, then the rotation of a pair (a, b) of y by its
// position's angle: (a c - b s, b c + a s). All of it in fp32, rounded once, to bf16, as it is stored; values
// are copied.
//
// A head is a group of 8 or 16 lanes with 16 bytes each, so its sum of squares takes three or four shuffles
// and a pair's other half (D / 2 further on, another lane's) four. A group takes up to four heads at once, so that
// their loads are in flight together, over all of a row's heads before the next CTA's rows; a CTA takes several
// rows where they have few heads. Everything is read and written once: bound by HBM over many rows, by a chain of
// three latencies (position, block id and angles, stores) over few.
#include "cdb_common.cuh"

namespace cdb {
namespace qknorm {

constexpr int kThreads = 256;
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
  int num_items, heads, kv_heads, rows_per_cta;
  int32_t* status;
};

__device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
  v[0] = bf16lo(w.x), v[1] = bf16hi(w.x), v[2] = bf16lo(w.y), v[3] = bf16hi(w.y);
  v[4] = bf16lo(w.z), v[5] = bf16hi(w.z), v[6] = bf16lo(w.w), v[7] = bf16hi(w.w);
}

template <int D, int MODE>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  constexpr int LANES = D / 8;                 // lanes that hold a head
  constexpr int GROUP = LANES <= 8 ? 8 : 16;   // lanes of a group (4 of 16 idle at 96)
  constexpr int GROUPS = kThreads / GROUP;
  const int c = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
  const bool lane_on = c < LANES;
  const int at = lane_on ? c * 8 : 0;
  const int other = c < LANES / 2 ? c + LANES / 2 : c - LANES / 2;  // the lane with the pair's other half
  const int row0 = blockIdx.x * p.rows_per_cta;
  const int all = p.heads + 2 * p.kv_heads;
  const int units = min(p.rows_per_cta, p.num_items - row0) * all;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  float wq[8], wk[8];
  unpack(*reinterpret_cast<const uint4*>(p.q_weight + at), wq);
  unpack(*reinterpret_cast<const uint4*>(p.k_weight + at), wk);

  for (int u0 = 0; u0 < units; u0 += GROUPS * kDepth) {
    uint4 x[kDepth], cs[kDepth][MODE == 0 ? 1 : 2];
    __nv_bfloat16* dst[kDepth];
    int kind[kDepth];  // 0 query, 1 key, 2 value
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int u = u0 + i * GROUPS + group;
      dst[i] = nullptr;
      kind[i] = 2;
      x[i] = none;
      if (MODE != 0) cs[i][0] = cs[i][MODE == 0 ? 0 : 1] = none;
      if (u >= units) continue;
      const int r = u / all, h = u - r * all, row = row0 + r;
      const int pos = p.item_pos[row];
      if (pos < 0) continue;
      kind[i] = h < p.heads ? 0 : (h < p.heads + p.kv_heads ? 1 : 2);
      if (kind[i] == 0 && p.q_out == nullptr) continue;
      const int slot = p.item_slot[row];
      int64_t cache_row = -1;
      if (slot >= 0 && slot < p.bt_rows && pos / kBlock < p.bt_width && (MODE == 0 || pos < p.rope_rows)) {
        const int64_t id = p.block_table[(int64_t)slot * p.bt_stride + pos / kBlock];
        if (id >= 0 && (id + 1) * kBlock <= p.kv_rows) cache_row = id * kBlock + pos % kBlock;
      }
      if (cache_row < 0) {
        if (c == 0) set_error(p.status, CDB_ERR_INDEX);
        continue;
      }
      if (kind[i] == 0)
        dst[i] = p.q_out + (int64_t)row * p.q_out_stride + h * D + at;
      else
        dst[i] = p.keys + ((kind[i] == 2 ? p.kv_rows : 0) + cache_row) * ((int64_t)p.kv_heads * D) +
                 (h - p.heads - (kind[i] == 2 ? p.kv_heads : 0)) * D + at;
      if (!lane_on) continue;
      x[i] = *reinterpret_cast<const uint4*>(p.qkv + (int64_t)row * p.qkv_stride + (int64_t)h * D + at);
      if (MODE == 1 && kind[i] != 2) {  // bf16 [positions][D]
        cs[i][0] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.rope_cos) + (int64_t)pos * D + at);
        cs[i][MODE == 0 ? 0 : 1] =
            *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.rope_sin) + (int64_t)pos * D + at);
      } else if (MODE == 2 && kind[i] != 2) {  // fp32 [positions][D / 2]
        cs[i][0] = *reinterpret_cast<const uint4*>(static_cast<const float*>(p.rope_cos) + (int64_t)pos * (D / 2) + at / 2);
        cs[i][MODE == 0 ? 0 : 1] =
            *reinterpret_cast<const uint4*>(static_cast<const float*>(p.rope_sin) + (int64_t)pos * (D / 2) + at / 2);
      }
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      float y[8];
      unpack(x[i], y);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum = fmaf(y[k], y[k], sum);
#pragma unroll
      for (int o = GROUP / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = rsqrtf(sum * (1.f / D) + p.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = y[k] * inv * (kind[i] == 0 ? wq[k] : wk[k]);
      if (MODE == 1) {
        float cv[8], sv[8];
        unpack(cs[i][0], cv);
        unpack(cs[i][MODE == 0 ? 0 : 1], sv);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float z = __shfl_sync(0xffffffffu, y[k], other, GROUP);
          y[k] = fmaf(y[k], cv[k], (c < LANES / 2 ? -z : z) * sv[k]);
        }
      } else if (MODE == 2) {
        const uint4 cw = cs[i][0], sw = cs[i][MODE == 0 ? 0 : 1];
        const float cv[4] = {__uint_as_float(cw.x), __uint_as_float(cw.y), __uint_as_float(cw.z), __uint_as_float(cw.w)};
        const float sv[4] = {__uint_as_float(sw.x), __uint_as_float(sw.y), __uint_as_float(sw.z), __uint_as_float(sw.w)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = y[2 * k], b = y[2 * k + 1];
          y[2 * k] = fmaf(a, cv[k], -b * sv[k]);
          y[2 * k + 1] = fmaf(b, cv[k], a * sv[k]);
        }
      }
      if (dst[i] == nullptr || !lane_on) continue;
      *reinterpret_cast<uint4*>(dst[i]) =
          kind[i] == 2 ? x[i]
                       : make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                    pack_bf16x2(y[6], y[7]));
    }
  }
}

template <int D>
static int launch(const Params& p, int mode, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)p.num_items + p.rows_per_cta - 1) / p.rows_per_cta));
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
  const int group = head_dim == 64 ? 8 : 16, places = kThreads / group * kDepth;
  const int rows = places / (num_heads + 2 * num_kv_heads);
  p.rows_per_cta = rows > 1 ? rows : 1;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch<128>(p, rope_mode, st);
  if (head_dim == 96) return launch<96>(p, rope_mode, st);
  return launch<64>(p, rope_mode, st);
}
