// Decode attention over the bf16 paged cache for requests that share a prompt.
//
// Every row by itself: a CTA per (row, head) reads the row's pages, a warp a page at a time, with a running
// maximum and sum; the warps' parts are joined at the end.
#include "cdb_common.cuh"

namespace cdb {
namespace prefix {

constexpr int kBlock = 16;
constexpr int kWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const __nv_bfloat16* keys;
  int64_t kv_rows;
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int32_t* item_slot;
  const int32_t* item_pos;
  int num_items, kv_heads, heads_per_kv;
  const int32_t* group_start;
  const int32_t* prefix_len;
  int num_groups;
  float scale_log2;
  int32_t* status;
};

template <int D>
__global__ void __launch_bounds__(kWarps * 32) decode_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  constexpr int PER = D / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][D];
  const int heads = p.kv_heads * p.heads_per_kv;
  const int item = blockIdx.x / heads, head = blockIdx.x % heads, kvh = head / p.heads_per_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0)
    for (int g = threadIdx.x; g < p.num_groups; g += kWarps * 32)
      if (p.group_start[g] < 0 || p.group_start[g + 1] < p.group_start[g] || p.group_start[g + 1] > p.num_items)
        set_error(p.status, CDB_ERR_INDEX);
  const int pos = p.item_pos[item], slot = p.item_slot[item];
  if (pos < 0) return;
  if (slot < 0 || slot >= p.bt_rows || pos / kBlock >= p.bt_width) {
    if (threadIdx.x == 0) set_error(p.status, CDB_ERR_INDEX);
    return;
  }
  float q[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    q[i] = bf16_to_f(p.q[(int64_t)item * p.q_stride + (int64_t)head * D + i * 32 + lane]) * p.scale_log2;
    o[i] = 0.f;
  }
  for (int key = warp; key <= pos; key += kWarps) {
    const int64_t id = p.block_table[(int64_t)slot * p.bt_stride + key / kBlock];
    if (id < 0 || (id + 1) * kBlock > p.kv_rows) {
      if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
      continue;
    }
    const __nv_bfloat16* k = p.keys + ((id * kBlock + key % kBlock) * p.kv_heads + kvh) * D + lane;
    const __nv_bfloat16* v = k + p.kv_rows * p.kv_heads * D;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) x += q[i] * bf16_to_f(k[i * 32]);
    x = warp_sum(x);
    const float to = fmaxf(m, x), down = m == -INFINITY ? 0.f : exp2f(m - to), w = exp2f(x - to);
    m = to;
    l = l * down + w;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = o[i] * down + w * bf16_to_f(v[i * 32]);
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int i = 0; i < PER; ++i) s_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = -INFINITY, sum = 0.f, acc = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWarps; ++w) {
    const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - top);
    sum += s_l[w] * f;
    acc += s_o[w][threadIdx.x] * f;
  }
  p.out[(int64_t)item * p.out_stride + (int64_t)head * D + threadIdx.x] = f_to_bf16(sum == 0.f ? 0.f : acc / sum);
}

}  // namespace prefix
}  // namespace cdb

extern "C" int64_t cdb_prefix_decode_workspace_floats(int num_items, int num_groups, int num_heads, int num_kv_heads,
                                                      int head_dim, int num_sms) {
  return num_items >= 0 && num_groups >= 0 && num_heads > 0 && num_kv_heads > 0 && head_dim > 0 && num_sms > 0 ? 1 : 0;
}
extern "C" int64_t cdb_prefix_decode_counters(int num_items, int num_heads, int num_kv_heads) {
  return num_items >= 0 && num_heads > 0 && num_kv_heads > 0 ? 1 : 0;
}

extern "C" int cdb_prefix_decode_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                           const void* kv_base, int num_cache_layers, int64_t kv_rows, int cache_layer,
                                           const int32_t* block_table, int64_t block_table_stride, int table_rows,
                                           int table_width, const int32_t* item_slot, const int32_t* item_pos,
                                           int num_items, const int32_t* group_start, const int32_t* prefix_len,
                                           int num_groups, int num_heads, int num_kv_heads, int head_dim, float scale,
                                           int num_sms, float* workspace, int64_t workspace_floats, int32_t* counters,
                                           int64_t num_counters, int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::prefix;
  if (cache_layer < 0 || cache_layer >= num_cache_layers || kv_rows < kBlock || num_items < 0 || num_groups < 0 ||
      num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0 ||
      num_sms <= 0 || !(scale > 0.f) || scale > 1e30f)
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_stride & 7) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (out_stride & 7) || (reinterpret_cast<uintptr_t>(kv_base) & 15))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_items == 0) return CDB_OK;
  if (q == nullptr || out == nullptr || kv_base == nullptr || block_table == nullptr || item_slot == nullptr ||
      item_pos == nullptr || (num_groups > 0 && (group_start == nullptr || prefix_len == nullptr)))
    return CDB_ERR_INVALID_ARGUMENT;
  (void)workspace, (void)workspace_floats, (void)counters, (void)num_counters;
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.keys = static_cast<const __nv_bfloat16*>(kv_base) + 2 * (int64_t)cache_layer * kv_rows * num_kv_heads * head_dim;
  p.kv_rows = kv_rows;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.num_items = num_items;
  p.kv_heads = num_kv_heads;
  p.heads_per_kv = num_heads / num_kv_heads;
  p.group_start = group_start;
  p.prefix_len = prefix_len;
  p.num_groups = num_groups;
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t ctas = (int64_t)num_items * num_heads;
  if (ctas > 0x7fffffff) return CDB_ERR_UNSUPPORTED;
  auto* kernel = head_dim == 128 ? decode_kernel<128> : head_dim == 96 ? decode_kernel<96> : decode_kernel<64>;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kWarps * 32), 0, st, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}
