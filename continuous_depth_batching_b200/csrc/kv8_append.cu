// Writing and reading back the 8-bit paged KV cache (layout and scale rule in kv8.cuh).
//
// Append. The rows of a call that fall in one block form a run: the same slot, consecutive
// positions. One warp owns a (run, kv head, K or V) tile: it loads the run's up to 16 rows, adds the
// bias and rotates in fp32, takes the tile's largest magnitude, settles the block's scale, rescales
// the codes that were there when the scale grew, and writes codes and scale. Nobody else touches the
// tile, so no atomics and no second pass over the new values. The query heads are rotated by other
// warps of the same launch. Bound by bytes for prompts (q, k, v in, q and codes out) and by the chain
// of dependent loads (position, block id, values) for a decode step.
#include "kv8.cuh"

namespace cdb {
namespace kv8 {

struct AppendParams {
  const __nv_bfloat16* qkv;  // q | k | v heads of each row
  int64_t qkv_stride;
  __nv_bfloat16* q_out;  // may be the q columns of qkv; null: q is left alone
  int64_t q_out_stride;
  uint8_t* codes;  // this cache layer's
  float* scales;
  int num_blocks;
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int32_t* item_slot;
  const int32_t* item_pos;
  int rope_mode;
  const void* rope_cos;
  const void* rope_sin;
  int rope_rows;
  const __nv_bfloat16* qk_bias;  // [heads + kv heads][D] or null
  int num_items, num_heads, num_kv_heads;
  int group;  // rows whose runs one CTA starts
  int32_t* status;
};

__device__ __forceinline__ uint4 ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ void unpack8(uint4 w, float (&a)[8]) {
  a[0] = bf16lo(w.x), a[1] = bf16hi(w.x), a[2] = bf16lo(w.y), a[3] = bf16hi(w.y);
  a[4] = bf16lo(w.z), a[5] = bf16hi(w.z), a[6] = bf16lo(w.w), a[7] = bf16hi(w.w);
}

// Dims [x0, x0 + 8) of one head vector, biased and rotated in fp32 with no rounding in between (the
// caller rounds once: to bf16 for q, to e4m3 for k). Every lane of the warp calls it, `on` or not:
// the split-half partner chunk comes from the lane that holds it. Angles are the tables' values.
template <int D>
__device__ __forceinline__ void rotated8(const AppendParams& p, const __nv_bfloat16* x, const __nv_bfloat16* bias,
                                         int mode, int pos, int x0, bool on, float (&y)[8]) {
  constexpr int LPR = D / 8;  // lanes per row
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  unpack8(on ? ld16(x + x0) : z, y);
  if (bias != nullptr) {
    float b[8];
    unpack8(on ? ld16(bias + x0) : z, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += b[e];
  }
  if (mode == 1) {
    const int lane = threadIdx.x & 31;
    const bool low = x0 < D / 2;
    const int src = (low ? lane + LPR / 2 : lane - LPR / 2) & 31;
    float c[8], s[8];
    unpack8(on ? ld16(static_cast<const __nv_bfloat16*>(p.rope_cos) + (int64_t)pos * D + x0) : z, c);
    unpack8(on ? ld16(static_cast<const __nv_bfloat16*>(p.rope_sin) + (int64_t)pos * D + x0) : z, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float o = __shfl_sync(0xffffffffu, y[e], src);
      s[e] *= low ? -o : o;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], c[e], s[e]);
  } else if (mode == 2) {
    const float4 zf = make_float4(0.f, 0.f, 0.f, 0.f);
    const int64_t at = (int64_t)pos * (D / 2) + x0 / 2;
    const float4 c = on ? *reinterpret_cast<const float4*>(static_cast<const float*>(p.rope_cos) + at) : zf;
    const float4 s = on ? *reinterpret_cast<const float4*>(static_cast<const float*>(p.rope_sin) + at) : zf;
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = y[2 * i], b = y[2 * i + 1];
      y[2 * i] = fmaf(a, cc[i], -b * ss[i]);
      y[2 * i + 1] = fmaf(b, cc[i], a * ss[i]);
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // infinities saturate and NaN stays NaN, under the others' scale
}

template <int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int LPR = D / 8;       // lanes of one row, 8 dims each
  constexpr int RPI = 32 / LPR;    // rows per iteration (96: lanes 24..31 idle)
  constexpr int IT = kBlock / RPI;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * p.group;
  const int rows = min(p.group, p.num_items - row0);
  const bool in_row = lane < LPR * RPI;
  const int sub = in_row ? lane / LPR : 0, x0 = in_row ? (lane % LPR) * 8 : 0;
  const int q_tasks = p.q_out != nullptr ? p.num_heads : 0;
  const int tasks = q_tasks + 2 * p.num_kv_heads;
  const int64_t k_col = (int64_t)p.num_heads * D, v_col = k_col + (int64_t)p.num_kv_heads * D;

  for (int task = blockIdx.y * 8 + warp; task < tasks; task += gridDim.y * 8) {
    if (task < q_tasks) {
      const __nv_bfloat16* bias = p.qk_bias != nullptr ? p.qk_bias + (int64_t)task * D : nullptr;
      for (int i = 0; i < rows; i += RPI) {
        const int r = row0 + i + sub;
        const int pos = in_row && i + sub < rows ? p.item_pos[r] : -1;
        const bool on = pos >= 0 && (p.rope_mode == 0 || pos < p.rope_rows);
        if (!__any_sync(0xffffffffu, on)) continue;
        float y[8];
        rotated8<D>(p, p.qkv + (int64_t)r * p.qkv_stride + (int64_t)task * D, bias, p.rope_mode, pos, x0, on, y);
        if (on)
          *reinterpret_cast<uint4*>(p.q_out + (int64_t)r * p.q_out_stride + (int64_t)task * D + x0) =
              make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                         pack_bf16x2(y[6], y[7]));
      }
      continue;
    }
    const int kt = task - q_tasks;
    const bool is_v = kt >= p.num_kv_heads;
    const int head = is_v ? kt - p.num_kv_heads : kt;
    const int mode = is_v ? 0 : p.rope_mode;
    const __nv_bfloat16* bias =
        !is_v && p.qk_bias != nullptr ? p.qk_bias + (int64_t)(p.num_heads + head) * D : nullptr;
    const int64_t col = (is_v ? v_col : k_col) + (int64_t)head * D;

    for (int i = 0; i < rows; ++i) {
      // Rows i .. i + 15 of the call: where the run that starts at row i ends.
      const int r = row0 + i;
      const int pos = p.item_pos[r];
      if (pos < 0) continue;
      const int slot = p.item_slot[r];
      if (r > 0) {
        const int before = p.item_pos[r - 1];
        if (before >= 0 && p.item_slot[r - 1] == slot && before / kBlock == pos / kBlock) {
          // a later row of a run; one that does not follow its predecessor has no place in the block
          if (before + 1 != pos && lane == 0) set_error(p.status, CDB_ERR_INDEX);
          continue;
        }
      }
      bool next = false;
      if (lane < kBlock && r + lane < p.num_items)
        next = p.item_slot[r + lane] == slot && p.item_pos[r + lane] == pos + lane &&
               pos % kBlock + lane < kBlock;
      const int n = __ffs(~__ballot_sync(0xffffffffu, next)) - 1;
      int blk = -1;
      if (slot >= 0 && slot < p.bt_rows && pos / kBlock < p.bt_width &&
          (p.rope_mode == 0 || pos + n <= p.rope_rows))
        blk = p.block_table[(int64_t)slot * p.bt_stride + pos / kBlock];
      if (blk < 0 || blk >= p.num_blocks) {
        if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
        continue;
      }
      const int off = pos % kBlock;
      const int64_t tile = ((int64_t)(is_v ? p.num_blocks : 0) + blk) * p.num_kv_heads + head;
      uint8_t* codes = p.codes + tile * (kBlock * D);
      const float was = off > 0 ? p.scales[tile] : 0.f;

      float y[IT][8];
      float amax = 0.f;
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        if (it * RPI >= n) break;
        const int j = it * RPI + sub;
        const bool on = in_row && j < n;
        rotated8<D>(p, p.qkv + (int64_t)(r + j) * p.qkv_stride + col, bias, mode, pos + j, x0, on, y[it]);
        if (on) {
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(y[it][e]));
        }
      }
      amax = warp_max(amax);
      float scale = block_scale(amax);
      if (off > 0) {
        if (was >= scale) {
          scale = was;
        } else {  // the block grows: its old codes move down by a power of two
          const float ratio = was / scale;
          for (int c = lane; c < off * LPR; c += 32) {
            uint2* at = reinterpret_cast<uint2*>(codes + c * 8);
            const uint2 old = *at;
            const uint32_t w[2] = {old.x, old.y};
            uint32_t o[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float a, b, c2, d;
              unpack_f16x2(cvt_e4m3x2_f16x2(w[k] & 0xffffu), a, b);
              unpack_f16x2(cvt_e4m3x2_f16x2(w[k] >> 16), c2, d);
              o[k] = cvt_f32x2_e4m3x2(a * ratio, b * ratio) | (cvt_f32x2_e4m3x2(c2 * ratio, d * ratio) << 16);
            }
            *at = make_uint2(o[0], o[1]);
          }
        }
      }
      const float inv = 1.f / scale;
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        if (it * RPI >= n) break;
        const int j = it * RPI + sub;
        if (in_row && j < n) {
          const uint32_t lo = cvt_f32x2_e4m3x2(y[it][0] * inv, y[it][1] * inv) |
                              (cvt_f32x2_e4m3x2(y[it][2] * inv, y[it][3] * inv) << 16);
          const uint32_t hi = cvt_f32x2_e4m3x2(y[it][4] * inv, y[it][5] * inv) |
                              (cvt_f32x2_e4m3x2(y[it][6] * inv, y[it][7] * inv) << 16);
          *reinterpret_cast<uint2*>(codes + (off + j) * D + x0) = make_uint2(lo, hi);
        }
      }
      if (lane == 0) p.scales[tile] = scale;
    }
  }
}

// Blocks blocks[i] of one cache layer as bf16 [n][2][kv heads][16][D]: a code times a power of two
// is a bf16 value, so nothing is rounded. One thread per 16 codes: 16 bytes in, 32 out.
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t* codes, const float* scales, int num_blocks,
                                                     int kv_heads, int D, const int32_t* blocks, int64_t chunks,
                                                     __nv_bfloat16* out, int32_t* status) {
  pdl_trigger();
  pdl_wait();
  const int per_tile = kBlock * D / 16;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per_tile;  // (block, kv, head)
    const int c = (int)(i - t * per_tile);
    const int head = (int)(t % kv_heads);
    const int64_t bk = t / kv_heads;
    const int blk = blocks[bk >> 1];
    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
    if (blk >= 0 && blk < num_blocks) {
      const int64_t tile = ((bk & 1) * num_blocks + blk) * kv_heads + head;
      const uint4 w = ld16(codes + tile * (kBlock * D) + c * 16);
      const float s = scales[tile];
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      uint32_t o[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpack_f16x2(cvt_e4m3x2_f16x2(in[k] & 0xffffu), a, b);
        o[2 * k] = pack_bf16x2(a * s, b * s);
        unpack_f16x2(cvt_e4m3x2_f16x2(in[k] >> 16), a, b);
        o[2 * k + 1] = pack_bf16x2(a * s, b * s);
      }
      lo = make_uint4(o[0], o[1], o[2], o[3]);
      hi = make_uint4(o[4], o[5], o[6], o[7]);
    } else if (c == 0) {
      set_error(status, CDB_ERR_INDEX);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + i * 16);
    dst[0] = lo;
    dst[1] = hi;
  }
}

static int done() { return cudaPeekAtLastError() == cudaSuccess ? CDB_OK : CDB_ERR_CUDA; }

}  // namespace kv8
}  // namespace cdb

static bool kv8_cache_ok(const void* codes, const void* scales, int num_cache_layers, int cache_layer, int num_blocks,
                         int num_kv_heads, int head_dim) {
  return codes != nullptr && scales != nullptr && (reinterpret_cast<uintptr_t>(codes) & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(scales) & 3) == 0 && cache_layer >= 0 && cache_layer < num_cache_layers &&
         num_blocks > 0 && num_kv_heads > 0 && head_dim > 0;
}

extern "C" int cdb_kv8_append(const void* qkv, int64_t qkv_stride, void* q_out, int64_t q_out_stride, void* codes,
                              float* scales, int num_cache_layers, int cache_layer, int num_blocks,
                              const int32_t* block_table, int64_t block_table_stride, int table_rows, int table_width,
                              const int32_t* item_slot, const int32_t* item_pos, int rope_mode, const void* rope_cos,
                              const void* rope_sin, int rope_rows, const void* qk_bias, int num_items, int num_heads,
                              int num_kv_heads, int head_dim, int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::kv8;
  if (!kv8_cache_ok(codes, scales, num_cache_layers, cache_layer, num_blocks, num_kv_heads, head_dim) ||
      num_items < 0 || num_heads <= 0 || table_rows < 0 || table_width < 0 || rope_mode < 0 || rope_mode > 2 ||
      (rope_mode != 0 && (rope_cos == nullptr || rope_sin == nullptr || rope_rows < 0)))
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
                         reinterpret_cast<uintptr_t>(rope_cos) | reinterpret_cast<uintptr_t>(rope_sin) |
                         reinterpret_cast<uintptr_t>(qk_bias);
  if ((bits & 15) || (qkv_stride & 7) || (q_out != nullptr && (q_out_stride & 7))) return CDB_ERR_INVALID_ARGUMENT;
  if (num_items == 0) return CDB_OK;
  if (qkv == nullptr || block_table == nullptr || item_slot == nullptr || item_pos == nullptr)
    return CDB_ERR_INVALID_ARGUMENT;
  AppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.qkv_stride = qkv_stride;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_out_stride = q_out_stride;
  const int64_t tiles = (int64_t)num_blocks * num_kv_heads * 2 * cache_layer;
  p.codes = static_cast<uint8_t*>(codes) + tiles * kBlock * head_dim;
  p.scales = scales + tiles;
  p.num_blocks = num_blocks;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.rope_mode = rope_mode;
  p.rope_cos = rope_cos;
  p.rope_sin = rope_sin;
  p.rope_rows = rope_rows;
  p.qk_bias = static_cast<const __nv_bfloat16*>(qk_bias);
  p.num_items = num_items;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.status = status;
  // Decode steps have a run per row: one row per CTA spreads them. Prompts have a run per 16 rows, and
  // a CTA per row would start 15 of 16 kv warps for nothing.
  p.group = num_items <= 1024 ? 1 : kBlock;
  const int tasks = (q_out != nullptr ? num_heads : 0) + 2 * num_kv_heads;
  const dim3 grid((num_items + p.group - 1) / p.group, min(65535, (tasks + 7) / 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    launch_pdl(append_kernel<128>, grid, dim3(256), 0, st, p);
  else if (head_dim == 96)
    launch_pdl(append_kernel<96>, grid, dim3(256), 0, st, p);
  else
    launch_pdl(append_kernel<64>, grid, dim3(256), 0, st, p);
  return done();
}

extern "C" int cdb_kv8_gather(const void* codes, const float* scales, int num_cache_layers, int cache_layer,
                              int num_blocks, int num_kv_heads, int head_dim, const int32_t* blocks, int n, void* out,
                              int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::kv8;
  if (!kv8_cache_ok(codes, scales, num_cache_layers, cache_layer, num_blocks, num_kv_heads, head_dim) || n < 0 ||
      (head_dim & 15) || (reinterpret_cast<uintptr_t>(out) & 15))
    return CDB_ERR_INVALID_ARGUMENT;
  if (n == 0) return CDB_OK;
  if (blocks == nullptr || out == nullptr) return CDB_ERR_INVALID_ARGUMENT;
  const int64_t tiles = (int64_t)num_blocks * num_kv_heads * 2 * cache_layer;
  const int64_t chunks = (int64_t)n * 2 * num_kv_heads * head_dim;  // 16 codes each
  const int64_t ctas = (chunks + 255) / 256;
  const int grid = (int)(ctas < 148 * 16 ? ctas : 148 * 16);
  launch_pdl(gather_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream),
             static_cast<const uint8_t*>(codes) + tiles * kBlock * head_dim, scales + tiles, num_blocks, num_kv_heads,
             head_dim, blocks, chunks, static_cast<__nv_bfloat16*>(out), status);
  return done();
}
