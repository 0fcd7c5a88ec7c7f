// Writing and reading back the 8-bit paged KV cache (layout and scale rule in kv8.cuh).
//
// Append. The rows of a call that fall in one block form a run: the same slot, consecutive positions. One warp
// owns the (run, head) tiles of a few heads of K or V: it brings a head's up to 16 rows, adds the bias and
// rotates in fp32, takes the tile's largest magnitude, settles the block's scale, rescales the codes that were
// there when the scale grew, and writes codes and scale. Nobody else touches the tile, so no atomics and no
// second pass over the new values. The query heads are rotated by other warps of the same launch.
//
// Bound: for prompts bytes (q, k, v in, q and codes out) and the instructions around a value, some 100 for 8 of
// them in a lane; for a decode step the chain of dependent loads (position, block id, values). Measured: 4096
// rows of prompts, 16 heads of 128: 22 us (84 MB, 3.8 TB/s); some 4000 rows of 55 heads of 96 with biases: 65 us
// (3.4 TB/s; 85 us with the rows' angles read from global memory for each head and one head to a warp); 80
// decode rows, 16 heads of 128: 3.9 us.
//
// Read-back (gather): 1 byte in, 2 out a code. 29 us for those 4000 rows (132 MB, 4.5 TB/s; 20 us of bytes), half of
// the issue slots busy with the index divisions of each 16 codes.
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
  int heads;  // kv heads of a warp's task
  int32_t* status;
};

__device__ __forceinline__ uint4 ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ void unpack8(uint4 w, float (&a)[8]) {
  a[0] = bf16lo(w.x), a[1] = bf16hi(w.x), a[2] = bf16lo(w.y), a[3] = bf16hi(w.y);
  a[4] = bf16lo(w.z), a[5] = bf16hi(w.z), a[6] = bf16lo(w.w), a[7] = bf16hi(w.w);
}

// The cos and sin entries of dims [x0, x0 + 8) at one position: 8 + 8 bf16 (mode 1) or 4 + 4 fp32 (mode 2).
struct Angles {
  uint4 c, s;
};

template <int D>
__device__ __forceinline__ Angles load_angles(const AppendParams& p, int mode, int pos, int x0, bool on) {
  Angles a;
  a.c = a.s = make_uint4(0u, 0u, 0u, 0u);
  if (on && mode == 1) {
    const int64_t at = (int64_t)pos * D + x0;
    a.c = ld16(static_cast<const __nv_bfloat16*>(p.rope_cos) + at);
    a.s = ld16(static_cast<const __nv_bfloat16*>(p.rope_sin) + at);
  } else if (on && mode == 2) {
    const int64_t at = (int64_t)pos * (D / 2) + x0 / 2;
    a.c = ld16(static_cast<const float*>(p.rope_cos) + at);
    a.s = ld16(static_cast<const float*>(p.rope_sin) + at);
  }
  return a;
}

// One head vector's dims [x0, x0 + 8), biased and rotated in fp32 with no rounding in between (the caller
// rounds once: to bf16 for q, to e4m3 for k). Every lane of the warp calls it: the split-half partner
// chunk comes from the lane that holds it.
template <int D>
__device__ __forceinline__ void rotated8(uint4 raw, uint4 bias, int mode, const Angles& a, int x0, float (&y)[8]) {
  constexpr int LPR = D / 8;  // lanes per row
  unpack8(raw, y);
  float b[8];
  unpack8(bias, b);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] += b[e];
  if (mode == 1) {
    const int lane = threadIdx.x & 31;
    const bool low = x0 < D / 2;
    const int src = (low ? lane + LPR / 2 : lane - LPR / 2) & 31;
    float c[8], s[8];
    unpack8(a.c, c);
    unpack8(a.s, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float o = __shfl_sync(0xffffffffu, y[e], src);
      s[e] *= low ? -o : o;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], c[e], s[e]);
  } else if (mode == 2) {
    const uint32_t cc[4] = {a.c.x, a.c.y, a.c.z, a.c.w}, ss[4] = {a.s.x, a.s.y, a.s.z, a.s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = y[2 * i], v = y[2 * i + 1], c = __uint_as_float(cc[i]), s = __uint_as_float(ss[i]);
      y[2 * i] = fmaf(u, c, -v * s);
      y[2 * i + 1] = fmaf(v, c, u * s);
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // infinities saturate and NaN stays NaN, under the others' scale
}

// q: a warp rotates HB heads of rows [row0, end), RPI rows at a time, with the rows' angles in registers, the
// heads' loads in flight together and the next rows' behind them.
constexpr int HB = 4;

template <int D>
__device__ __forceinline__ void rotate_q(const AppendParams& p, int row0, int end, int head0) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int sub = lane / LPR, x0 = (lane % LPR) * 8;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 raw[HB];
  Angles a;
  auto fetch = [&](int r) {
    const int pos = sub < RPI && r < end ? p.item_pos[r] : -1;
    const bool on = pos >= 0 && (p.rope_mode == 0 || pos < p.rope_rows);
#pragma unroll
    for (int h = 0; h < HB; ++h)
      raw[h] = on && head0 + h < p.num_heads ? ld16(p.qkv + (int64_t)r * p.qkv_stride + (int64_t)(head0 + h) * D + x0)
                                             : zero;
    a = load_angles<D>(p, p.rope_mode, pos, x0, on);
    return on;
  };
  bool on = fetch(row0 + sub);
  for (int r = row0 + sub; r - sub < end; r += RPI) {
    uint4 now[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h) now[h] = raw[h];
    const Angles angles = a;
    const bool had = on;
    on = fetch(r + RPI);
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const uint4 bias = had && p.qk_bias != nullptr && head0 + h < p.num_heads
                             ? ld16(p.qk_bias + (int64_t)(head0 + h) * D + x0)
                             : zero;
      float y[8];
      rotated8<D>(now[h], bias, p.rope_mode, angles, x0, y);
      if (had && head0 + h < p.num_heads)
        *reinterpret_cast<uint4*>(p.q_out + (int64_t)r * p.q_out_stride + (int64_t)(head0 + h) * D + x0) =
            make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                       pack_bf16x2(y[6], y[7]));
    }
  }
}

// Shared memory of a warp: one head of a run of 16 rows, and their cos and sin, a whole warp's chunks at a time.
__host__ __device__ constexpr int stage_bytes(int dim) { return 3 * kBlock / (32 / (dim / 8)) * 32 * 16; }

__device__ __forceinline__ void async_copy16(uint4* dst, const void* src, bool on) {  // zeros where not on
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// A run of rows of one block.
struct Run {
  int slot, pos, n;
};

// The runs that start in rows [row0, row0 + 16): lane L looks at row row0 - 1 + L, so that the warp sees the
// row before the group and every row that a run of the group can reach.
struct Runs {
  int slot, pos;             // this lane's row
  unsigned starts, follows;  // lanes that start a run / follow their predecessor in one
};

__device__ __forceinline__ Runs find_runs(const AppendParams& p, int row0, int rows) {
  const int lane = threadIdx.x & 31, at = row0 - 1 + lane;
  const bool in = at >= 0 && at < p.num_items;
  Runs r;
  r.pos = in ? p.item_pos[at] : -1;
  r.slot = in ? p.item_slot[at] : -1;
  const int before = __shfl_up_sync(0xffffffffu, r.pos, 1), before_slot = __shfl_up_sync(0xffffffffu, r.slot, 1);
  const bool same = lane > 0 && r.pos >= 0 && before >= 0 && before_slot == r.slot && before / kBlock == r.pos / kBlock;
  const bool here = lane >= 1 && lane <= rows;
  // a row that does not follow its predecessor in their block has no place there
  if (here && same && before + 1 != r.pos) set_error(p.status, CDB_ERR_INDEX);
  r.starts = __ballot_sync(0xffffffffu, here && r.pos >= 0 && !same);
  r.follows = __ballot_sync(0xffffffffu, same && before + 1 == r.pos);
  return r;
}

// The run that starts at lane s.
__device__ __forceinline__ Run take_run(const Runs& r, int s) {
  Run run;
  run.slot = __shfl_sync(0xffffffffu, r.slot, s);
  run.pos = __shfl_sync(0xffffffffu, r.pos, s);
  run.n = s == 31 ? 1 : __ffs(~(r.follows >> (s + 1)));
  return run;
}

// The block that the run's rows lie in, -1 where its indexes do not fit.
__device__ __forceinline__ int block_of(const AppendParams& p, const Run& run) {
  if (run.slot < 0 || run.slot >= p.bt_rows || run.pos / kBlock >= p.bt_width ||
      (p.rope_mode != 0 && run.pos > p.rope_rows - run.n))
    return -1;
  return p.block_table[(int64_t)run.slot * p.bt_stride + run.pos / kBlock];
}

// k or v of heads [head, end) of a run. ROWS: the most rows a run may have here (16, or what one pass holds).
// A head's rows and the rows' angles come asynchronously into shared memory (`stage`: every lane's own chunks,
// so no barrier), the first head's beside the block id, each next head's while the one before is turned into
// codes: registers hold one head's rotated rows only. Those stay in registers from there to the codes (rotating them twice,
// for a third CTA on the SM, measured 138 us against 114 on 55 x 96 prompts). The magnitude is taken over
// everything first, and again over the finite values in the rare tile that has others.
template <int D, int ROWS, bool IS_V>
__device__ __forceinline__ void write_tiles(const AppendParams& p, int r, const Run& run, int head, int end,
                                            uint4* stage) {
  constexpr int LPR = D / 8, RPI = 32 / LPR, IT = (ROWS + RPI - 1) / RPI;
  const int lane = threadIdx.x & 31;
  const int sub = lane / LPR, x0 = (lane % LPR) * 8;
  const int off = run.pos % kBlock;
  const int blk = block_of(p, run);
  const __nv_bfloat16* src = p.qkv + (int64_t)(r + sub) * p.qkv_stride +
                             (int64_t)(p.num_heads + (IS_V ? p.num_kv_heads : 0) + head) * D + x0;
  const int64_t step = (int64_t)RPI * p.qkv_stride;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const int rows = sub < RPI ? run.n - sub : 0;  // this lane's: it * RPI < rows
  const bool biased = !IS_V && p.qk_bias != nullptr && sub < RPI;
  const __nv_bfloat16* bias_at = p.qk_bias + (int64_t)(p.num_heads + head) * D + x0;
  uint4* place = stage + lane;             // [IT][32 lanes] rows
  uint4* turn = stage + kBlock / RPI * 32 + lane;  // [IT][cos, sin][32 lanes]
  auto fetch = [&]() {
#pragma unroll
    for (int it = 0; it < IT; ++it)
      async_copy16(place + it * 32, it * RPI < rows ? src + it * step : p.qkv, it * RPI < rows);
    src += D;
  };
  fetch();
  if (!IS_V && p.rope_mode != 0) {
    const char *c = static_cast<const char*>(p.rope_cos), *s = static_cast<const char*>(p.rope_sin);
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int pos = run.pos + it * RPI + sub;
      const bool on = it * RPI < rows && pos < p.rope_rows;
      // 2 D bytes a position in either mode, 16 of them for 8 dims
      const int64_t at = on ? ((int64_t)pos * D + x0) * 2 : 0;
      async_copy16(turn + it * 64, c + at, on);
      async_copy16(turn + it * 64 + 32, s + at, on);
    }
  }
  if (blk < 0 || blk >= p.num_blocks) {
    if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  int64_t tile = ((int64_t)(IS_V ? p.num_blocks : 0) + blk) * p.num_kv_heads + head;
  for (; head < end; ++head, ++tile) {
    uint8_t* codes = p.codes + tile * (kBlock * D);
    const float was = off > 0 ? p.scales[tile] : 0.f;
    const uint4 bias = biased ? ld16(bias_at) : zero;
    bias_at += D;
    asm volatile("cp.async.wait_all;" ::: "memory");
    float y[IT][8];
    float amax = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const uint4 raw = place[it * 32];
      if constexpr (IS_V) {
        unpack8(raw, y[it]);
      } else {
        Angles a;
        if (p.rope_mode != 0) a.c = turn[it * 64], a.s = turn[it * 64 + 32];
        rotated8<D>(raw, it * RPI < rows ? bias : zero, p.rope_mode, a, x0, y[it]);  // zeros where no row is
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(y[it][e]));  // (a NaN is passed over)
    }
    if (head + 1 < end) fetch();  // over the rows just read: each lane's own
    amax = warp_max(amax);
    if (amax > 3.402823466e38f) {  // infinities saturate, under the others' scale
      amax = 0.f;
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(y[it][e]));
      amax = warp_max(amax);
    }
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
    uint8_t* dst = codes + (off + sub) * D + x0;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (it * RPI < rows) {
        const uint32_t lo = cvt_f32x2_e4m3x2(y[it][0] * inv, y[it][1] * inv) |
                            (cvt_f32x2_e4m3x2(y[it][2] * inv, y[it][3] * inv) << 16);
        const uint32_t hi = cvt_f32x2_e4m3x2(y[it][4] * inv, y[it][5] * inv) |
                            (cvt_f32x2_e4m3x2(y[it][6] * inv, y[it][7] * inv) << 16);
        *reinterpret_cast<uint2*>(dst + it * RPI * D) = make_uint2(lo, hi);
      }
    }
    if (lane == 0) p.scales[tile] = scale;
  }
}

// A CTA takes `group` rows: blockIdx.y first counts the q warps' tasks (HB heads), then those of the k and v
// warps (`heads` heads of one of them, every run that starts in the group).
template <int D>
__global__ void __launch_bounds__(256, 2) append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int RPI = 32 / (D / 8);
  const int warp = threadIdx.x >> 5;
  extern __shared__ uint4 smem[];
  uint4* stage = smem + warp * (stage_bytes(D) / 16);
  const int row0 = blockIdx.x * p.group;
  const int rows = min(p.group, p.num_items - row0);
  const int q_tasks = p.q_out != nullptr ? (p.num_heads + HB - 1) / HB : 0;
  const int kv_tasks = (p.num_kv_heads + p.heads - 1) / p.heads, tasks = q_tasks + 2 * kv_tasks;
  const Runs runs = find_runs(p, row0, rows);
  for (int task = blockIdx.y * 8 + warp; task < tasks; task += gridDim.y * 8) {
    if (task < q_tasks) {
      rotate_q<D>(p, row0, row0 + rows, task * HB);
      continue;
    }
    const int kt = task - q_tasks;
    const bool is_v = kt >= kv_tasks;
    const int head = (is_v ? kt - kv_tasks : kt) * p.heads, end = min(head + p.heads, p.num_kv_heads);
    for (unsigned left = runs.starts; left; left &= left - 1) {
      const int at = __ffs(left) - 1;
      const Run run = take_run(runs, at);
      const int r = row0 - 1 + at;
      if (run.n <= RPI) {
        if (is_v) write_tiles<D, RPI, true>(p, r, run, head, end, stage);
        else write_tiles<D, RPI, false>(p, r, run, head, end, stage);
      } else {
        if (is_v) write_tiles<D, kBlock, true>(p, r, run, head, end, stage);
        else write_tiles<D, kBlock, false>(p, r, run, head, end, stage);
      }
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

template <int D>
static cudaError_t launch_append(const AppendParams& p, dim3 grid, cudaStream_t st) {
  constexpr int smem = 8 * stage_bytes(D);
  const cudaError_t e = cudaFuncSetAttribute(append_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e != cudaSuccess ? e : launch_pdl(append_kernel<D>, grid, dim3(256), smem, st, p);
}

static int launched(cudaError_t e) { return e == cudaSuccess ? CDB_OK : CDB_ERR_CUDA; }

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
  // Decode steps have a run per row: a CTA per row and a head per warp spread them. Prompts have a run per 16
  // rows, and a CTA per row would start 15 of 16 kv warps for nothing. Measured with 16 heads of 128, a row per
  // CTA against 16: 80 decode rows 3.9 us (38), 512 16 (39), 1024 35 (54); prompts of 512 rows 10.5 (11.3), of
  // 1024 19.7 (15.4), of 4096 72 (22). A warp's heads in prompts: 2, 3, 4, 6, 8 take 96, 95, 96, 99, 100 us on the
  // 55 x 96 case (with its read-back), 11 take 113.
  p.group = num_items <= 1024 ? 1 : kBlock;
  p.heads = p.group == 1 ? 1 : 4;
  const int tasks = (q_out != nullptr ? (num_heads + HB - 1) / HB : 0) + 2 * ((num_kv_heads + p.heads - 1) / p.heads);
  const dim3 grid((num_items + p.group - 1) / p.group, min(65535, (tasks + 7) / 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launched(launch_append<128>(p, grid, st));
  if (head_dim == 96) return launched(launch_append<96>(p, grid, st));
  return launched(launch_append<64>(p, grid, st));
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
  return launched(launch_pdl(gather_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream),
                             static_cast<const uint8_t*>(codes) + tiles * kBlock * head_dim, scales + tiles, num_blocks,
                             num_kv_heads, head_dim, blocks, chunks, static_cast<__nv_bfloat16*>(out), status));
}
