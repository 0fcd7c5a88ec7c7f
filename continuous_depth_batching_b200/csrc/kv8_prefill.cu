// Causal prefill attention over the 8-bit paged cache (layout in kv8.cuh): tiles of up to 64
// consecutive query rows of one request, as cdb_prefill_attention takes them, any number of query heads
// per kv head.
//
// A CTA takes one tile and one query head: 4 warps of 16 query rows. The tile's keys come in steps of
// 64 (4 blocks): bulk copies bring the codes (8 contiguous tiles of 16 x D bytes) two steps ahead, the
// CTA turns them into f16 (exact) in shared memory once, and the warps multiply from there (f16
// m16n8k16, fp32 accumulators). Arithmetic as in the decode kernel: q over a power of two, x = S *
// (scale log2e 2^e s_k) in fp32, an online base-2 softmax with l relative to the maximum m of x, and the
// weights of V, 2^(x-m) s_v, relative to their own maximum M of x + log2 s_v, rounded to f16 (2^-11).
// Bound by the tensor cores' mma.sync rate and by the softmax between the two products.
//
// A masked key never counts, whatever it holds: its x is replaced, and a NaN in its V, which a product
// with weight zero would spread, is taken out of the tiles that the diagonal crosses and put back for
// the rows that see it.
#include "kv8.cuh"
#include "smem_tile.cuh"

namespace cdb {
namespace kv8 {

using prefill::ldsm_x4;
using prefill::ldsm_x4_t;
using prefill::RowPitch;
using prefill::swz;

constexpr int TQ = 64, TK = 64;
constexpr uint32_t kAll = 0xffffffffu;

struct PrefillParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const uint8_t* codes;
  const float* scales;
  int num_blocks, kv_heads, heads_per_kv;
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int4* tiles;  // {first row, rows, slot, position of the first row}
  int num_rows;       // rows of q and out
  float scale_log2;
  int32_t* status;
};

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

template <int D>
__global__ void __launch_bounds__(128, 3) prefill_kernel(const PrefillParams p) {
  pdl_trigger();
  constexpr int KS = D / 16, NT = D / 8, PITCH = RowPitch<D>::BYTES;
  constexpr int BLK = kBlock * D;     // bytes of one block's codes
  constexpr int STAGE = 8 * BLK;      // 4 blocks of K, 4 of V
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sk = smem;                 // f16 [64][D]
  uint8_t* sv = sk + TK * PITCH;      // f16 [64][D]
  uint8_t* stage = sv + TK * PITCH;   // [2][STAGE]
  __shared__ __align__(8) uint64_t s_bar[2];
  __shared__ float s_scale[4][2][4];  // [step % 4][K, V][block]; a negative K scale: no such block
  __shared__ unsigned long long s_nan;
  const uint32_t sk_u = smem_u32(sk), sv_u = smem_u32(sv);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) {
    mbar_init(&s_bar[0], 4);
    mbar_init(&s_bar[1], 4);
    s_nan = 0ull;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();

  const int4 tile = p.tiles[blockIdx.y];
  const int head = blockIdx.x, kvh = head / p.heads_per_kv;
  const int row0 = tile.x, nrows = tile.y, slot = tile.z, pos0 = tile.w;
  if (nrows <= 0) return;  // an unused entry of the list
  if (nrows > TQ || row0 < 0 || row0 > p.num_rows - nrows || slot < 0 || slot >= p.bt_rows || pos0 < 0 ||
      (pos0 + nrows - 1) / kBlock >= p.bt_width) {
    if (tid == 0) set_error(p.status, CDB_ERR_INDEX);
    return;
  }
  const int kv_len = pos0 + nrows;
  const int steps = (kv_len + TK - 1) / TK;
  const int blocks = (kv_len + kBlock - 1) / kBlock;
  const int32_t* bt = p.block_table + (int64_t)slot * p.bt_stride;
  const int64_t v_tiles = (int64_t)p.num_blocks * p.kv_heads;

  // Threads 0..3 bring one block of every step each: the id a step ahead of its copies, the copies two
  // steps ahead of their use, the scales with them.
  int id = -1;
  auto fetch_id = [&](int step) {
    const int b = step * 4 + tid;
    id = step < steps && b < blocks ? bt[b] : -1;
  };
  float hold_k = -1.f, hold_v = 1.f;
  auto issue = [&](int step) {
    if (step >= steps) return;
    uint64_t* bar = &s_bar[step & 1];
    const bool used = step * 4 + tid < blocks;
    const bool known = used && id >= 0 && id < p.num_blocks;
    hold_k = -1.f;
    hold_v = 1.f;
    if (known) {
      const int64_t at = (int64_t)id * p.kv_heads + kvh;
      mbar_arrive_expect_tx(bar, 2 * BLK);
      const uint32_t dst = smem_u32(stage) + (step & 1) * STAGE + tid * BLK;
      bulk_copy(dst, p.codes + at * BLK, BLK, smem_u32(bar));
      bulk_copy(dst + 4 * BLK, p.codes + (v_tiles + at) * BLK, BLK, smem_u32(bar));
      hold_k = p.scales[at];
      hold_v = p.scales[v_tiles + at];
    } else {
      if (used) set_error(p.status, CDB_ERR_INDEX);
      mbar_arrive(bar);
    }
  };
  auto post = [&](int step) {
    s_scale[step & 3][0][tid] = hold_k;
    s_scale[step & 3][1][tid] = hold_v > 0.f ? __log2f(hold_v) : -126.f;
  };
  if (tid < 4) {
    fetch_id(0);
    issue(0);
    post(0);
    fetch_id(1);
    issue(1);
    fetch_id(2);
  }

  // q fragments, divided by a power of two per row
  uint32_t qa[KS][4];
  float factor[2];
  const int qr[2] = {warp * 16 + g, warp * 16 + g + 8};
  {
    float amax[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool on = qr[r] < nrows;
      const __nv_bfloat16* src = p.q + (int64_t)(row0 + (on ? qr[r] : 0)) * p.q_stride + (int64_t)head * D + 2 * t;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        qa[kk][r] = on ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
        qa[kk][2 + r] = on ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
        amax[r] = fmaxf(amax[r], fmaxf(fmaxf(fabsf(bf16lo(qa[kk][r])), fabsf(bf16hi(qa[kk][r]))),
                                       fmaxf(fabsf(bf16lo(qa[kk][2 + r])), fabsf(bf16hi(qa[kk][2 + r])))));
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      amax[r] = fmaxf(amax[r], __shfl_xor_sync(kAll, amax[r], 1));
      amax[r] = fmaxf(amax[r], __shfl_xor_sync(kAll, amax[r], 2));
      int e = (int)(__float_as_uint(amax[r]) >> 23) - 127;
      e = amax[r] == 0.f ? 0 : max(-126, min(126, e));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      factor[r] = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        qa[kk][r] = pack_f16x2(bf16lo(qa[kk][r]) * down, bf16hi(qa[kk][r]) * down);
        qa[kk][2 + r] = pack_f16x2(bf16lo(qa[kk][2 + r]) * down, bf16hi(qa[kk][2 + r]) * down);
      }
    }
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, mw[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int qpos[2] = {pos0 + qr[0], pos0 + qr[1]};

  for (int st = 0; st < steps; ++st) {
    // also: the f16 tiles of the last step have been read
    if (!__syncthreads_and(mbar_wait(&s_bar[st & 1], (st >> 1) & 1, p.status))) {
      // a copy that never came: the error is recorded; wait for the next step's, in flight
      if (st + 1 < steps) mbar_wait(&s_bar[(st + 1) & 1], ((st + 1) >> 1) & 1, p.status);
      break;
    }
    const int key0 = st * TK;
    const bool diagonal = key0 + TK - 1 > pos0;
    const uint8_t* src = stage + (st & 1) * STAGE;
    // codes -> f16: a thread takes 16 bytes at a time
    for (int i = tid; i < 2 * TK * D / 16; i += 128) {
      const int r = i / (D / 16), c = i % (D / 16);  // rows 0..63 K, 64..127 V
      uint4 w = *reinterpret_cast<const uint4*>(src + (int64_t)i * 16);
      const int key = r & 63;
      if (r >= TK) {
        if (key0 + key >= kv_len || s_scale[st & 3][0][key >> 4] < 0.f) w = make_uint4(0u, 0u, 0u, 0u);
        if (diagonal) {
          uint32_t ws[4] = {w.x, w.y, w.z, w.w};
          uint32_t any = 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t nan = ((ws[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // the bytes 0x7f and 0xff
            any |= nan;
            ws[e] &= ~(nan | (nan - (nan >> 7)));
          }
          if (any) atomicOr(&s_nan, 1ull << key);
          w = make_uint4(ws[0], ws[1], ws[2], ws[3]);
        }
      }
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
      uint32_t f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = cvt_e4m3x2_f16x2(ws[e] & 0xffffu);
        f[2 * e + 1] = cvt_e4m3x2_f16x2(ws[e] >> 16);
      }
      uint8_t* dst = r >= TK ? sv : sk;
      *reinterpret_cast<uint4*>(dst + swz<D>(key, 2 * c)) = make_uint4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<uint4*>(dst + swz<D>(key, 2 * c + 1)) = make_uint4(f[4], f[5], f[6], f[7]);
    }
    __syncthreads();
    const unsigned long long nans = diagonal ? s_nan : 0ull;
    if (nans) {  // rare: the rows that see a NaN of V get it here
      for (unsigned long long b = nans; b; b &= b - 1) {
        const int key = __ffsll((long long)b) - 1;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint8_t code = src[4 * BLK + key * D + j * 8 + 2 * t + e];
            if ((code & 0x7fu) == 0x7fu) {
              if (key0 + key <= qpos[0]) o[j][e] = NAN;
              if (key0 + key <= qpos[1]) o[j][2 + e] = NAN;
            }
          }
        }
      }
      __syncthreads();
      if (tid == 0) s_nan = 0ull;
    }
    if (tid < 4) {  // this step's codes have been read
      post(st + 1);
      issue(st + 2);
      fetch_id(st + 3);
    }

    float s[TK / 8][4];
#pragma unroll
    for (int j = 0; j < TK / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
      for (int np = 0; np < TK / 16; ++np) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(sk_u + swz<D>(np * 16 + (lane & 7) + 8 * (lane >> 4), 2 * kk + ((lane >> 3) & 1)), b0, b1, b2, b3);
        mma_f16(s[2 * np], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b0, b1);
        mma_f16(s[2 * np + 1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b2, b3);
      }
    }
    // logits, their maxima, and the maxima of logit + log2 s_v
    float mx[2] = {-INFINITY, -INFINITY}, mz[2] = {-INFINITY, -INFINITY};
    float ev[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float ks = s_scale[st & 3][0][b];
      ev[b] = s_scale[st & 3][1][b];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = factor[r] * ks;
        float bm = -INFINITY;
#pragma unroll
        for (int j = 2 * b; j < 2 * b + 2; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[j][2 * r + e];
            x *= f;
            if (diagonal && key0 + j * 8 + 2 * t + e > qpos[r]) x = -INFINITY;
            if (ks < 0.f) x = -INFINITY;
            bm = fmaxf(bm, x);
          }
        }
        mx[r] = fmaxf(mx[r], bm);
        mz[r] = fmaxf(mz[r], bm + ev[b]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(kAll, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(kAll, mx[r], 2));
      mz[r] = fmaxf(mz[r], __shfl_xor_sync(kAll, mz[r], 1));
      mz[r] = fmaxf(mz[r], __shfl_xor_sync(kAll, mz[r], 2));
      const float nm = fmaxf(m[r], mx[r]), nw = fmaxf(mw[r], mz[r]);
      l[r] *= nm == -INFINITY ? 1.f : ex2(m[r] - nm);
      m[r] = nm;
      const float down = nw == -INFINITY ? 1.f : ex2(mw[r] - nw);
      mw[r] = nw;
      if (__any_sync(kAll, down != 1.f)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][2 * r] *= down, o[j][2 * r + 1] *= down;
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = m[r] == -INFINITY ? 0.f : ex2(ev[b] + m[r] - mw[r]);
#pragma unroll
        for (int j = 2 * b; j < 2 * b + 2; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[j][2 * r + e];
            const float w = x == -INFINITY ? 0.f : ex2(x - m[r]);
            l[r] += w;
            x = w * f;
          }
        }
      }
    }
#pragma unroll
    for (int k2 = 0; k2 < TK / 16; ++k2) {
      const uint32_t a0 = pack_f16x2(s[2 * k2][0], s[2 * k2][1]), a1 = pack_f16x2(s[2 * k2][2], s[2 * k2][3]);
      const uint32_t a2 = pack_f16x2(s[2 * k2 + 1][0], s[2 * k2 + 1][1]),
                     a3 = pack_f16x2(s[2 * k2 + 1][2], s[2 * k2 + 1][3]);
#pragma unroll
      for (int cp = 0; cp < NT / 2; ++cp) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(sv_u + swz<D>(k2 * 16 + (lane & 7) + 8 * ((lane >> 3) & 1), 2 * cp + (lane >> 4)), b0, b1, b2, b3);
        mma_f16(o[2 * cp], a0, a1, a2, a3, b0, b1);
        mma_f16(o[2 * cp + 1], a0, a1, a2, a3, b2, b3);
      }
    }
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(kAll, l[r], 1);
    l[r] += __shfl_xor_sync(kAll, l[r], 2);
    if (qr[r] >= nrows) continue;
    const float f = l[r] > 0.f ? ex2(mw[r] - m[r]) / l[r] : (l[r] == 0.f ? 0.f : l[r]);
    __nv_bfloat16* dst = p.out + (int64_t)(row0 + qr[r]) * p.out_stride + (int64_t)head * D + 2 * t;
#pragma unroll
    for (int j = 0; j < NT; ++j)
      *reinterpret_cast<uint32_t*>(dst + j * 8) = pack_bf16x2(o[j][2 * r] * f, o[j][2 * r + 1] * f);
  }
}

template <int D>
static int launch_prefill(const PrefillParams& p, int num_heads, int num_tiles, cudaStream_t st) {
  constexpr int SMEM = 2 * TK * RowPitch<D>::BYTES + 2 * 8 * kBlock * D;
  if (cudaFuncSetAttribute(prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
    return CDB_ERR_CUDA;
  launch_pdl(prefill_kernel<D>, dim3(num_heads, num_tiles), dim3(128), SMEM, st, p);
  return cudaPeekAtLastError() == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

}  // namespace kv8
}  // namespace cdb

extern "C" int cdb_kv8_prefill_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, int num_rows,
                                         const void* codes, const float* scales, int num_cache_layers, int cache_layer,
                                         int num_blocks, const int32_t* block_table, int64_t block_table_stride,
                                         int table_rows, int table_width, const void* tiles, int num_tiles,
                                         int num_heads, int num_kv_heads, int head_dim, float scale, int32_t* status,
                                         void* stream) {
  using namespace cdb;
  using namespace cdb::kv8;
  if (codes == nullptr || scales == nullptr || (reinterpret_cast<uintptr_t>(codes) & 15) || cache_layer < 0 ||
      cache_layer >= num_cache_layers || num_blocks <= 0 || num_rows < 0 || num_tiles < 0 || num_tiles > 65535 ||
      num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0)
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_stride & 7) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (out_stride & 7) || (reinterpret_cast<uintptr_t>(tiles) & 15))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_tiles == 0) return CDB_OK;
  if (q == nullptr || out == nullptr || block_table == nullptr || tiles == nullptr) return CDB_ERR_INVALID_ARGUMENT;
  PrefillParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  const int64_t at = (int64_t)num_blocks * num_kv_heads * 2 * cache_layer;
  p.codes = static_cast<const uint8_t*>(codes) + at * kBlock * head_dim;
  p.scales = scales + at;
  p.num_blocks = num_blocks;
  p.kv_heads = num_kv_heads;
  p.heads_per_kv = num_heads / num_kv_heads;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.tiles = static_cast<const int4*>(tiles);
  p.num_rows = num_rows;
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_prefill<128>(p, num_heads, num_tiles, st);
  if (head_dim == 96) return launch_prefill<96>(p, num_heads, num_tiles, st);
  return launch_prefill<64>(p, num_heads, num_tiles, st);
}
