// Products of a few token rows with 4-bit weights:
//   out[m][n] = bf16( sum over groups j of s[n][j] * sum over k in group j of (q[n][k] - z[n][j]) x[m][k] )
// Weights q are nibbles, two to a byte along k (low nibble first), as they are stored; no layout pass.
//
// Bound by the weights' bytes, N K / 2, which are read once per 32 tokens. A warp owns 16 weight rows
// and streams its share of k through a ring in shared memory (TMA boxes of 16 rows x 128 bytes = 256 k,
// 128-byte swizzle, so that the fragment loads below hit every bank once). Few row tiles are made up
// for by splitting k over a cluster of CTAs, whose fp32 partials meet in distributed shared memory in
// rank order. The token rows lie in shared memory for the CTA's eight warps.
//
// The products run on the tensor cores (bf16 m16n8k16: 16 weight rows, 8 tokens). A nibble q becomes
// the bf16 number 128 + q by one AND and one OR into the mantissa, exactly, and the offset is taken
// off per group with the group's sum of x:
//   sum (q - z) x = sum (128 + q) x - (128 + z) sum x,
// both sums in fp32, then times the group's scale into the fp32 result: no weight is rounded. What the
// offset cancels costs fp32's 2^-24 of 128 sum |x|, far below bf16's rounding of the result.
#include <cuda.h>

#include "cdb_common.cuh"

namespace cdb {
namespace w4 {

constexpr int kWarps = 8;
constexpr int kRows = 16;             // weight rows of a warp
constexpr int kSub = 256;             // k of one TMA box (128 bytes of a row)
constexpr int kTile = kRows * kSub / 2;
constexpr int kStages = 4;
constexpr int kMaxCluster = 8;
constexpr uint32_t kFull = 0xffffffffu;

struct Params {
  const __nv_bfloat16* x;
  int64_t ldx;
  const __nv_bfloat16* scales;  // [N][groups]
  const uint8_t* zeros;         // [N][groups] or null (8)
  __nv_bfloat16* out;
  int64_t ldo;
  int m, n, k, groups;
  int group_boxes;  // 128-k spans of one group, for groups of 128 and more
  int subs;        // boxes along k
  int subs_cta;    // boxes of one CTA of the cluster
  int chunk_subs;  // boxes whose token rows are staged at a time
  int cluster;
  int32_t* status;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Nibbles s and s + 4 of a word as the bf16 pair (128 + q_s, 128 + q_{s+4}).
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int s) { return ((w >> (4 * s)) & 0x000f000fu) | 0x43004300u; }

__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NT: tiles of 8 tokens. GI: 32-k blocks that share a scale within a box (1, 2, or 4 for groups of 128
// and multiples of it).
template <int NT, int GI>
__global__ void __launch_bounds__(kWarps * 32, 2) gemv_kernel(const __grid_constant__ CUtensorMap wmap, const Params p) {
  pdl_trigger();
  constexpr int MP = NT * 8;
  constexpr int GN = 8 / GI;  // scales of a row in one box
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t s_bar[kWarps][kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = p.cluster > 1 ? blockIdx.x % p.cluster : 0;
  const int row_cta = blockIdx.x / p.cluster * (kWarps * kRows);
  const int row0 = row_cta + warp * kRows;
  const int sub0 = rank * p.subs_cta;
  const int subs = max(0, min(p.subs_cta, p.subs - sub0));
  const int tok0 = blockIdx.y * MP;
  uint8_t* ring = smem + warp * kStages * kTile;
  const uint32_t ring_u = smem_u32(ring);
  // token rows: 16-byte chunks of 8 k in the order (0,4) (1,5) (2,6) (3,7), rows 4 chunks (mod 8) apart
  uint8_t* xs = smem + kWarps * kStages * kTile;
  const int pitch = p.chunk_subs * 512 + 64;
  float* xsum = reinterpret_cast<float*>(xs + MP * pitch);  // [chunk_subs * GN][MP]
  const bool live = row0 < p.n;

  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&s_bar[warp][i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  auto issue = [&](int i) {  // box i of this warp's share; lane 0
    const uint32_t bar = smem_u32(&s_bar[warp][i % kStages]);
    mbar_arrive_expect_tx(&s_bar[warp][i % kStages], kTile);
    tma_load_2d(ring_u + (i % kStages) * kTile, &wmap, bar, (sub0 + i) * (kSub / 2), row0);
  };
  // The weights come from no kernel of this library, so their loads need not wait for the predecessor.
  int issued = 0;
  if (live)
    for (; issued < kStages && issued < subs; ++issued)
      if (lane == 0) issue(issued);
  pdl_wait();

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  const int64_t ra = (int64_t)min(row0 + g, p.n - 1) * p.groups, rb = (int64_t)min(row0 + g + 8, p.n - 1) * p.groups;
  const __nv_bfloat16 *scale_a = p.scales + ra, *scale_b = p.scales + rb;
  const uint8_t *zero_a = p.zeros + ra, *zero_b = p.zeros + rb;
  bool ok = true;

  for (int c0 = 0; c0 < subs; c0 += p.chunk_subs) {
    const int cn = min(p.chunk_subs, subs - c0);
    if (c0 > 0) __syncthreads();
    // stage this chunk's token rows and their group sums: a warp takes one box of one token at a time
    for (int j = warp; j < MP * cn; j += kWarps) {
      const int tok = j / cn, sb = j - tok * cn;
      const int k = (sub0 + c0 + sb) * kSub + lane * 8;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (tok0 + tok < p.m && k < p.k) v = *reinterpret_cast<const uint4*>(p.x + (int64_t)(tok0 + tok) * p.ldx + k);
      uint4 o;
      o.x = __byte_perm(v.x, v.z, 0x5410);
      o.y = __byte_perm(v.x, v.z, 0x7632);
      o.z = __byte_perm(v.y, v.w, 0x5410);
      o.w = __byte_perm(v.y, v.w, 0x7632);
      *reinterpret_cast<uint4*>(xs + tok * pitch + sb * 512 + lane * 16) = o;
      float sum = ((bf16lo(v.x) + bf16hi(v.x)) + (bf16lo(v.y) + bf16hi(v.y))) +
                  ((bf16lo(v.z) + bf16hi(v.z)) + (bf16lo(v.w) + bf16hi(v.w)));
#pragma unroll
      for (int d = 1; d < 4 * GI; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
      if (lane % (4 * GI) == 0) xsum[(sb * GN + lane / (4 * GI)) * MP + tok] = sum;
    }
    __syncthreads();
    if (!live || !ok) continue;  // (every warp passes the CTA's barriers)
    for (int i = c0; i < c0 + cn; ++i) {
      // this box's scales and offsets 128 + z, two weight rows a lane
      float sa[GN], sb[GN], za[GN], zb[GN];
#pragma unroll
      for (int j = 0; j < GN; ++j) {
        int grp = (sub0 + i) * GN + j;
        if (GI == 4 && p.group_boxes > 1) grp /= p.group_boxes;
        grp = min(grp, p.groups - 1);  // a box may reach past k: its x are zeros there
        sa[j] = bf16_to_f(scale_a[grp]);
        sb[j] = bf16_to_f(scale_b[grp]);
        za[j] = zb[j] = 136.f;
        if (p.zeros != nullptr) {
          za[j] = (float)(128 + zero_a[grp]);
          zb[j] = (float)(128 + zero_b[grp]);
        }
      }
      ok = ok && __all_sync(kFull, mbar_wait(&s_bar[warp][i % kStages], (i / kStages) & 1, p.status));
      if (!ok) break;
      const uint8_t* w = ring + (i % kStages) * kTile + g * 128 + t * 4;
      const uint8_t* xr = xs + g * pitch + (i - c0) * 512 + t * 16;
      float part[NT][4];
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        if (b % GI == 0) {
#pragma unroll
          for (int j = 0; j < NT; ++j) part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.f;
        }
        const uint32_t wa = *reinterpret_cast<const uint32_t*>(w + ((b ^ g) << 4));
        const uint32_t wb = *reinterpret_cast<const uint32_t*>(w + 1024 + ((b ^ g) << 4));
        uint32_t ea[4], eb[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) ea[s] = nibbles(wa, s), eb[s] = nibbles(wb, s);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 xv = *reinterpret_cast<const uint4*>(xr + j * 8 * pitch + b * 64);
          mma_bf16(part[j], ea[0], eb[0], ea[1], eb[1], xv.x, xv.y);
          mma_bf16(part[j], ea[2], eb[2], ea[3], eb[3], xv.z, xv.w);
        }
        if (b % GI == GI - 1) {
          const int grp = b / GI;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float2 sx =
                *reinterpret_cast<const float2*>(xsum + ((i - c0) * GN + grp) * MP + j * 8 + 2 * t);
            acc[j][0] = fmaf(sa[grp], fmaf(-za[grp], sx.x, part[j][0]), acc[j][0]);
            acc[j][1] = fmaf(sa[grp], fmaf(-za[grp], sx.y, part[j][1]), acc[j][1]);
            acc[j][2] = fmaf(sb[grp], fmaf(-zb[grp], sx.x, part[j][2]), acc[j][2]);
            acc[j][3] = fmaf(sb[grp], fmaf(-zb[grp], sx.y, part[j][3]), acc[j][3]);
          }
        }
      }
      __syncwarp();
      if (issued < subs) {
        if (lane == 0) issue(issued);
        ++issued;
      }
    }
    if (!ok) {  // a box that never came: the error is recorded; wait for the others in flight
      for (int i = c0; i < issued; ++i) mbar_wait(&s_bar[warp][i % kStages], (i / kStages) & 1, p.status);
    }
  }
  __syncthreads();

  // partials [token][128 rows] over the token rows' place, then summed over the cluster and written
  float* part = reinterpret_cast<float*>(xs);
  constexpr int PR = kWarps * kRows + 4;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* at = part + (j * 8 + 2 * t) * PR + warp * kRows + g;
    at[0] = acc[j][0];
    at[PR] = acc[j][1];
    at[8] = acc[j][2];
    at[PR + 8] = acc[j][3];
  }
  const int tokens = min(MP, p.m - tok0);
  if (p.cluster > 1) cluster_sync(); else __syncthreads();
  const uint32_t part_u = smem_u32(part);
  for (int i = rank * (kWarps * 32) + threadIdx.x; i < tokens * (kWarps * kRows); i += p.cluster * kWarps * 32) {
    const int tok = i / (kWarps * kRows), r = i - tok * (kWarps * kRows);
    float v = 0.f;
    if (p.cluster > 1) {
      for (int c = 0; c < p.cluster; ++c) v += ld_cluster(map_to_rank(part_u + (tok * PR + r) * 4, c));
    } else {
      v = part[tok * PR + r];
    }
    if (row_cta + r < p.n) p.out[(int64_t)(tok0 + tok) * p.ldo + row_cta + r] = f_to_bf16(v);
  }
  if (p.cluster > 1) cluster_sync();  // nobody leaves while its partials are read
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &st) != cudaSuccess ||
        st != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  return fn;
}

template <int NT, int GI>
static int launch(const CUtensorMap& map, const Params& p, dim3 grid, cudaStream_t st) {
  constexpr int MP = NT * 8;
  size_t tail = (size_t)MP * (p.chunk_subs * 512 + 64) + (size_t)p.chunk_subs * (8 / GI) * MP * 4;
  const size_t parts = (size_t)MP * (kWarps * kRows + 4) * 4;
  if (tail < parts) tail = parts;
  const size_t smem = 1024 + (size_t)kWarps * kStages * kTile + tail;
  auto kernel = gemv_kernel<NT, GI>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return CDB_ERR_CUDA;
  prefer_max_shared(reinterpret_cast<const void*>(kernel));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, map, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

template <int GI>
static int launch_tokens(const CUtensorMap& map, const Params& p, dim3 grid, int nt, cudaStream_t st) {
  if (nt == 1) return launch<1, GI>(map, p, grid, st);
  if (nt == 2) return launch<2, GI>(map, p, grid, st);
  if (nt == 3) return launch<3, GI>(map, p, grid, st);
  return launch<4, GI>(map, p, grid, st);
}

}  // namespace w4
}  // namespace cdb

extern "C" int cdb_gemv_w4(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* scales,
                           const void* zeros, void* out, int64_t ldo, int M, int N, int K, int group_size, int num_sms,
                           int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::w4;
  if (M < 0 || N <= 0 || K <= 0 || num_sms <= 0 || K % 32 != 0 || group_size <= 0 || K % group_size != 0 ||
      (group_size != 32 && group_size != 64 && group_size % 128 != 0))
    return CDB_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || (ldx & 7) || ldx < K || (reinterpret_cast<uintptr_t>(w) & 15) ||
      (ldw & 15) || ldw < K / 2 || (reinterpret_cast<uintptr_t>(scales) & 1) ||
      (reinterpret_cast<uintptr_t>(out) & 1) || ldo < N)
    return CDB_ERR_INVALID_ARGUMENT;
  if (M == 0) return CDB_OK;
  if (x == nullptr || w == nullptr || scales == nullptr || out == nullptr) return CDB_ERR_INVALID_ARGUMENT;
  if (M > 32 * 65535) return CDB_ERR_INVALID_ARGUMENT;
  EncodeFn encode = encode_fn();
  if (encode == nullptr) return CDB_ERR_TMA_ENCODE;
  CUtensorMap map;
  const cuuint64_t dims[2] = {(cuuint64_t)(K / 2), (cuuint64_t)N};
  const cuuint64_t strides[1] = {(cuuint64_t)ldw};
  const cuuint32_t box[2] = {kSub / 2, kRows};
  const cuuint32_t ones[2] = {1, 1};
  if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(w), dims, strides, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return CDB_ERR_TMA_ENCODE;
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.scales = static_cast<const __nv_bfloat16*>(scales);
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.m = M;
  p.n = N;
  p.k = K;
  p.group_boxes = group_size > 128 ? group_size / 128 : 1;
  p.groups = K / group_size;
  p.subs = (K + kSub - 1) / kSub;
  p.status = status;
  const int nt = M > 24 ? 4 : (M + 7) / 8;
  const int row_ctas = (N + kWarps * kRows - 1) / (kWarps * kRows);
  // Split k over the cluster size that leaves the fewest boxes to the busiest of the 2 num_sms resident
  // CTAs (rounds of CTAs times boxes of one); the smaller cluster where two are alike.
  int cluster = 1;
  for (int c = 1, best = 0; c <= kMaxCluster && c <= p.subs; c *= 2) {
    const int rounds = (row_ctas * c + 2 * num_sms - 1) / (2 * num_sms), cost = rounds * ((p.subs + c - 1) / c);
    if (best == 0 || cost < best) best = cost, cluster = c;
  }
  p.cluster = cluster;
  p.subs_cta = (p.subs + cluster - 1) / cluster;
  p.chunk_subs = p.subs_cta < 64 / (nt * 8) ? p.subs_cta : (64 / (nt * 8) > 0 ? 64 / (nt * 8) : 1);
  if (p.chunk_subs < 1) p.chunk_subs = 1;
  const dim3 grid(row_ctas * cluster, (M + nt * 8 - 1) / (nt * 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (group_size == 32) return launch_tokens<1>(map, p, grid, nt, st);
  if (group_size == 64) return launch_tokens<2>(map, p, grid, nt, st);
  return launch_tokens<4>(map, p, grid, nt, st);
}
