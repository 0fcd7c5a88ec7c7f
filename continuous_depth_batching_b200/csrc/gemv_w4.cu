// Products of a few token rows with 4-bit weights:
//   out[m][n] = bf16( sum over groups j of s[n][j] * sum over k in group j of (q[n][k] - z[n][j]) x[m][k] )
// Weights q are nibbles, two to a byte along k (low nibble first), as they are stored; no layout pass.
//
// Bound by the weights' bytes, N K / 2, and by the instructions around a weight: seven for eight weights to
// take nibbles apart, then the products and each group's scale. One CTA of 16 or 24 warps an SM
// keeps its token rows in shared memory for good; `wk` warps share a tile of 16 weight rows, each with its
// part of k, and add their parts through shared memory; the groups of wk warps walk over the row tiles.
// A warp streams its boxes (16 rows x 128 bytes = 256 k, TMA with a 128-byte swizzle, so that the loads
// below hit every bank once) through a ring of its own, across row tiles, so nobody waits but at the sum.
//
// The products run on the tensor cores (bf16 m16n8k16: 16 weight rows, 8 tokens). A nibble q becomes
// the bf16 number 128 + q, exactly, when a byte 0x43 is set above it, and the offset is taken
// off per group with the group's sum of x:
//   sum (q - z) x = sum (128 + q) x - (128 + z) sum x,
// both sums in fp32, then times the group's scale into the fp32 result: no weight is rounded. What the
// offset cancels costs fp32's 2^-24 of 128 sum |x|, far below bf16's rounding of the result.
//
// Token rows are kept whole, so only as many as fit beside the rings share one pass over the weights: 32 up to K =
// 1792, 27 to 29 by group size at K = 2048, 16 at 4096, 11 or 12 at 5632, 6 at 8192, 3 at 14336. More of them take
// another pass each time (grid y).
//
// Measured (weights of other layers between two calls, so from HBM; a graph of such calls; groups of 128): 2048 x 5632,
// 1 token 5.3 us; 11264 x 2048, 24 tokens 11.5 us, 32 tokens, in two passes, 17.5; 49152 x 2048, 8 tokens 19 us
// (2.8 TB/s; 20 us at groups of 64, 25 at 32). cdb_gemm_bf16 on the same shapes takes 9.2, 11.6, 11.6 and 37 us. A call
// costs some 4.5 us before and after its boxes: launch, token rows, the first box's latency, the sum. The rest goes
// on instructions, about 465 a box of 16 x 256 weights, all counted, with the ALU pipe, which takes a nibble apart,
// the fullest.
// 24 warps against 16 for 8 tokens: 18.1 against 19.5 us (49152 x 2048, weights in L2).
#include <cuda.h>

#include "cdb_common.cuh"

namespace cdb {
namespace w4 {

// Warps of a CTA (one CTA an SM) by its tiles of 8 tokens: one tile fits 80 registers a thread.
__host__ __device__ constexpr int warps_of(int nt) { return nt == 1 ? 24 : 16; }
constexpr int kRows = 16;  // weight rows of a tile
constexpr int kSub = 256;  // k of one TMA box (128 bytes of a row)
constexpr int kTile = kRows * kSub / 2;
constexpr int kPart = 20;  // pitch of 16 rows' sums: spreads the stores over the banks
constexpr int kMaxStages = 4;
constexpr int kSmem = 226 * 1024;  // dynamic shared memory that a CTA may take
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
  int subs;    // boxes along k
  int tiles;   // row tiles
  int wk;      // warps that share a row tile
  int tokens;  // token rows of a CTA (grid y counts blocks of them)
  int stages;
  // quotients, which the device would take some 30 instructions each for
  int by_wk, by_subs;      // 65536 / wk and / subs, rounded up: (warp * by_wk) >> 16 is warp / wk
  int each;                // boxes along k of one of wk warps
  int row_groups;          // groups of wk warps in the grid
  int rounds, rest;        // row tiles of each, and of how many one more
  int step_tok, step_sub;  // warps of a CTA / subs, and the remainder
  int32_t* status;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// The words of rows g and g + 8 of a box.
__device__ __forceinline__ void load_rows(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ld.shared.b32 %0, [%2];\n\tld.shared.b32 %1, [%2+1024];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B: the first product of a sum.
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The 8 nibbles of a word as bf16 pairs 128 + q, of k (0, 2) (4, 6) (1, 3) (5, 7): the nibbles become bytes,
// two at a time, and the byte 0x43 above one makes it 128 + q. Seven instructions for eight weights.
__device__ __forceinline__ void nibbles(uint32_t w, uint32_t (&e)[4]) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  e[0] = __byte_perm(even, 0x43434343u, 0x4140);
  e[1] = __byte_perm(even, 0x43434343u, 0x4342);
  e[2] = __byte_perm(odd, 0x43434343u, 0x4140);
  e[3] = __byte_perm(odd, 0x43434343u, 0x4342);
}

// The scales and zero points of a box for this lane's rows, g and g + 8: scale bits, and 128 + zero point (2^15 + z
// by bits, less 2^15 - 128).
__device__ __forceinline__ float zero_of(uint32_t word, int byte) {
  return __uint_as_float(__byte_perm(word, 0x47000000u, 0x7404 | byte << 4)) - 32640.f;
}

// WIDE: a row's scales of a box lie together and aligned, and every lane loads those of its two rows at once.
template <int GN, bool WIDE>
struct Entries;

template <int GN>
struct Entries<GN, true> {
  uint32_t s[2][GN / 2], z[2];  // per row: GN bf16, GN bytes (8 at most: two words)
  uint32_t z2[2];
  __device__ __forceinline__ void load(const __nv_bfloat16* scale, const uint8_t* zero, int to8, bool zeros) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const __nv_bfloat16* a = scale + r * to8;
      if constexpr (GN == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(a);
        s[r][0] = v.x, s[r][1] = v.y, s[r][2] = v.z, s[r][3] = v.w;
      } else if constexpr (GN == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(a);
        s[r][0] = v.x, s[r][1] = v.y;
      } else {
        s[r][0] = *reinterpret_cast<const uint32_t*>(a);
      }
      z[r] = z2[r] = 0x08080808u;
      if (zeros) {
        const uint8_t* b = zero + r * to8;
        if constexpr (GN == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(b);
          z[r] = v.x, z2[r] = v.y;
        } else if constexpr (GN == 4) {
          z[r] = *reinterpret_cast<const uint32_t*>(b);
        } else {
          z[r] = *reinterpret_cast<const uint16_t*>(b);
        }
      }
    }
  }
  __device__ __forceinline__ void get(int r, int grp, float& scale, float& zero) const {
    const uint32_t w = s[r][grp / 2];
    scale = __uint_as_float(grp & 1 ? w & 0xffff0000u : w << 16);
    zero = zero_of(grp < 4 ? z[r] : z2[r], grp & 3);
  }
};

// Otherwise: 2 GN (row half, group) entries, each loaded once in the four lanes of a row (entry e in lane e % 4) as
// scale bits and zero point in one word.
template <int GN>
struct Entries<GN, false> {
  uint32_t e[GN / 2];
  __device__ __forceinline__ void get(int r, int grp, float& scale, float& zero) const {
    const uint32_t w = __shfl_sync(kFull, e[(r * GN + grp) / 4], (r * GN + grp) % 4, 4);
    scale = __uint_as_float(w & 0xffff0000u);
    zero = zero_of(w, 0);
  }
};

// NT: tiles of 8 tokens. GI: 32-k blocks that share a scale within a box (1, 2, or 4 for groups of 128
// and multiples of it).
template <int NT, int GI, bool WIDE>
__global__ void __launch_bounds__(warps_of(NT) * 32, 1) gemv_kernel(const __grid_constant__ CUtensorMap wmap, const Params p) {
  pdl_trigger();
  constexpr int GN = 8 / GI;  // scales of a row in one box
  constexpr int kWarps = warps_of(NT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t s_bar[kWarps][kMaxStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tok0 = blockIdx.y * p.tokens;
  const int tokens = min(p.tokens, p.m - tok0);
  uint8_t* ring = smem + warp * p.stages * kTile;
  const uint32_t ring_u = smem_u32(ring), bar_u = smem_u32(&s_bar[warp][0]);
  // token rows: 16-byte chunks of 8 k in the order of nibbles(), rows 4 chunks (mod 8) apart
  uint8_t* xs = smem + kWarps * p.stages * kTile;
  const int pitch = p.subs * 512 + 64;
  float* xsum = reinterpret_cast<float*>(xs + p.tokens * pitch);  // [subs * GN][NT * 8]
  float* parts = xsum + p.subs * GN * NT * 8;                     // [warp][NT * 8][kPart], where wk > 1

  // this warp's place: part `part` of row tiles group, group + groups, ...
  const int team = (warp * p.by_wk) >> 16, part = warp - team * p.wk;
  const int groups = p.row_groups;
  const int group = blockIdx.x + gridDim.x * team;  // few tiles spread over the SMs first
  const int sub0 = part * p.each, subs = max(0, min(p.each, p.subs - sub0));
  const int rounds = p.rounds + (group < p.rest ? 1 : 0);
  const int boxes = rounds * subs;

  if (lane == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&s_bar[warp][i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  // The next box to load: box `at_sub` of row tile `at_tile`, into place `put`.
  int issued = 0, put = 0, at_sub = 0, at_tile = group;
  auto issue = [&]() {
    if (lane == 0) {
      mbar_arrive_expect_tx(&s_bar[warp][put], kTile);
      tma_load_2d(ring_u + put * kTile, &wmap, bar_u + put * 8, (sub0 + at_sub) * (kSub / 2), at_tile * kRows);
    }
    put = put + 1 == p.stages ? 0 : put + 1;
    ++issued;
    if (++at_sub == subs) {
      at_sub = 0;
      at_tile += groups;
    }
  };
  // The weights wait for the predecessor too, which may have written them: loading them ahead of it measured
  // 0.05 to 0.3 us a call.
  pdl_wait();
  while (issued < p.stages && issued < boxes) issue();
  // The scales and zero points of a box, loaded a box ahead of their use.
  constexpr int EN = WIDE ? 1 : GN / 2;
  Entries<GN, WIDE> entry;
  int64_t entry_at[EN];  // each row's first
  int to8 = 0;           // WIDE: from the scales of row g to those of row g + 8
  auto entry_tile = [&](int tile) {
#pragma unroll
    for (int k = 0; k < EN; ++k) {
      const int at = min(tile * kRows + g + (WIDE ? 0 : 8 * ((t + 4 * k) / GN)), p.n - 1);
      if (WIDE) to8 = (min(tile * kRows + g + 8, p.n - 1) - at) * p.groups;
      entry_at[k] = (int64_t)at * p.groups;
    }
  };
  auto load_entries = [&](int i) {
    if constexpr (WIDE) {
      const int64_t at = entry_at[0] + (sub0 + i) * GN;
      entry.load(p.scales + at, p.zeros + at, to8, p.zeros != nullptr);
    } else {
#pragma unroll
      for (int k = 0; k < EN; ++k) {
        int grp = (sub0 + i) * GN + (t + 4 * k) % GN;
        if (GI == 4 && p.group_boxes > 1) grp /= p.group_boxes;
        grp = min(grp, p.groups - 1);  // a box may reach past k, onto zeros of x
        const int64_t at = entry_at[k] + grp;
        entry.e[k] = ((uint32_t)__bfloat16_as_ushort(p.scales[at]) << 16) | (p.zeros != nullptr ? p.zeros[at] : 8u);
      }
    }
  };
  if (boxes > 0) {
    entry_tile(group);
    load_entries(0);
  }

  // the token rows and the sums of x over each group: a warp takes boxes of tokens, several loads in flight
  constexpr int AT_ONCE = 2 * NT;
  {
    int tok = (warp * p.by_subs) >> 16, sub = warp - tok * p.subs;  // this warp's next box of tokens
    while (tok < tokens) {
      uint4 v[AT_ONCE];
      int toks[AT_ONCE], places[AT_ONCE];
#pragma unroll
      for (int a = 0; a < AT_ONCE; ++a) {
        const int k = sub * kSub + lane * 8;
        v[a] = make_uint4(0u, 0u, 0u, 0u);
        if (tok < tokens && k < p.k) v[a] = *reinterpret_cast<const uint4*>(p.x + (int64_t)(tok0 + tok) * p.ldx + k);
        toks[a] = tok;
        places[a] = sub;
        tok += p.step_tok;
        sub += p.step_sub;
        if (sub >= p.subs) sub -= p.subs, ++tok;
      }
      float sum[AT_ONCE];
#pragma unroll
      for (int a = 0; a < AT_ONCE; ++a)
        sum[a] = ((bf16lo(v[a].x) + bf16hi(v[a].x)) + (bf16lo(v[a].y) + bf16hi(v[a].y))) +
                 ((bf16lo(v[a].z) + bf16hi(v[a].z)) + (bf16lo(v[a].w) + bf16hi(v[a].w)));
#pragma unroll
      for (int d = 1; d < 4 * GI; d <<= 1) {
#pragma unroll
        for (int a = 0; a < AT_ONCE; ++a) sum[a] += __shfl_xor_sync(kFull, sum[a], d);
      }
#pragma unroll
      for (int a = 0; a < AT_ONCE; ++a) {
        if (toks[a] >= tokens) break;
        *reinterpret_cast<uint4*>(xs + toks[a] * pitch + places[a] * 512 + lane * 16) =
            make_uint4(__byte_perm(v[a].x, v[a].y, 0x5410), __byte_perm(v[a].z, v[a].w, 0x5410),
                       __byte_perm(v[a].x, v[a].y, 0x7632), __byte_perm(v[a].z, v[a].w, 0x7632));
        if (lane % (4 * GI) == 0) xsum[(places[a] * GN + lane / (4 * GI)) * (NT * 8) + toks[a]] = sum[a];
      }
    }
  }
  __syncthreads();

  // columns past the tokens multiply the last one; nobody reads what comes of it
  const uint8_t* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) xrow[j] = xs + min(j * 8 + g, tokens - 1) * pitch + sub0 * 512 + t * 16;
  const float* sums = xsum + sub0 * GN * (NT * 8) + 2 * t;
  int get = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int round = 0, tile = group; round < rounds; ++round, tile += groups) {
    const int row0 = tile * kRows;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    for (int i = 0; i < subs; ++i) {
      const Entries<GN, WIDE> now = entry;
      if (i + 1 < subs) {
        load_entries(i + 1);
      } else if (round + 1 < rounds) {
        entry_tile(tile + groups);
        load_entries(0);
      }
      if (!__all_sync(kFull, mbar_try_wait(&s_bar[warp][get], phase)) &&
          !__all_sync(kFull, mbar_wait(&s_bar[warp][get], phase, p.status))) {
        ok = false;
        break;
      }
      // word b of row g lies at (b ^ g) * 16: the place of word 0, with b's bits turned over
      const uint32_t w = ring_u + get * kTile + g * 128 + (g << 4) + t * 4;
      float prod[NT][4];
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        uint32_t wa, wb;
        load_rows(w ^ (b << 4), wa, wb);
        uint32_t ea[4], eb[4];
        nibbles(wa, ea);
        nibbles(wb, eb);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 xv = *reinterpret_cast<const uint4*>(xrow[j] + i * 512 + b * 64);
          if (b % GI == 0) mma_bf16_first(prod[j], ea[0], eb[0], ea[1], eb[1], xv.x, xv.y);
          else mma_bf16(prod[j], ea[0], eb[0], ea[1], eb[1], xv.x, xv.y);
          mma_bf16(prod[j], ea[2], eb[2], ea[3], eb[3], xv.z, xv.w);
        }
        if (b % GI == GI - 1) {
          const int grp = b / GI;
          float sa, sb, za, zb;
          now.get(0, grp, sa, za);
          now.get(1, grp, sb, zb);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float2 sx = *reinterpret_cast<const float2*>(sums + (i * GN + grp) * (NT * 8) + j * 8);
            acc[j][0] = fmaf(sa, fmaf(-za, sx.x, prod[j][0]), acc[j][0]);
            acc[j][1] = fmaf(sa, fmaf(-za, sx.y, prod[j][1]), acc[j][1]);
            acc[j][2] = fmaf(sb, fmaf(-zb, sx.x, prod[j][2]), acc[j][2]);
            acc[j][3] = fmaf(sb, fmaf(-zb, sx.y, prod[j][3]), acc[j][3]);
          }
        }
      }
      get = get + 1 == p.stages ? (phase ^= 1u, 0) : get + 1;
      __syncwarp();
      if (issued < boxes) issue();
    }
    if (p.wk == 1) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int tok = j * 8 + 2 * t + (c & 1), row = row0 + g + 8 * (c >> 1);
          if (tok < tokens && row < p.n) p.out[(int64_t)(tok0 + tok) * p.ldo + row] = f_to_bf16(acc[j][c]);
        }
      }
      continue;
    }
    // the wk warps' parts, added in order
    constexpr int PART = NT * 8 * kPart;
    float* mine = parts + warp * PART;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 4; ++c) mine[(j * 8 + 2 * t + (c & 1)) * kPart + g + 8 * (c >> 1)] = acc[j][c];
    }
    const int id = 1 + team, threads = p.wk * 32;
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
    const float* from = parts + (warp - part) * PART;
    const int row = lane % kRows;
    __nv_bfloat16* dst = p.out + (int64_t)tok0 * p.ldo + row0 + row;
#pragma unroll 4
    for (int tok = part * 2 + lane / kRows; tok < tokens; tok += p.wk * 2) {
      float v = from[tok * kPart + row];
#pragma unroll 4
      for (int w = 1; w < p.wk; ++w) v += from[w * PART + tok * kPart + row];
      if (row0 + row < p.n) dst[(int64_t)tok * p.ldo] = f_to_bf16(v);
    }
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
  }
  if (!ok) {  // a box that never came: the error is recorded; wait for the others in flight
    for (int i = 0; i < p.stages; ++i) {
      get = get + 1 == p.stages ? (phase ^= 1u, 0) : get + 1;
      if (i + 1 < issued) mbar_wait(&s_bar[warp][get], phase, p.status);
    }
  }
}

// Bytes of a CTA's shared memory but for the ring.
static int64_t row_bytes(int subs, int nt, int gi, int tokens, int wk) {
  const int kWarps = warps_of(nt);
  return 1024 + (int64_t)tokens * (subs * 512 + 64) + (int64_t)subs * (8 / gi) * nt * 8 * 4 +
         (wk > 1 ? (int64_t)kWarps * kPart * nt * 8 * 4 : 0);
}

template <int NT, int GI, bool WIDE>
static int launch(const CUtensorMap& map, Params p, dim3 grid, cudaStream_t st) {
  constexpr int kWarps = warps_of(NT);
  const int64_t rest = row_bytes(p.subs, NT, GI, p.tokens, p.wk);
  p.stages = (int)((kSmem - rest) / (kWarps * kTile));
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const size_t smem = rest + (size_t)kWarps * p.stages * kTile;
  auto kernel = gemv_kernel<NT, GI, WIDE>;
  if (allow_shared(reinterpret_cast<const void*>(kernel), kSmem) != cudaSuccess) return CDB_ERR_CUDA;
  return launch_pdl(kernel, grid, dim3(kWarps * 32), smem, st, map, p) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

template <int GI, bool WIDE>
static int launch_tokens(const CUtensorMap& map, const Params& p, dim3 grid, int nt, cudaStream_t st) {
  if (nt == 1) return launch<1, GI, WIDE>(map, p, grid, st);
  if (nt == 2) return launch<2, GI, WIDE>(map, p, grid, st);
  if (nt == 3) return launch<3, GI, WIDE>(map, p, grid, st);
  return launch<4, GI, WIDE>(map, p, grid, st);
}

// A row's scales of a box are loaded together where every box has all its groups and their places are aligned.
// Against one at a time: 5.2 us for 5.5 (2048 x 5632, 1 token), 21.3 for 22.7 (49152 x 2048, 8 tokens, groups of
// 64), 12.8 for 14.7 (6144 x 2048, 32 tokens, groups of 64); the same at groups of 32.
template <int GI>
static int launch_groups(const CUtensorMap& map, const Params& p, dim3 grid, int nt, cudaStream_t st) {
  constexpr int GN = 8 / GI;
  const bool wide = p.group_boxes == 1 && p.groups % GN == 0 && reinterpret_cast<uintptr_t>(p.scales) % (2 * GN) == 0 &&
                    reinterpret_cast<uintptr_t>(p.zeros) % GN == 0;
  return wide ? launch_tokens<GI, true>(map, p, grid, nt, st) : launch_tokens<GI, false>(map, p, grid, nt, st);
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
  if (M > 65535) return CDB_ERR_INVALID_ARGUMENT;
  EncodeFn encode = tensor_map_encoder();
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
  p.tiles = (N + kRows - 1) / kRows;
  const int gi = group_size == 32 ? 1 : group_size == 64 ? 2 : 4;
  // Token rows of a CTA: as many (up to 32) as fit beside a ring of two boxes a warp, in equal blocks.
  int most = 0;
  for (int nt = 1; nt <= 4; ++nt)
    for (int tok = nt * 8 - 7; tok <= nt * 8; ++tok)
      if (row_bytes(p.subs, nt, gi, tok, 2) + 2 * warps_of(nt) * kTile <= kSmem) most = tok;
  if (most == 0) return CDB_ERR_UNSUPPORTED;  // K so long that one token row does not fit
  const int blocks = (M + most - 1) / most;
  p.tokens = (M + blocks - 1) / blocks;
  int nt = (p.tokens + 7) / 8;  // one tile's 24 rings may not fit where two tiles' 16 do
  while (row_bytes(p.subs, nt, gi, p.tokens, 2) + 2 * warps_of(nt) * kTile > kSmem) ++nt;
  // Warps on a row tile: the fewest boxes one after another in a warp (a sum over warps counted as half of
  // one), for the row tiles that an SM gets. Few row tiles spread over k that way
  const int ctas = p.tiles < num_sms ? p.tiles : num_sms, share = (p.tiles + ctas - 1) / ctas;
  p.wk = 1;
  const int warps = warps_of(nt);
  for (int w = 1, best = 0; w <= warps && w <= p.subs; ++w) {
    if (warps % w != 0) continue;
    const int rounds = (share + warps / w - 1) / (warps / w);
    const int cost = rounds * (2 * ((p.subs + w - 1) / w) + (w > 1 ? 1 : 0));
    if (best == 0 || cost < best) best = cost, p.wk = w;
  }
  p.by_wk = (65536 + p.wk - 1) / p.wk;
  p.by_subs = (65536 + p.subs - 1) / p.subs;
  p.each = (p.subs + p.wk - 1) / p.wk;
  p.row_groups = ctas * (warps / p.wk);
  p.rounds = p.tiles / p.row_groups;
  p.rest = p.tiles % p.row_groups;
  p.step_tok = warps / p.subs;
  p.step_sub = warps % p.subs;
  const dim3 grid(ctas, blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (gi == 1) return launch_groups<1>(map, p, grid, nt, st);
  if (gi == 2) return launch_groups<2>(map, p, grid, nt, st);
  return launch_groups<4>(map, p, grid, nt, st);
}
