// Causal prefill attention over the 8-bit paged cache (layout in kv8.cuh): tiles of up to 64
// consecutive query rows of one request, as cdb_prefill_attention takes them, any number of query heads
// per kv head.
//
// A CTA takes 128 query rows of one head: a tile and, where the list has it beside it, the request's next one (so
// a long chunk fills the tensor core's 128 rows; a lone tile leaves half of them idle). Keys come in steps of
// 64 (4 blocks). Roles:
//   warps 0..3   softmax: thread r owns query row r, so its maximum, sum and weights need no exchange;
//   warps 4..7   turn the codes into f16, exactly, in the tensor core's layout: K as it lies, V transposed;
//   warps 8, 9   issue the products, S = Q K^T (128 x 64 x D) and O += P V (128 x D x 64);
//   warps 10, 11 bring the codes of K and of V: bulk copies of whole (block, head) tiles, two steps ahead.
// The softmax takes 136 of the registers, the conversion 72 and the rest 32 a thread (setmaxnreg; 80 at launch).
// Both products are tcgen05 with f16 operands and fp32 accumulators in tensor memory. The softmax writes its
// weights P there too, over the S that they come from, so that P is as double as S and the softmax of a step
// need not wait for the product of the one before; V is double in shared memory for the same reason.
// Two CTAs share an SM (256 of its 512 tensor-memory columns, 113 KB of shared memory each): one computes
// exponentials while the other multiplies. A GEMM CTA that is launched early beside one of them holds its
// columns while it waits for this kernel; it has no room in shared memory beside two, and at most 256 columns
// where it fits beside one, so the allocation here never waits for a kernel that waits for this one.
//
// Arithmetic as in the decode kernel: q over a power of two per row, an online base-2 softmax with l relative
// to a maximum m of the logits x, the weights of V, w = 2^x s_v, relative to their own maximum M and rounded
// to f16 (kLift in kv8.cuh: by 2^-11, or 2^-32 of the largest). m and M move only when passed by 8, and then the row's
// O is rescaled in tensor memory.
// One exponential a key: w 2^(kLift - M) = 2^(S f + log2 s_v - M + kLift), and l takes the sum of a block's weights
// times the block's 2^(M - kLift - m) / s_v, unless that factor is so far from 1 that the weights could have underflowed.
//
// Measured: 4096 rows at positions 4096 .. 8191, 16 heads of 128: 312 us, 660 TFLOP/s; chunks of up to 400
// rows of 12 requests: 44 us, mostly the steps of the longest and a CTA's start. What bounds it is the softmax's way
// through a step, some 2600 of 3200 cycles a step of each of the two CTAs: load S, maximum, exponentials, store P,
// none of them long enough to hide the next one's latency. Tensor pipe 33% busy, shared memory's load and store
// path 45%, issue slots 55%, exponentials 36%. Tried: eight softmax warps with 16 rows each (four lanes a row) 349
// us, for a third more instructions; four more conversion warps 321 us; masks and the second sums in loops of their
// own, for less code, 313 us.
//
// A masked key never counts, whatever it holds: its logit is replaced, and a NaN in its V, which a product
// with weight zero would spread, is taken out in the steps that the diagonal crosses and put back at the end
// for the rows that see it.
#include "kv8.cuh"

namespace cdb {
namespace kv8 {

constexpr int TR = 64;   // rows of a listed tile
constexpr int TM = 128;  // rows of a CTA
constexpr int TK = 64;   // keys of a step
constexpr int kSoftmax = 128, kConvert = 128;  // threads of the softmax and of the conversion
constexpr int kPrefillThreads = kSoftmax + kConvert + 128;
constexpr int kMeta = 8;            // steps whose scales are kept (keys run up to five steps ahead of the softmax)
constexpr int kDiagonal = 3;        // steps that the diagonal of 128 rows can cross
static_assert(kPrefillThreads < 1024, "ten bits count a list of as many tiles");
constexpr uint32_t kTmemCols = 256;
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
  int num_tiles;
  int num_rows;  // rows of q and out
  float scale_log2;
  int32_t* status;
};

template <int D>
struct Tile {
  static constexpr int BLK = kBlock * D;          // bytes of one block's codes
  static constexpr int ATOMS = (D + 63) / 64;     // 128-byte swizzle atoms of a row of D f16
  static constexpr int VBLK = BLK + 32;           // a staged block of V: 32 bytes on spread the banks
  static constexpr int OFF_Q = 0;                 // f16 [ATOMS][128][64]
  static constexpr int OFF_K = OFF_Q + ATOMS * TM * 128;  // f16 [ATOMS][64][64]
  static constexpr int OFF_V = OFF_K + ATOMS * TK * 128;  // f16 [2][D][64 keys]
  static constexpr int OFF_SK = OFF_V + 2 * D * 128;      // codes [2][4 blocks]
  static constexpr int OFF_SV = OFF_SK + 2 * 4 * BLK;
  static constexpr int OFF_BAR = (OFF_SV + 2 * 4 * VBLK + 15) / 16 * 16;
  static constexpr int SMEM = OFF_BAR + 512;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

// Barriers and small state behind the tiles.
struct Shared {
  uint64_t staged_k[2], staged_v[2];  // a step's codes have landed (4 threads announce them)
  uint64_t qfull;            // q in f16 written
  uint64_t kready[2], vready[2];  // a step's K, V in f16 written (and its codes read)
  uint64_t sfull[2];         // a step's S product done (and K's place free) and its scales there
  uint64_t pfull[2], odone[2];  // weights written / a step's O product done (and its V's and S's places free)
  uint64_t meta[kMeta];      // a step's scales written
  uint64_t drain[2];         // all products done
  alignas(16) float scale[kMeta][2][4];  // K's (< 0: no such block) and V's, then V's log2
  unsigned long long nan[kDiagonal];
  uint32_t tmem;
  int abort;
  uint32_t counts;           // of the search for the tile's partner, and that one's rows
  int next;
};
static_assert(sizeof(Shared) <= 512 && alignof(Shared) == 16, "room behind the tiles");

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// 4 bytes to shared memory, asynchronously; async_arrive lets `bar` count their completion.
__device__ __forceinline__ void async_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Matrix descriptor of a K-major operand in 128-byte swizzled rows of 64 f16, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// D[tmem] (+)= A B^T, kind::f16 with f16 operands: fp32 accumulators, M = 128.
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  const uint32_t none = 0, acc = add;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(operand(a)), "l"(operand(b)), "r"(idesc), "r"(acc), "r"(none)
      : "memory");
}
// The same with A in tensor memory: two f16 to a 32-bit column, rows on lanes.
__device__ __forceinline__ void product_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  const uint32_t none = 0, acc = add;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(operand(b)), "r"(idesc), "r"(acc), "r"(none)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 tensor-memory lanes.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// 16 columns, there and back: the rescaling of O goes through few registers, beside the 64 of S.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}

// Waits for this thread's tensor-memory loads; the registers pass through it, so no use can move ahead.
__device__ __forceinline__ void wait_loads(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
               "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
               "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
               "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait that also gives up once another role has.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *abort) return false;
  }
  set_error(status, CDB_ERR_DEVICE_TIMEOUT);
  *abort = 1;
  return false;
}

// What a CTA does with the list entry that it was started for: its own rows and the partner's.
struct Rows {
  int row0, n, slot, pos;
};

__device__ __forceinline__ bool fits(const PrefillParams& p, int4 tile) {
  return tile.y <= TR && tile.x >= 0 && tile.x <= p.num_rows - tile.y && tile.z >= 0 && tile.z < p.bt_rows &&
         tile.w >= 0 && tile.w <= 0x7fffffff - 2 * TM && (tile.w + tile.y - 1) / kBlock < p.bt_width;
}

// Entry b holds the 64 rows after entry a's.
__device__ __forceinline__ bool follows(const PrefillParams& p, int4 a, int4 b) {
  return a.y == TR && b.y > 0 && fits(p, a) && fits(p, b) && b.z == a.z && b.w == a.w + TR && b.x == a.x + TR;
}

// Decides whether this entry stands alone, takes the request's next rows along, or is itself taken along (then n
// = 0), so that both ends of a pair decide alike and no row is left out (entries listed twice may be computed
// twice). Against every tile for itself: 16 requests of 1024 rows 266 us for 371.
//
// A list of up to a CTA's threads is searched whole, one entry to a thread (`mine`): a request's tiles are counted
// in order of position, one with an even count before it leads, entries that overlap another of their slot do not.
// In a longer list a tile whose position lies in an even 64 leads where its partner is beside it in the list,
// which costs no search: lone tiles, 1000 and 2000 of them, take 603 and 1200 us, searched 643 and 1352; pairs
// 600 and 1194, searched 643 and 1333. The order matters there: prompts of 384 rows, 16 heads of 128, longest tiles
// first (so few pairs) against request order, 64 prompts (384 tiles, searched) 216 us for 278, 80 (480) 345 for 335; 250
// prompts of 256 rows (1000 tiles) 637 for 599.
__device__ __forceinline__ Rows choose_rows(const PrefillParams& p, Shared& sh, int4 tile, int4 before, int4 after,
                                            int4 mine) {
  Rows me = {tile.x, tile.y, tile.z, tile.w};
  if (p.num_tiles > kPrefillThreads) {
    if ((tile.w / TR) % 2 == 0)
      me.n += max(follows(p, tile, before) ? before.y : 0, follows(p, tile, after) ? after.y : 0);
    else if (follows(p, before, tile) || follows(p, after, tile))
      me.n = 0;
    return me;
  }
  uint32_t counts = 0;  // of the slot's tiles before the one that may lead this, before this, before the next one
  bool lead = false;
  if (mine.y > 0 && mine.z == tile.z) {
    counts = (uint32_t)(mine.w < tile.w - TR) | (uint32_t)(mine.w < tile.w) << 10 | (uint32_t)(mine.w < tile.w + TR) << 20;
    lead = follows(p, mine, tile);
    if (follows(p, tile, mine)) atomicMax(&sh.next, mine.y);
  }
  counts = __reduce_add_sync(kAll, counts);
  if ((threadIdx.x & 31) == 0) atomicAdd(&sh.counts, counts);
  const bool led = __syncthreads_or(lead);
  const uint32_t c0 = sh.counts & 1023u, c1 = (sh.counts >> 10) & 1023u, c2 = sh.counts >> 20;
  if (led && c0 % 2 == 0 && c1 == c0 + 1) me.n = 0;
  else if (c1 % 2 == 0 && c2 == c1 + 1) me.n += sh.next;
  return me;
}

template <int D>
__global__ void __launch_bounds__(kPrefillThreads, 2) prefill_kernel(const PrefillParams p) {
  using T = Tile<D>;
  pdl_trigger();
  constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(TK >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  constexpr uint32_t kIdescO = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem + T::OFF_BAR);
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.staged_k[i], 4);
      mbar_init(&sh.staged_v[i], 4);
      mbar_init(&sh.drain[i], 1);
      mbar_init(&sh.kready[i], kConvert);
      mbar_init(&sh.vready[i], kConvert);
      mbar_init(&sh.sfull[i], 2);
      mbar_init(&sh.pfull[i], kSoftmax);
      mbar_init(&sh.odone[i], 1);
    }
    for (int i = 0; i < kMeta; ++i) mbar_init(&sh.meta[i], 8);
    mbar_init(&sh.qfull, kSoftmax);
    for (int i = 0; i < kDiagonal; ++i) sh.nan[i] = 0ull;
    sh.counts = 0u;
    sh.next = 0;
    sh.abort = (base & 1023u) != 0u;  // the swizzle counts on it
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();

  const int at_tile = blockIdx.y;
  const int4 tile = p.tiles[at_tile], none = make_int4(0, 0, 0, 0);
  const int4 before = at_tile > 0 ? p.tiles[at_tile - 1] : none;
  const int4 after = at_tile + 1 < p.num_tiles ? p.tiles[at_tile + 1] : none;
  const int4 mine = tid < p.num_tiles ? p.tiles[tid] : none;  // for the search below
  if (tile.y <= 0) return;  // an unused entry of the list
  if (!fits(p, tile) || sh.abort) {
    if (tid == 0) set_error(p.status, CDB_ERR_INDEX);
    return;
  }
  const Rows me = choose_rows(p, sh, tile, before, after, mine);
  if (me.n == 0) return;  // a neighbour takes these rows along
  const int head = blockIdx.x, kvh = head / p.heads_per_kv;
  const int kv_len = me.pos + me.n;
  const int steps = (kv_len + TK - 1) / TK, blocks = (kv_len + kBlock - 1) / kBlock;
  const int diagonal = me.pos / TK;  // the first step that holds a key which some row may not see
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;          // S: two buffers of 64 columns; O: 128 columns on
  const uint32_t tmem_o = tmem + 2 * TK;
  volatile int* abort = &sh.abort;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp >= 10) {
      // ------------------------------------------------------------ codes into shared memory
      const bool values = warp == 11;
      const int32_t* bt = p.block_table + (int64_t)me.slot * p.bt_stride;
      const int64_t first_tile = values ? (int64_t)p.num_blocks * p.kv_heads : 0;
      uint64_t* staged = values ? sh.staged_v : sh.staged_k;
      uint64_t* ready = values ? sh.vready : sh.kready;
      // Lanes 0..3 bring one block of every step each, its id a step ahead of its copies.
      int id = -1;
      auto fetch_id = [&](int step) {
        const int b = step * 4 + lane;
        id = lane < 4 && step < steps && b < blocks ? bt[b] : -1;
      };
      auto issue = [&](int step) {
        if (step >= steps || lane >= 4) return;
        uint64_t *bar = &staged[step & 1], *meta = &sh.meta[step & (kMeta - 1)];
        float* scale = &sh.scale[step & (kMeta - 1)][values][lane];
        const bool used = step * 4 + lane < blocks;
        if (used && id >= 0 && id < p.num_blocks) {
          const int64_t at = first_tile + (int64_t)id * p.kv_heads + kvh;
          const uint32_t place = (step & 1) * 4 + lane;
          mbar_arrive_expect_tx(bar, T::BLK);
          bulk_copy(base + (values ? T::OFF_SV + place * T::VBLK : T::OFF_SK + place * T::BLK), p.codes + at * T::BLK,
                    T::BLK, smem_u32(bar));
          async_copy4(smem_u32(scale), p.scales + at);
          async_arrive(smem_u32(meta));
        } else {
          if (used) set_error(p.status, CDB_ERR_INDEX);
          *scale = -1.f;
          mbar_arrive(meta);
          mbar_arrive(bar);
        }
      };
      fetch_id(0);
      issue(0);
      fetch_id(1);
      issue(1);
      fetch_id(2);
      int announced = min(2, steps);
      for (int n = 0; n + 2 < steps; ++n) {  // step n's codes have been read: their place takes step n + 2's
        if (!__all_sync(kAll, wait_for(&ready[n & 1], (n >> 1) & 1, p.status, abort))) break;
        issue(n + 2);
        fetch_id(n + 3);
        announced = n + 3;
      }
      for (int j = max(0, announced - 2); j < announced; ++j) mbar_wait(&staged[j & 1], (j >> 1) & 1, p.status);
    } else {
      // ------------------------------------------------------------ products
      if (warp == 8) {
        for (int n = 0; n < steps; ++n) {
          // The step's scales (the softmax wants V's logarithms), K and q; later also that the weights which lay
          // over the place of this S have been used.
          const int sl = n & (kMeta - 1);
          bool ok = wait_for(&sh.meta[sl], (n / kMeta) & 1, p.status, abort);
          if (lane < 4) sh.scale[sl][1][lane] = sh.scale[sl][1][lane] > 0.f ? __log2f(sh.scale[sl][1][lane]) : -126.f;
          ok = ok && wait_for(&sh.kready[n & 1], (n >> 1) & 1, p.status, abort) &&
               (n < 2 ? wait_for(&sh.qfull, 0, p.status, abort)
                      : wait_for(&sh.odone[n & 1], ((n - 2) >> 1) & 1, p.status, abort));
          if (!__all_sync(kAll, ok)) break;
          __syncwarp();  // lane 0's arrival releases the scales that the other lanes stored
          if (lane == 0) {
            fence_after();
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              product(tmem + (n & 1) * TK, base + T::OFF_Q + (kk >> 2) * (TM * 128) + (kk & 3) * 32,
                      base + T::OFF_K + (kk >> 2) * (TK * 128) + (kk & 3) * 32, kIdescS, kk > 0);
            commit(&sh.sfull[n & 1]);
            mbar_arrive(&sh.sfull[n & 1]);  // releases the scales to whoever waits for S
          }
          __syncwarp();
        }
      } else if (lane == 0) {
        for (int j = 0; j < steps; ++j) {
          if (!wait_for(&sh.vready[j & 1], (j >> 1) & 1, p.status, abort) ||
              !wait_for(&sh.pfull[j & 1], (j >> 1) & 1, p.status, abort))
            break;
          fence_after();
#pragma unroll
          for (int kk = 0; kk < TK / 16; ++kk)
            product_tmem(tmem_o, tmem + (j & 1) * TK + kk * 8, base + T::OFF_V + (j & 1) * (D * 128) + kk * 32, kIdescO,
                         j > 0 || kk > 0);
          commit(&sh.odone[j & 1]);
        }
      }
      if (lane == 0) {  // on every path: no product may run when the tensor memory is freed
        commit(&sh.drain[warp - 8]);
        mbar_wait(&sh.drain[warp - 8], 0, p.status);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ codes to f16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int ct = tid - kSoftmax, cw = warp - 4;
    // K of step j into place: 16 codes of a key at a time; a quarter warp covers four chunks of two keys, of 128
    // bytes the lower half of one and the upper half of the other, so that it reads and writes every bank once.
    auto convert_k = [&](int j) {
      constexpr int C = D / 16;  // chunks of a key
      const uint8_t* src = smem + T::OFF_SK + (j & 1) * 4 * T::BLK;
#pragma unroll
      for (int i0 = 0; i0 < TK * C; i0 += kConvert) {
        const int i = i0 + ct;
        int key, c;
        if (C == 6) {
          key = i / 6;
          c = i - key * 6;
        } else {
          const int rest = i >> 2;
          key = C == 8 ? (rest & 7) + ((rest >> 4) << 3) : rest;
          c = (i & 3) + (C == 8 ? ((rest ^ (rest >> 3)) & 1) * 4 : 0);
        }
        const uint4 w = *reinterpret_cast<const uint4*>(src + key * D + c * 16);
        uint8_t* dst = smem + T::OFF_K + (c >> 2) * (TK * 128) + key * 128;
        const int ch = (c & 3) * 2;
        *reinterpret_cast<uint4*>(dst + ((ch ^ (key & 7)) << 4)) =
            make_uint4(cvt_e4m3x2_f16x2(w.x & 0xffffu), cvt_e4m3x2_f16x2(w.x >> 16), cvt_e4m3x2_f16x2(w.y & 0xffffu),
                       cvt_e4m3x2_f16x2(w.y >> 16));
        *reinterpret_cast<uint4*>(dst + (((ch + 1) ^ (key & 7)) << 4)) =
            make_uint4(cvt_e4m3x2_f16x2(w.z & 0xffffu), cvt_e4m3x2_f16x2(w.z >> 16), cvt_e4m3x2_f16x2(w.w & 0xffffu),
                       cvt_e4m3x2_f16x2(w.w >> 16));
      }
    };
    // V of step j into place, transposed: 8 tokens of 4 dims at a time; lanes over the 4 blocks and 8 groups
    // of dims. Of two dims, every other group of lanes writes the second first: a quarter warp's rows then differ
    // by an odd number, and its chunks lie in different banks.
    auto convert_v = [&](int j) {
      const int b = lane & 3, turn = (lane >> 2) & 1;
      const bool have = sh.scale[j & (kMeta - 1)][0][b] >= 0.f;
      const bool full = kv_len - j * TK >= TK && __all_sync(kAll, have);
#pragma unroll
      for (int u0 = 0; u0 < 2 * (D / 32); u0 += 4) {
        const int u = u0 + cw;
        if (2 * (D / 32) % 4 != 0 && u >= 2 * (D / 32)) break;
        const int half = u & 1, d0 = (u >> 1) * 32 + (lane >> 2) * 4;
        const uint8_t* src = smem + T::OFF_SV + ((j & 1) * 4 + b) * T::VBLK + half * 8 * D + d0;
        const int key0 = b * kBlock + half * 8;
        const int live = have ? kv_len - j * TK - key0 : 0;  // of these 8 tokens
        uint32_t w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          w[r] = *reinterpret_cast<const uint32_t*>(src + r * D);
        }
        if (!full) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r >= live) w[r] = 0u;
        }
        if (j >= diagonal) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const uint32_t nan = ((w[r] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // the bytes 0x7f and 0xff
            if (nan) {
              w[r] &= ~(nan | (nan - (nan >> 7)));
              atomicOr(&sh.nan[j - diagonal], 1ull << (key0 + r));
            }
          }
        }
        const int ch = key0 >> 3;
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t sel = e == 0 ? (turn ? 0x4051u : 0x5140u) : (turn ? 0x6273u : 0x7362u);
          uint32_t lo[4], hi[4];  // of dims first and second
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t pair = __byte_perm(w[2 * r], w[2 * r + 1], sel);
            lo[r] = cvt_e4m3x2_f16x2(pair & 0xffffu);
            hi[r] = cvt_e4m3x2_f16x2(pair >> 16);
          }
          const int first = d0 + e + turn, second = d0 + e + 1 - turn;
          uint8_t* to = smem + T::OFF_V + (j & 1) * (D * 128);
          *reinterpret_cast<uint4*>(to + first * 128 + ((ch ^ (first & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<uint4*>(to + second * 128 + ((ch ^ (second & 7)) << 4)) =
              make_uint4(hi[0], hi[1], hi[2], hi[3]);
        }
      }
    };
    for (int n = 0; n < steps; ++n) {
      bool ok = wait_for(&sh.staged_k[n & 1], (n >> 1) & 1, p.status, abort);
      if (n > 0) ok = ok && wait_for(&sh.sfull[(n - 1) & 1], ((n - 1) >> 1) & 1, p.status, abort);  // K's place is free
      if (!__all_sync(kAll, ok)) break;
      convert_k(n);
      fence_proxy_async_shared();
      mbar_arrive(&sh.kready[n & 1]);
      ok = wait_for(&sh.staged_v[n & 1], (n >> 1) & 1, p.status, abort) &&
           wait_for(&sh.meta[n & (kMeta - 1)], (n / kMeta) & 1, p.status, abort);
      if (n > 1) ok = ok && wait_for(&sh.odone[n & 1], ((n - 2) >> 1) & 1, p.status, abort);  // V's place is free
      if (!__all_sync(kAll, ok)) break;
      convert_v(n);
      fence_proxy_async_shared();
      mbar_arrive(&sh.vready[n & 1]);
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    const int r = tid;  // query row, and tensor-memory lane
    const bool mine = r < me.n;
    const bool rows_here = warp * 32 < me.n;  // a warp without rows only keeps the barriers going
    const int qpos = me.pos + r;
    float factor = 0.f;
    {
      const __nv_bfloat16* src = p.q + (int64_t)(me.row0 + (mine ? r : 0)) * p.q_stride + (int64_t)head * D;
      uint4 w[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        w[c] = mine ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        amax = fmaxf(fmaxf(amax, fabsf(bf16lo(w[c].x))), fabsf(bf16hi(w[c].x)));
        amax = fmaxf(fmaxf(amax, fabsf(bf16lo(w[c].y))), fabsf(bf16hi(w[c].y)));
        amax = fmaxf(fmaxf(amax, fabsf(bf16lo(w[c].z))), fabsf(bf16hi(w[c].z)));
        amax = fmaxf(fmaxf(amax, fabsf(bf16lo(w[c].w))), fabsf(bf16hi(w[c].w)));
      }
      int e = (int)(__float_as_uint(amax) >> 23) - 127;
      e = amax == 0.f ? 0 : max(-126, min(126, e));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      factor = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint8_t* dst = smem + T::OFF_Q + (c >> 3) * (TM * 128) + r * 128;
        *reinterpret_cast<uint4*>(dst + (((c & 7) ^ (r & 7)) << 4)) =
            make_uint4(pack_f16x2(bf16lo(w[c].x) * down, bf16hi(w[c].x) * down),
                       pack_f16x2(bf16lo(w[c].y) * down, bf16hi(w[c].y) * down),
                       pack_f16x2(bf16lo(w[c].z) * down, bf16hi(w[c].z) * down),
                       pack_f16x2(bf16lo(w[c].w) * down, bf16hi(w[c].w) * down));
      }
    }
    fence_proxy_async_shared();
    mbar_arrive(&sh.qfull);

    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    float m = -INFINITY, mw = -INFINITY, l = 0.f;  // mw: M - kLift
    for (int j = 0; j < steps; ++j) {
      if (!__all_sync(kAll, wait_for(&sh.sfull[j & 1], (j >> 1) & 1, p.status, abort))) break;
      bool stop = false;
      if (rows_here) {
        fence_after();
        uint32_t s[TK];
        tmem_load(tmem + lanes + (j & 1) * TK, s);
        tmem_load(tmem + lanes + (j & 1) * TK + 32, s + 32);
        wait_loads(s);
        wait_loads(s + 32);
        const float4 ks = *reinterpret_cast<const float4*>(sh.scale[j & (kMeta - 1)][0]);
        const float4 vs = *reinterpret_cast<const float4*>(sh.scale[j & (kMeta - 1)][1]);
        // logits are S * f; f stays above 0 (an all-zero block under a tiny q), below it no such block
        auto logit_factor = [&](float k) { return k < 0.f ? -1.f : fmaxf(factor * k, 1.2e-38f); };
        const float f[4] = {logit_factor(ks.x), logit_factor(ks.y), logit_factor(ks.z), logit_factor(ks.w)};
        const float ev[4] = {vs.x, vs.y, vs.z, vs.w};
        if (j >= diagonal || f[0] < 0.f || f[1] < 0.f || f[2] < 0.f || f[3] < 0.f) {
          const int seen = qpos - j * TK;  // the last key of the step that the row sees
#pragma unroll
          for (int k = 0; k < TK; ++k)
            if (k > seen || f[k >> 4] < 0.f) s[k] = f[k >> 4] < 0.f ? 0x7f800000u : 0xff800000u;
        }
        float mx = -INFINITY, mz = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          // (a missing block's f is negative and its entries +inf: the largest product is -inf too)
          float t0 = fmaxf(__uint_as_float(s[b * 16]), __uint_as_float(s[b * 16 + 1]));
          float t1 = fmaxf(__uint_as_float(s[b * 16 + 2]), __uint_as_float(s[b * 16 + 3]));
#pragma unroll
          for (int k = 4; k < kBlock; k += 4) {  // (three operands to a maximum)
            t0 = fmaxf(fmaxf(t0, __uint_as_float(s[b * 16 + k])), __uint_as_float(s[b * 16 + k + 1]));
            t1 = fmaxf(fmaxf(t1, __uint_as_float(s[b * 16 + k + 2])), __uint_as_float(s[b * 16 + k + 3]));
          }
          const float x = fmaxf(t0, t1) * f[b];
          mx = fmaxf(mx, x);
          mz = fmaxf(mz, x + ev[b]);
        }
        if (mx > m + 8.f) {
          l *= ex2(m - mx);
          m = mx;
        }
        const bool up = mz > mw + (8.f + kLift);
        if (__any_sync(kAll, up)) {
          const float to = up ? mz - kLift : mw;
          if (j > 0)  // the products so far have to be in O
            stop = !__all_sync(kAll, wait_for(&sh.odone[(j - 1) & 1], ((j - 1) >> 1) & 1, p.status, abort));
          if (j > 0 && !stop) {
            const float down = mw == -INFINITY ? (up ? 0.f : 1.f) : ex2(mw - to);
            fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_load16(tmem_o + lanes + c, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
              tmem_store16(tmem_o + lanes + c, o);
            }
            wait_stores();
          }
          mw = to;
        }
        if (!stop) {
          const float off = m - mw;  // log2 of weight over probability, but for the block's log2 s_v
          const bool far = __any_sync(kAll, off + fminf(fminf(ev[0], ev[1]), fminf(ev[2], ev[3])) < -90.f);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float add = mw == -INFINITY ? 0.f : ev[b] - mw;  // (nothing seen yet: every entry is -inf)
            float sum = 0.f, more = 0.f;
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float w0 = ex2(fmaf(__uint_as_float(s[b * 16 + 2 * k]), f[b], add));
              const float w1 = ex2(fmaf(__uint_as_float(s[b * 16 + 2 * k + 1]), f[b], add));
              sum += w0;
              more += w1;
              w[k] = pack_f16x2(w0, w1);
            }
            tmem_store8(tmem + lanes + (j & 1) * TK + b * 8, w);
            if (!far) l += mw == -INFINITY ? 0.f : (sum + more) * ex2(-off - ev[b]);
          }
          // The weights may have underflowed, so the probabilities are summed themselves. Also taken in the last step
          // of a row whose end leaves a whole block of it unused, which counts as log2 s_v = -126.
          if (far) {
#pragma unroll
            for (int k = 0; k < TK; ++k) {
              const float x = __uint_as_float(s[k]) * f[k >> 4];
              l += x == -INFINITY ? 0.f : ex2(x - m);
            }
          }
          wait_stores();
        }
      }
      if (stop) break;
      fence_before();
      mbar_arrive(&sh.pfull[j & 1]);
    }
    if (rows_here && __all_sync(kAll, wait_for(&sh.odone[(steps - 1) & 1], ((steps - 1) >> 1) & 1, p.status, abort))) {
      fence_after();
      const float g = l > 0.f ? ex2(mw + kLift - m) * kUnlift / l : (l == 0.f ? 0.f : l);
      __nv_bfloat16* dst = p.out + (int64_t)(me.row0 + (mine ? r : 0)) * p.out_stride + (int64_t)head * D;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_load(tmem_o + lanes + c, o);
        wait_loads(o);
        if (mine) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_bf16x2(__uint_as_float(o[k + 2 * e]) * g, __uint_as_float(o[k + 2 * e + 1]) * g);
            *reinterpret_cast<uint4*>(dst + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      // NaN that were taken out of V: back into the rows that see them, dim by dim (rare, so from global memory)
      const int32_t* bt = p.block_table + (int64_t)me.slot * p.bt_stride;
      for (int i = 0; i < kDiagonal; ++i) {
        for (unsigned long long bits = sh.nan[i]; bits; bits &= bits - 1) {
          const int key = (diagonal + i) * TK + __ffsll((long long)bits) - 1;
          if (!mine || key > qpos) continue;
          const int64_t at = (int64_t)p.num_blocks * p.kv_heads + (int64_t)bt[key / kBlock] * p.kv_heads + kvh;
          const uint8_t* v = p.codes + at * T::BLK + (key % kBlock) * D;
          for (int d = 0; d < D; ++d)
            if ((v[d] & 0x7fu) == 0x7fu) dst[d] = f_to_bf16(NAN);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <int D>
static int launch_prefill(const PrefillParams& p, int num_heads, cudaStream_t st) {
  if (cudaFuncSetAttribute(prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<D>::SMEM) != cudaSuccess)
    return CDB_ERR_CUDA;
  return launch_pdl(prefill_kernel<D>, dim3(num_heads, p.num_tiles), dim3(kPrefillThreads), Tile<D>::SMEM, st, p) ==
                 cudaSuccess
             ? CDB_OK
             : CDB_ERR_CUDA;
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
      num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0 ||
      !(scale > 0.f) || scale > 1e30f)
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_stride & 7) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (out_stride & 7) || (reinterpret_cast<uintptr_t>(tiles) & 15))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_tiles == 0) return CDB_OK;
  if ((num_rows > 0 && (q == nullptr || out == nullptr)) || block_table == nullptr || tiles == nullptr)
    return CDB_ERR_INVALID_ARGUMENT;  // (with no rows no tile fits, and q and out are not touched)
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
  p.num_tiles = num_tiles;
  p.num_rows = num_rows;
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_prefill<128>(p, num_heads, st);
  if (head_dim == 96) return launch_prefill<96>(p, num_heads, st);
  return launch_prefill<64>(p, num_heads, st);
}
