// Decode attention over the bf16 paged cache for requests that share a prompt.
//
// Rows of a group see the same blocks first. For those, Q K^T and P V are matrix products of all the group's
// rows, so a block is read once for up to 128 of them; behind them every row has pages of its own. Softmax parts (m a
// maximum of the logits, l the sum of 2^(x - m), o that of 2^(x - m) v) of any set of keys join by rescaling to
// one m, so the two kinds of work need not wait for each other: one launch does both side by side, and a
// last one joins. Three launches in all:
//   plan    one CTA: how many blocks each group shares, how the work is cut into equal shares;
//   attend  two CTAs an SM, each of one kind: `Shared` steps (below) or pages of single rows;
//   join    a warp (or a CTA) per row and head adds up its parts. Rows with one part are written by attend.
// No counters and no atomics between CTAs: parts lie where the plan says, and are added in that order.
//
// Shared steps. A CTA takes 128 rows (request x query head of one kv head) over a share of the group's 64-key
// steps. Warps 0..3 are the softmax, thread r owns row r; warp 4 brings pages (TMA, 128-byte swizzle, two steps
// ahead); warp 5 issues the products: S = Q K^T (tcgen05, 128 x 64 x D) and O += P V (128 x D x 64), P written over
// the S that it comes from in tensor memory, V as it lies in the cache (the product's inner index across
// its rows). Two CTAs an SM, so that one's exponentials run beside the other's products.
//
// Pages of single rows. The pages of all (row, kv head, up to 8 query heads) form one stream that is cut into equal
// shares for the warps of the other CTAs. A page's K and V go straight from memory into the registers
// of m16n8k16 products: the inner index may be permuted at will, so lanes load 16 bytes side by side and q is
// loaded by the same permutation. K of the next page is requested before this one's softmax, V after its product.
//
// The weights P are rounded to bf16 for their product with V (2^-8 of each), V's type; l is the sum of the
// rounded weights, so what is common to them cancels. m only moves when passed by 8, which bf16's range allows.
#include <cuda.h>

#include "tcgen05.cuh"

namespace cdb {
namespace prefix {

constexpr int kBlock = 16;  // tokens of a page
constexpr int TM = 128;     // rows of a shared step
constexpr int TK = 64;      // keys of a shared step
constexpr int kStepPages = TK / kBlock;
constexpr int kStages = 2;
constexpr int kThreads = 192;
constexpr int kWarps = kThreads / 32;
constexpr int kPlanThreads = 1024;
constexpr int kPlanGroups = 2048;  // groups whose state fits the plan's shared memory
constexpr int kHeads = 8;          // query heads of one single-row segment (n of an m16n8k16 product)
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kAll = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

// What the plan leaves for the others.
struct Header {
  int shared_ctas;   // CTAs of attend that take shared steps
  int pieces;        // of shared steps
  int64_t pages;     // (row, kv head, head group) pages of single rows
  int64_t share;     // of them a warp takes
};
struct Item {
  int pos, slot;  // pos -1: skipped
  int group;      // -1: alone
  int shared;     // its first pages, which the group's steps cover
};
struct Group {
  int splits;  // pieces of one (tile, kv head)
  int pages;   // shared
  int rows;    // requests x query heads of a kv head
  int leader;  // the request whose block table is read
  int base;    // row (of the parts) of its first part
  int piece;   // its first piece
};

struct Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const __nv_bfloat16* keys;  // this cache layer's; values follow kv_rows rows later
  int64_t kv_rows;
  int blocks;
  const int32_t* block_table;
  int64_t bt_stride;
  int bt_rows, bt_width;
  const int32_t* item_slot;
  const int32_t* item_pos;
  int num_items, kv_heads, heads_per_kv;
  int head_groups;   // of up to kHeads query heads, per kv head
  int stored_heads;  // min(heads_per_kv, kHeads)
  int tile_items;    // requests of a tile (0: heads do not fit one, nothing is shared)
  const int32_t* group_start;
  const int32_t* prefix_len;
  int num_groups;
  int num_ctas;  // of attend
  float scale_log2;
  // the workspace
  Header* header;
  Item* items;
  int64_t* before;   // [num_items + 1]: pages of the rows before each
  Group* groups;     // [num_groups + 1]
  int2* state;       // [num_groups]: the plan's, where it does not fit shared memory
  float* shared_o;   // parts of shared steps: per (group, kv head, split) [D / 8][rows][8]
  float2* shared_ml;  // [rows of parts] {m, l}
  float* single;     // parts of single rows: [segment + warp][stored_heads][D + 4], m and l behind o
  int32_t* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a / b for a, b >= 0: a 64-bit division takes some 400 cycles, and the numbers nearly always fit 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// ---------------------------------------------------------------------------------------------- plan

// Sums of the threads' values before this thread's, and of all.
template <typename T>
__device__ __forceinline__ T scan(T mine, T& all, T* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(kAll, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  T w = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(kAll, w, o);
    if (lane >= o) w += y;
  }
  all = __shfl_sync(kAll, w, 31);
  const T base = __shfl_sync(kAll, w, (warp + 31) & 31);
  return (warp ? base : T(0)) + x - mine;
}

__global__ void __launch_bounds__(kPlanThreads, 1) plan_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int64_t red[32];
  __shared__ int s_start[kPlanGroups + 1];
  __shared__ int2 s_state[kPlanGroups];  // {least whole pages that a row sees, live rows}
  __shared__ int s_leader[kPlanGroups];
  __shared__ int64_t s_share[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int ng = p.tile_items > 0 ? p.num_groups : 0;
  const bool fits = ng <= kPlanGroups;
  int2* state = fits ? s_state : p.state;
  // (a group's leader is kept in the group's own place where shared memory does not hold it)
  bool bad = false;
  for (int g = tid; g < p.num_groups; g += kPlanThreads) {
    const int a = p.group_start[g], b = p.group_start[g + 1];
    bad |= a < 0 || b < a || b > p.num_items;
    if (g < ng) {
      if (fits) s_start[g] = a, s_leader[g] = INT32_MAX;
      else p.groups[g].leader = INT32_MAX;
      if (fits && g + 1 == ng) s_start[ng] = b;
      state[g] = make_int2(INT32_MAX, 0);
    }
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) set_error(p.status, CDB_ERR_INDEX);
    ng = 0;
  }
  // rows: their groups, and what those have in common
  for (int i = tid; i < p.num_items; i += kPlanThreads) {
    Item it;
    it.pos = p.item_pos[i];
    it.slot = p.item_slot[i];
    it.group = -1;
    it.shared = 0;
    if (it.pos >= 0 && (it.slot < 0 || it.slot >= p.bt_rows || it.pos / kBlock >= p.bt_width)) {
      set_error(p.status, CDB_ERR_INDEX);
      it.pos = -1;
    }
    if (it.pos < 0) it.pos = -1;
    if (ng > 0) {
      const int* start = fits ? s_start : p.group_start;
      int lo = -1, hi = ng + 1;  // the last bound at or before i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid;
        else hi = mid;
      }
      if (lo >= 0 && lo < ng && it.pos >= 0) {
        it.group = lo;
        atomicMin(&state[lo].x, (it.pos + 1) / kBlock);
        atomicAdd(&state[lo].y, 1);
        atomicMin(fits ? &s_leader[lo] : &p.groups[lo].leader, i);
      }
    }
    p.items[i] = it;
  }
  __syncthreads();
  // groups: a stretch of them to a thread
  auto pages_of = [&](int g) {
    const int2 st = fits ? s_state[g] : __ldcg(p.state + g);  // (atomics pass the first cache by)
    return st.y >= 2 ? min(max(p.prefix_len[g], 0) / kBlock, st.x) : 0;  // one row alone has nothing to share
  };
  auto bound = [&](int g) { return fits ? s_start[g] : p.group_start[g]; };
  auto tiles_of = [&](int g) { return (bound(g + 1) - bound(g) + p.tile_items - 1) / p.tile_items; };
  const int per_g = (ng + kPlanThreads - 1) / kPlanThreads;
  const int g0 = min(ng, tid * per_g), g1 = min(ng, g0 + per_g);
  int64_t steps = 0, all_steps;
  for (int g = g0; g < g1; ++g)
    steps += (int64_t)tiles_of(g) * p.kv_heads * ((pages_of(g) + kStepPages - 1) / kStepPages);
  scan(steps, all_steps, red);
  // rows: their own pages
  const int per_i = (p.num_items + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(p.num_items, tid * per_i), i1 = min(p.num_items, i0 + per_i);
  int64_t own = 0, all_own;
  auto own_of = [&](int i) {
    const Item it = p.items[i];
    return it.pos < 0 ? 0 : it.pos / kBlock + 1 - (it.group >= 0 ? pages_of(it.group) : 0);
  };
  for (int i = i0; i < i1; ++i) own += own_of(i);
  int64_t run = scan(own, all_own, red);
  for (int i = i0; i < i1; ++i) {
    p.before[i] = run;
    run += own_of(i);
    if (p.items[i].group >= 0) p.items[i].shared = pages_of(p.items[i].group);
  }
  if (tid == 0) p.before[p.num_items] = all_own;
  // CTAs by the bytes of either kind of work, and shares of them
  const int64_t pages = all_own * p.kv_heads * p.head_groups;
  const int64_t shared_pages = all_steps * kStepPages;
  int ctas = 0;
  if (all_steps > 0)
    ctas = pages == 0 ? p.num_ctas
                      : (int)min((int64_t)p.num_ctas - 1, max((int64_t)1, quotient((int64_t)p.num_ctas * shared_pages, shared_pages + pages)));
  // Pieces end with their (tile, kv head). The shortest of 32 shares, from an even one to 2.9 of it, whose pieces
  // do not outnumber the CTAs; where none is, an even one, and CTAs take several.
  const int64_t even = ctas ? quotient(all_steps + ctas - 1, ctas) : 1;
  const int64_t mine = max((int64_t)1, even + even * warp * 2 / 33);
  int64_t pieces = 0;
  for (int g = lane; g < ng; g += 32) {
    const int n = (pages_of(g) + kStepPages - 1) / kStepPages;
    if (n) pieces += (int64_t)tiles_of(g) * p.kv_heads * quotient(n + mine - 1, mine);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) pieces += __shfl_xor_sync(kAll, pieces, o);
  if (lane == 0) s_share[warp] = pieces <= ctas ? mine : INT64_MAX;
  __syncthreads();
  int64_t share = s_share[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) share = min(share, __shfl_xor_sync(kAll, share, o));
  if (share == INT64_MAX) share = max((int64_t)1, even);
  int64_t np = 0, rows = 0, all_np, all_rows;
  for (int g = g0; g < g1; ++g) {
    const int n = (pages_of(g) + kStepPages - 1) / kStepPages;
    const int64_t splits = quotient(n + share - 1, share);
    np += (int64_t)tiles_of(g) * p.kv_heads * splits;
    rows += (int64_t)(bound(g + 1) - bound(g)) * p.heads_per_kv * p.kv_heads * splits;
  }
  np = scan(np, all_np, red);
  rows = scan(rows, all_rows, red);
  for (int g = g0; g < g1; ++g) {
    Group gr;
    gr.pages = pages_of(g);
    const int n = (gr.pages + kStepPages - 1) / kStepPages;
    gr.splits = (int)quotient(n + share - 1, share);
    gr.rows = (bound(g + 1) - bound(g)) * p.heads_per_kv;
    gr.leader = fits ? s_leader[g] : __ldcg(&p.groups[g].leader);
    gr.base = (int)rows;
    gr.piece = (int)np;
    np += (int64_t)tiles_of(g) * p.kv_heads * gr.splits;
    rows += (int64_t)gr.rows * p.kv_heads * gr.splits;
    p.groups[g] = gr;
  }
  if (tid == 0) {
    Header h;
    h.shared_ctas = ctas;
    h.pieces = (int)all_np;
    h.pages = pages;
    const int64_t warps = (int64_t)(p.num_ctas - ctas) * kWarps;
    h.share = max((int64_t)1, warps ? quotient(pages + warps - 1, warps) : 1);
    *p.header = h;
  }
}

// ---------------------------------------------------------------------------------------------- attend

template <int D>
struct Tile {
  static constexpr int ATOMS = (D + 63) / 64;  // 128-byte swizzle atoms of a row of D (96: the second one's end is zero)
  static constexpr int OFF_K = ATOMS * TM * 128;                       // behind q [ATOMS][128][64]
  static constexpr int STAGE = ATOMS * TK * 128;                       // K or V of a step, [ATOMS][64][64]
  static constexpr int OFF_V = OFF_K + kStages * STAGE;
  static constexpr int OFF_BAR = OFF_V + kStages * STAGE;
  static constexpr int SMEM = OFF_BAR + 256;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

struct Shared {
  uint64_t kfull[kStages], vfull[kStages];  // a step's K, V have landed
  uint64_t qfull;                           // q of a piece written
  uint64_t sfull[2];                        // S done (and K's place free), and the step's pages known
  uint64_t pfull[2];                        // weights written
  uint64_t odone[2];                        // O product done (V's and S's places free)
  uint64_t drain;
  int missing[4];                           // a step's pages that do not exist
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Shared) <= 256, "room behind the tiles");

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

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int col, int head, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(head), "r"(row), "r"(bar)
      : "memory");
}

// A piece of shared steps.
struct Piece {
  int group, tile, kvh, split;
  int first, steps;  // its steps of the group's
  int rows;          // of the tile
  int pages;         // of the group
  int leader;
  int64_t part;  // row of the parts where its (group, kv head, split) begins
};

__device__ __forceinline__ Piece find_piece(const Params& p, int index) {
  // the last group that begins at or before it (those without pieces begin where their successor does)
  const int lane = threadIdx.x & 31;
  int lo = 0, n = p.num_groups;
  while (n > 1) {
    const int stride = (n + 31) / 32, at = lo + lane * stride;
    const unsigned hit = __ballot_sync(kAll, at < lo + n && p.groups[at].piece <= index);
    const int k = 31 - __clz(hit);
    n = min(stride, n - k * stride);
    lo += k * stride;
  }
  const Group g = p.groups[lo];
  Piece me;
  const int local = index - g.piece, per_head = g.splits;
  const int unit = local / per_head;
  me.split = local - unit * per_head;
  me.tile = unit / p.kv_heads;
  me.kvh = unit - me.tile * p.kv_heads;
  me.group = lo;
  const int n_steps = (g.pages + kStepPages - 1) / kStepPages;
  me.first = (int)((int64_t)n_steps * me.split / per_head);
  me.steps = (int)((int64_t)n_steps * (me.split + 1) / per_head) - me.first;
  me.rows = min(p.tile_items * p.heads_per_kv, g.rows - me.tile * p.tile_items * p.heads_per_kv);
  me.pages = g.pages;
  me.leader = g.leader;
  me.part = g.base + ((int64_t)me.kvh * per_head + me.split) * g.rows;
  return me;
}

template <int D>
__device__ __forceinline__ void shared_steps(const CUtensorMap& map, const Params& p, const Header& h, uint8_t* smem) {
  using T = Tile<D>;
  constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10);  // fp32 accumulators, bf16 operands
  constexpr uint32_t kIdescS = kBf16 | ((uint32_t)(TK >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  constexpr uint32_t kIdescO = kBf16 | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  Shared& sh = *reinterpret_cast<Shared*>(smem + T::OFF_BAR);
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.kfull[i], 1);
      mbar_init(&sh.vfull[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.sfull[i], 2);
      mbar_init(&sh.pfull[i], TM);
      mbar_init(&sh.odone[i], 1);
    }
    mbar_init(&sh.qfull, TM);
    mbar_init(&sh.drain, 1);
    sh.abort = (base & 1023u) != 0u;  // the swizzle counts on it
    if (sh.abort) set_error(p.status, CDB_ERR_INVALID_ARGUMENT);
    fence_barrier_init();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // Only now may the next kernel's CTAs come: one that holds tensor memory and waits for this kernel could otherwise
  // be what the allocation above waits for.
  pdl_trigger();
  const uint32_t tmem = sh.tmem;  // S: two buffers of 64 columns; O: 128 columns on
  const uint32_t tmem_o = tmem + 2 * TK;
  volatile int* abort = &sh.abort;

  // `t` counts the steps of all of the CTA's pieces, `c` the pieces: every barrier's phases follow from them.
  if (warp == 4) {
    // ------------------------------------------------------------ pages
    int t = 0;
    bool ok = true;
    for (int index = blockIdx.x; index < h.pieces && ok; index += h.shared_ctas) {
      const Piece me = find_piece(p, index);
      const int32_t* bt = p.block_table + (int64_t)p.items[me.leader].slot * p.bt_stride;
      // lane: page (lane & 3) of the step, columns 64 * ((lane >> 2) & 1); lanes 0..7 of K, 16..23 of V
      const int page_of = lane & 3, atom = (lane >> 2) & 1;
      const bool loads = (lane & 8) == 0 && atom < T::ATOMS;
      auto fetch = [&](int n) {
        const int page = (me.first + n) * kStepPages + page_of;
        return n < me.steps && page < me.pages ? bt[page] : INT32_MIN;
      };
      int id = fetch(0);
      for (int n = 0; n < me.steps; ++n, ++t) {
        const int next = fetch(n + 1);
        const int stage = t % kStages;
        const bool have = id >= 0 && id < p.blocks;
        const unsigned gone = __ballot_sync(kAll, !have) & 15u;
        if (lane < kStepPages && !have && id != INT32_MIN) set_error(p.status, CDB_ERR_INDEX);
        // behind the cache's rows a box comes as zeros
        const int row = have ? id * kBlock : 2 * (int)p.kv_rows;
        if (t >= kStages) ok = __all_sync(kAll, wait_for(&sh.sfull[t & 1], ((t - 2) >> 1) & 1, p.status, abort));
        if (!ok) break;
        const uint32_t at = base + (lane < 16 ? T::OFF_K : T::OFF_V) + stage * T::STAGE + atom * (TK * 128) + page_of * (kBlock * 128);
        if (lane == 0) {
          sh.missing[t & 3] = (int)gone;
          mbar_arrive_expect_tx(&sh.kfull[stage], T::STAGE);
        }
        __syncwarp();
        if (loads && lane < 16) load_box(at, &map, atom * 64, me.kvh, row, smem_u32(&sh.kfull[stage]));
        if (t >= kStages) ok = __all_sync(kAll, wait_for(&sh.odone[t & 1], ((t - 2) >> 1) & 1, p.status, abort));
        if (!ok) {
          if (lane == 0) mbar_wait(&sh.kfull[stage], (t / kStages) & 1, p.status);
          __syncwarp();
          break;
        }
        if (lane == 16) mbar_arrive_expect_tx(&sh.vfull[stage], T::STAGE);
        __syncwarp();
        if (loads && lane >= 16)
          load_box(at, &map, atom * 64, me.kvh, have ? row + (int)p.kv_rows : row, smem_u32(&sh.vfull[stage]));
        id = next;
      }
    }
    // nothing may be on its way when the CTA ends
    for (int j = max(0, t - kStages); j < t; ++j) {
      mbar_wait(&sh.kfull[j % kStages], (j / kStages) & 1, p.status);
      mbar_wait(&sh.vfull[j % kStages], (j / kStages) & 1, p.status);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ products
    int t = 0, c = 0;
    bool ok = true;
    auto weigh = [&](int j, bool add) {  // O (+)= P V of step j
      ok = ok && wait_for(&sh.vfull[j % kStages], (j / kStages) & 1, p.status, abort) &&
           wait_for(&sh.pfull[j & 1], (j >> 1) & 1, p.status, abort);
      if (!ok) return;
      fence_after();
#pragma unroll
      for (int kk = 0; kk < TK / 16; ++kk)
        product_tmem(tmem_o, tmem + (j & 1) * TK + kk * 8,
                     operand(base + T::OFF_V + (j % kStages) * T::STAGE + kk * 2048, TK * 128), kIdescO, add || kk > 0);
      commit(&sh.odone[j & 1]);
    };
    for (int index = blockIdx.x; index < h.pieces; index += h.shared_ctas, ++c) {
      const Piece me = find_piece(p, index);
      if (lane == 0) {
        for (int n = 0; n < me.steps && ok; ++n, ++t) {
          ok = wait_for(&sh.kfull[t % kStages], (t / kStages) & 1, p.status, abort);
          if (n == 0) ok = ok && wait_for(&sh.qfull, c & 1, p.status, abort);
          if (t >= 2) ok = ok && wait_for(&sh.odone[t & 1], ((t - 2) >> 1) & 1, p.status, abort);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            product(tmem + (t & 1) * TK, operand(base + (kk >> 2) * (TM * 128) + (kk & 3) * 32),
                    operand(base + T::OFF_K + (t % kStages) * T::STAGE + (kk >> 2) * (TK * 128) + (kk & 3) * 32), kIdescS,
                    kk > 0);
          commit(&sh.sfull[t & 1]);
          mbar_arrive(&sh.sfull[t & 1]);  // releases `missing` to whoever waits for S
          if (n > 0) weigh(t - 1, n > 1);
        }
        if (ok) weigh(t - 1, me.steps > 1);
      }
      __syncwarp();
    }
    if (lane == 0) {  // on every path: no product may run when the tensor memory is freed
      commit(&sh.drain);
      mbar_wait(&sh.drain, 0, p.status);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int r = tid;  // row of the tile, and tensor-memory lane
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    int t = 0;
    bool ok = true;
    for (int index = blockIdx.x; index < h.pieces && ok; index += h.shared_ctas) {
      const Piece me = find_piece(p, index);
      const bool mine = r < me.rows;
      const bool rows_here = warp * 32 < me.rows;  // a warp without rows only keeps the barriers going
      {
        const int local = r / p.heads_per_kv;
        const int first = p.group_start[me.group] + me.tile * p.tile_items;
        const __nv_bfloat16* src = p.q + (int64_t)(first + (mine ? local : 0)) * p.q_stride +
                                   (int64_t)(me.kvh * p.heads_per_kv + (mine ? r - local * p.heads_per_kv : 0)) * D;
        uint4 w[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          w[i] = mine ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<uint4*>(smem + (i >> 3) * (TM * 128) + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = w[i];
      }
      fence_proxy_async_shared();
      mbar_arrive(&sh.qfull);
      float m = -INFINITY, l = 0.f;
      for (int n = 0; n < me.steps; ++n, ++t) {
        ok = __all_sync(kAll, wait_for(&sh.sfull[t & 1], (t >> 1) & 1, p.status, abort));
        if (!ok) break;
        if (rows_here) {
          fence_after();
          uint32_t s[TK];
          tmem_load(tmem + lanes + (t & 1) * TK, s);
          tmem_load(tmem + lanes + (t & 1) * TK + 32, s + 32);
          wait_loads(s);
          wait_loads(s + 32);
          const int gone = sh.missing[t & 3];
          if (gone) {
#pragma unroll
            for (int k = 0; k < TK; ++k)
              if ((gone >> (k / kBlock)) & 1) s[k] = 0xff800000u;
          }
          float t0 = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
          float t1 = fmaxf(__uint_as_float(s[2]), __uint_as_float(s[3]));
#pragma unroll
          for (int k = 4; k < TK; k += 4) {  // (three operands to a maximum)
            t0 = fmaxf(fmaxf(t0, __uint_as_float(s[k])), __uint_as_float(s[k + 1]));
            t1 = fmaxf(fmaxf(t1, __uint_as_float(s[k + 2])), __uint_as_float(s[k + 3]));
          }
          const float mx = fmaxf(t0, t1) * p.scale_log2;
          const bool up = mx > m + 8.f;
          if (__any_sync(kAll, up)) {
            const float to = up ? mx : m;
            if (n > 0) {  // the products so far have to be in O
              ok = __all_sync(kAll, wait_for(&sh.odone[(t - 1) & 1], ((t - 1) >> 1) & 1, p.status, abort));
              if (!ok) break;
              const float down = m == -INFINITY ? (up ? 0.f : 1.f) : ex2(m - to);
              l *= down;
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
            m = to;
          }
          const float off = m == -INFINITY ? 0.f : -m;  // (nothing seen yet)
          float sum = 0.f, more = 0.f;
#pragma unroll
          for (int b = 0; b < TK / 16; ++b) {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              w[k] = pack_bf16x2(ex2(fmaf(__uint_as_float(s[b * 16 + 2 * k]), p.scale_log2, off)),
                                 ex2(fmaf(__uint_as_float(s[b * 16 + 2 * k + 1]), p.scale_log2, off)));
              sum += bf16lo(w[k]);
              more += bf16hi(w[k]);
            }
            tmem_store8(tmem + lanes + (t & 1) * TK + b * 8, w);
          }
          l += sum + more;
          wait_stores();
        }
        fence_before();
        mbar_arrive(&sh.pfull[t & 1]);
      }
      if (!ok) break;
      ok = __all_sync(kAll, wait_for(&sh.odone[(t - 1) & 1], ((t - 1) >> 1) & 1, p.status, abort));
      if (!ok) break;
      if (rows_here) {
        fence_after();
        const int64_t all = p.groups[me.group].rows;
        const int64_t at = (int64_t)me.tile * p.tile_items * p.heads_per_kv + r;
        float* dst = p.shared_o + me.part * D + at * 8;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_load(tmem_o + lanes + c, o);
          wait_loads(o);
          if (mine) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              __stcg(reinterpret_cast<float4*>(dst + ((c + k) / 8) * all * 8 + (k & 4)),
                     make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]),
                                 __uint_as_float(o[k + 3])));
          }
        }
        if (mine) __stcg(p.shared_ml + me.part + at, make_float2(m, l));
        fence_before();
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 5)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// ---------------------------------------------------------------- pages of single rows

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* a) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(a));
  return v;
}
__device__ __forceinline__ uint2 load8(const __nv_bfloat16* a) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(a));
  return v;
}
// D += A B on bf16 operands, fp32 accumulators (m16n8k16).
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// A place in the stream: page `page` of row `row`, head group `grp` of kv head `kvh`.
struct Cursor {
  int row, kvh, grp, page;
  Item it;
};
__device__ __forceinline__ int last_page(const Cursor& c) { return c.it.pos / kBlock; }
__device__ __forceinline__ int own_pages(const Item& it) { return it.pos < 0 ? 0 : it.pos / kBlock + 1 - it.shared; }

__device__ __forceinline__ void advance(const Params& p, Cursor& c) {
  if (++c.page <= last_page(c)) return;
  c.page = c.it.shared;
  if (++c.grp < p.head_groups) return;
  c.grp = 0;
  if (++c.kvh < p.kv_heads) return;
  c.kvh = 0;
  do {
    if (++c.row >= p.num_items) return;  // the stream's end
    c.it = p.items[c.row];
  } while (own_pages(c.it) == 0);
  c.page = c.it.shared;
}

template <int D>
struct Page {
  uint4 k[2][D / 32];  // tokens g, g + 8: dims i * 32 + t * 8
  uint4 v[4][D / 64];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9: dims i * 64 + g * 8
  uint2 w[4];          // of a head of 96: dims 64 + g * 4
};

template <int D>
__device__ __forceinline__ void load_k(const Params& p, int64_t row, int kvh, Page<D>& x) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      x.k[j][i] = load16(p.keys + ((row + g + 8 * j) * p.kv_heads + kvh) * D + i * 32 + t * 8);
}
template <int D>
__device__ __forceinline__ void load_v(const Params& p, int64_t row, int kvh, Page<D>& x) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat16* src = p.keys + ((p.kv_rows + row + 2 * t + (j & 1) + 8 * (j >> 1)) * p.kv_heads + kvh) * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) x.v[j][i] = load16(src + i * 64 + g * 8);
    if (D == 96) x.w[j] = load8(src + 64 + g * 4);
  }
}

template <int D>
__device__ __forceinline__ void single_rows(const Params& p, const Header& h) {
  pdl_trigger();
  constexpr int MT = D / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t warp = (int64_t)(blockIdx.x - h.shared_ctas) * kWarps + (threadIdx.x >> 5);
  const int64_t begin = warp * h.share, end = min(begin + h.share, h.pages);
  if (begin >= end) return;
  const int vheads = p.kv_heads * p.head_groups;
  // the last row that begins at or before `begin` and has pages
  Cursor c;
  {
    int lo = 0, n = p.num_items;
    while (n > 1) {
      const int stride = (n + 31) / 32, at = lo + lane * stride;
      const unsigned hit = __ballot_sync(kAll, at < lo + n && p.before[at] * vheads <= begin);
      const int k = 31 - __clz(hit);
      n = min(stride, n - k * stride);
      lo += k * stride;
    }
    c.row = lo;
    c.it = p.items[lo];
    const int own = own_pages(c.it);
    const int64_t at = begin - p.before[lo] * vheads;
    const int vh = (int)quotient(at, own);
    c.page = c.it.shared + (int)(at - (int64_t)vh * own);
    c.kvh = vh / p.head_groups;
    c.grp = vh - c.kvh * p.head_groups;
  }
  // lane i holds the block id of page i of a window of 32 pages of the row that is being loaded
  int win_row = -1, win_first = 0, win_id = -1;
  auto page_row = [&](const Cursor& a) -> int64_t {
    const int first = a.page & ~31;
    if (a.row != win_row || first != win_first) {
      win_row = a.row;
      win_first = first;
      win_id = first + lane <= last_page(a) ? p.block_table[(int64_t)a.it.slot * p.bt_stride + first + lane] : -1;
    }
    const int id = __shfl_sync(kAll, win_id, a.page & 31);
    if (id >= 0 && id < p.blocks) return (int64_t)id * kBlock;
    if (lane == 0) set_error(p.status, CDB_ERR_INDEX);
    return -1;
  };
  uint32_t qf[D / 16][2];
  auto load_q = [&]() {
    const int in_kv = c.grp * kHeads + g;
    const bool on = in_kv < p.heads_per_kv;
    const __nv_bfloat16* src =
        p.q + (int64_t)c.row * p.q_stride + (int64_t)(c.kvh * p.heads_per_kv + (on ? in_kv : 0)) * D + t * 8;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 w = on ? *reinterpret_cast<const uint4*>(src + i * 32) : make_uint4(0u, 0u, 0u, 0u);
      qf[2 * i][0] = w.x, qf[2 * i][1] = w.y, qf[2 * i + 1][0] = w.z, qf[2 * i + 1][1] = w.w;
    }
  };
  load_q();
  Page<D> x;
  int64_t row = page_row(c), next_row = -1;
  if (row >= 0) {
    load_k<D>(p, row, c.kvh, x);
    load_v<D>(p, row, c.kvh, x);
  }
  Cursor ahead = c;
  float acc[MT][4], m[2], l[2];
  bool fresh = true, whole = false;
  for (int64_t i = begin; i < end; ++i) {
    if (fresh) {
      if (i > begin) load_q();
      whole = c.page == c.it.shared;
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    const bool seg_end = c.page == last_page(c);
    const bool more = i + 1 < end;
    if (more) {
      advance(p, ahead);
      next_row = page_row(ahead);
    }
    if (row >= 0) {
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        mma_bf16(s[0], x.k[0][j].x, x.k[1][j].x, x.k[0][j].y, x.k[1][j].y, qf[2 * j][0], qf[2 * j][1]);
        mma_bf16(s[1], x.k[0][j].z, x.k[1][j].z, x.k[0][j].w, x.k[1][j].w, qf[2 * j + 1][0], qf[2 * j + 1][1]);
      }
      if (more && next_row >= 0) load_k<D>(p, next_row, ahead.kvh, x);
      // y[hd][j]: token g + 8 j, head 2t + hd
      float y[2][2];
#pragma unroll
      for (int hd = 0; hd < 2; ++hd)
#pragma unroll
        for (int j = 0; j < 2; ++j) y[hd][j] = (s[0][2 * j + hd] + s[1][2 * j + hd]) * p.scale_log2;
      if (seg_end) {
        const int live = c.it.pos % kBlock + 1;
#pragma unroll
        for (int hd = 0; hd < 2; ++hd)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (g + 8 * j >= live) y[hd][j] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j)  // what lies behind the row's end may be anything, NaN too
          if (2 * t + (j & 1) + 8 * (j >> 1) >= live) {
#pragma unroll
            for (int k = 0; k < D / 64; ++k) x.v[j][k] = make_uint4(0u, 0u, 0u, 0u);
            if (D == 96) x.w[j] = make_uint2(0u, 0u);
          }
      }
      const bool up = fmaxf(y[0][0], y[0][1]) > m[0] + 8.f || fmaxf(y[1][0], y[1][1]) > m[1] + 8.f;
      if (__any_sync(kAll, up)) {
#pragma unroll
        for (int hd = 0; hd < 2; ++hd) {
          float to = fmaxf(y[hd][0], y[hd][1]);
          to = fmaxf(to, __shfl_xor_sync(kAll, to, 4));
          to = fmaxf(to, __shfl_xor_sync(kAll, to, 8));
          to = fmaxf(to, __shfl_xor_sync(kAll, to, 16));
          to = fmaxf(m[hd], to);
          const float down = m[hd] == -INFINITY ? 1.f : ex2(m[hd] - to);
          m[hd] = to;
          l[hd] *= down;
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[j][hd] *= down, acc[j][2 + hd] *= down;
        }
      }
      uint32_t pw[2];
      const float off0 = m[0] == -INFINITY ? 0.f : m[0], off1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = pack_bf16x2(ex2(y[0][j] - off0), ex2(y[1][j] - off1));
        l[0] += bf16lo(w);
        l[1] += bf16hi(w);
        pw[j] = transpose8(w);
      }
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const uint32_t a[4][4] = {{x.v[0][k].x, x.v[0][k].y, x.v[0][k].z, x.v[0][k].w},
                                  {x.v[1][k].x, x.v[1][k].y, x.v[1][k].z, x.v[1][k].w},
                                  {x.v[2][k].x, x.v[2][k].y, x.v[2][k].z, x.v[2][k].w},
                                  {x.v[3][k].x, x.v[3][k].y, x.v[3][k].z, x.v[3][k].w}};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mma_bf16(acc[4 * k + e], __byte_perm(a[0][e], a[1][e], 0x5410), __byte_perm(a[0][e], a[1][e], 0x7632),
                   __byte_perm(a[2][e], a[3][e], 0x5410), __byte_perm(a[2][e], a[3][e], 0x7632), pw[0], pw[1]);
      }
      if (D == 96) {
        const uint32_t a[4][2] = {{x.w[0].x, x.w[0].y}, {x.w[1].x, x.w[1].y}, {x.w[2].x, x.w[2].y}, {x.w[3].x, x.w[3].y}};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          mma_bf16(acc[D == 96 ? 4 + e : 0], __byte_perm(a[0][e], a[1][e], 0x5410), __byte_perm(a[0][e], a[1][e], 0x7632),
                   __byte_perm(a[2][e], a[3][e], 0x5410), __byte_perm(a[2][e], a[3][e], 0x7632), pw[0], pw[1]);
      }
      if (more && next_row >= 0) load_v<D>(p, next_row, ahead.kvh, x);
    } else if (more && next_row >= 0) {
      load_k<D>(p, next_row, ahead.kvh, x);
      load_v<D>(p, next_row, ahead.kvh, x);
    }
    if (seg_end || !more) {
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        l[hd] += __shfl_xor_sync(kAll, l[hd], 4);
        l[hd] += __shfl_xor_sync(kAll, l[hd], 8);
        l[hd] += __shfl_xor_sync(kAll, l[hd], 16);
      }
      const bool direct = seg_end && whole && c.it.shared == 0;
      const int64_t seg = (int64_t)c.row * vheads + c.kvh * p.head_groups + c.grp;
      // o of head 2t + hd: dims 64 k + 8 g + 2 e + {0, 1} in acc[4 k + e][hd], [2 + hd]; of 96's end 64 + 4 g + 2 e
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        const int head = 2 * t + hd, in_kv = c.grp * kHeads + head;
        if (in_kv >= p.heads_per_kv) continue;
        if (direct) {
          const float f = l[hd] == 0.f ? 0.f : 1.f / l[hd];
          __nv_bfloat16* dst = p.out + (int64_t)c.row * p.out_stride + (int64_t)(c.kvh * p.heads_per_kv + in_kv) * D;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(acc[4 * k + e][hd] * f, acc[4 * k + e][2 + hd] * f);
            *reinterpret_cast<uint4*>(dst + 64 * k + 8 * g) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (D == 96)
            *reinterpret_cast<uint2*>(dst + 64 + 4 * g) =
                make_uint2(pack_bf16x2(acc[MT - 2][hd] * f, acc[MT - 2][2 + hd] * f),
                           pack_bf16x2(acc[MT - 1][hd] * f, acc[MT - 1][2 + hd] * f));
        } else {
          float* dst = p.single + ((seg + warp) * p.stored_heads + head) * (D + 4);
#pragma unroll
          for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
              __stcg(reinterpret_cast<float4*>(dst + 64 * k + 8 * g + 2 * e),
                     make_float4(acc[4 * k + e][hd], acc[4 * k + e][2 + hd], acc[4 * k + e + 1][hd], acc[4 * k + e + 1][2 + hd]));
          if (D == 96)
            __stcg(reinterpret_cast<float4*>(dst + 64 + 4 * g),
                   make_float4(acc[MT - 2][hd], acc[MT - 2][2 + hd], acc[MT - 1][hd], acc[MT - 1][2 + hd]));
          if (g == 0) __stcg(reinterpret_cast<float2*>(dst + D), make_float2(m[hd], l[hd]));
        }
      }
    }
    fresh = seg_end;
    row = next_row;
    c = ahead;
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
    attend_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  const Header h = *p.header;
  if ((int)blockIdx.x < h.shared_ctas) shared_steps<D>(map, p, h, smem);
  else single_rows<D>(p, h);
}

// ---------------------------------------------------------------------------------------------- join

// WARPS warps to a (row, head), each over some of its parts.
template <int D, int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float4 s_o[4][32];
  __shared__ float2 s_ml[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = p.kv_heads * p.heads_per_kv;
  const int64_t unit = WARPS == 1 ? (int64_t)blockIdx.x * 4 + warp : blockIdx.x;
  const int item = (int)(unit / heads), head = (int)(unit - (int64_t)item * heads);
  if (item >= p.num_items) return;
  const Item it = p.items[item];
  if (it.pos < 0) return;
  const Header h = *p.header;
  const int kvh = head / p.heads_per_kv, in_kv = head - kvh * p.heads_per_kv;
  const int grp = in_kv / kHeads, vheads = p.kv_heads * p.head_groups;
  const int own = own_pages(it);
  const int64_t seg = (int64_t)item * vheads + kvh * p.head_groups + grp;
  const int64_t seg0 = p.before[item] * vheads + (int64_t)(kvh * p.head_groups + grp) * own;
  const int64_t c0 = own ? quotient(seg0, h.share) : 0, c1 = own ? quotient(seg0 + own - 1, h.share) : -1;
  Group gr = {};
  int64_t first = 0;
  if (it.shared > 0) {
    gr = p.groups[it.group];
    first = (int64_t)(item - p.group_start[it.group]) * p.heads_per_kv + in_kv;
  }
  const int shared = it.shared > 0 ? gr.splits : 0;
  if (shared == 0 && c0 == c1) return;  // written already
  const int parts = shared + (int)(c1 - c0 + 1);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = (WARPS == 1 ? 0 : warp) * 32; j0 < parts; j0 += WARPS * 32) {
    const int j = j0 + lane;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (j < shared)
      ml = __ldcg(p.shared_ml + gr.base + ((int64_t)kvh * shared + j) * gr.rows + first);
    else if (j < parts)
      ml = __ldcg(reinterpret_cast<const float2*>(
          p.single + ((seg + c0 + j - shared) * p.stored_heads + in_kv - grp * kHeads) * (D + 4) + D));
    const float to = fmaxf(m, warp_max(ml.x));
    const float down = m == -INFINITY ? 0.f : ex2(m - to), f = ml.x == -INFINITY ? 0.f : ex2(ml.x - to);
    m = to;
    l = l * down + warp_sum(ml.y * f);
    o.x *= down, o.y *= down, o.z *= down, o.w *= down;
    const int n = min(32, parts - j0);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float fk = __shfl_sync(kAll, f, k);
      const int jj = j0 + k;
      if (lane < D / 4 && fk != 0.f) {
        const float* src;
        if (jj < shared)
          src = p.shared_o + (gr.base + ((int64_t)kvh * shared + jj) * gr.rows) * D + ((int64_t)(lane >> 1) * gr.rows + first) * 8 + (lane & 1) * 4;
        else
          src = p.single + ((seg + c0 + jj - shared) * p.stored_heads + in_kv - grp * kHeads) * (D + 4) + lane * 4;
        const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
        o.x = fmaf(v.x, fk, o.x), o.y = fmaf(v.y, fk, o.y), o.z = fmaf(v.z, fk, o.z), o.w = fmaf(v.w, fk, o.w);
      }
    }
  }
  if (WARPS > 1) {
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    s_o[warp][lane] = o;
    __syncthreads();
    if (warp != 0) return;
    float to = s_ml[0].x;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) to = fmaxf(to, s_ml[w].x);
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = s_ml[w].x == -INFINITY ? 0.f : ex2(s_ml[w].x - to);
      if (f == 0.f) continue;
      l += s_ml[w].y * f;
      const float4 v = s_o[w][lane];
      o.x += v.x * f, o.y += v.y * f, o.z += v.z * f, o.w += v.w * f;
    }
  }
  if (lane < D / 4) {
    const float f = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + (int64_t)item * p.out_stride + (int64_t)head * D + lane * 4) =
        make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
  }
}

// ---------------------------------------------------------------------------------------------- host

struct Layout {
  int64_t header, items, before, groups, state, shared_o, shared_ml, single, floats;
};

static int64_t padded(int64_t floats) { return (floats + 3) / 4 * 4; }

static Layout layout(int64_t items, int64_t groups, int64_t heads, int64_t kv_heads, int64_t dim, int64_t sms) {
  const int64_t ratio = heads / kv_heads, head_groups = (ratio + kHeads - 1) / kHeads;
  const int64_t stored = ratio < kHeads ? ratio : kHeads, ctas = 2 * sms;
  const int64_t rows = groups > 0 ? TM * ctas + items * heads : 0;  // pieces' shares are no shorter than an even one
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += padded((bytes + 3) / 4);
    return was;
  };
  l.header = take(sizeof(Header));
  l.items = take(items * sizeof(Item));
  l.before = take((items + 1) * sizeof(int64_t));
  l.groups = take((groups + 1) * sizeof(Group));
  l.state = take(groups * sizeof(int2));
  l.shared_o = take(rows * dim * 4);
  l.shared_ml = take(rows * 8);
  l.single = take((items * kv_heads * head_groups + ctas * kWarps) * stored * (dim + 4) * 4);
  l.floats = at;
  return l;
}

template <int D>
static int launch(const Params& p, cudaStream_t st) {
  CUtensorMap map = {};
  EncodeFn encode = tensor_map_encoder();
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.kv_heads, (cuuint64_t)(2 * p.kv_rows)};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.kv_heads * D * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)kBlock}, ones[3] = {1, 1, 1};
  if (encode == nullptr ||
      encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(p.keys), dims, strides, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return CDB_ERR_TMA_ENCODE;
  auto attend = attend_kernel<D>;
  if (allow_shared(reinterpret_cast<const void*>(attend), Tile<D>::SMEM) != cudaSuccess) return CDB_ERR_CUDA;
  if (launch_pdl(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p) != cudaSuccess) return CDB_ERR_CUDA;
  if (launch_pdl(attend, dim3(p.num_ctas), dim3(kThreads), Tile<D>::SMEM, st, map, p) != cudaSuccess)
    return CDB_ERR_CUDA;
  const int64_t units = (int64_t)p.num_items * p.kv_heads * p.heads_per_kv;
  const cudaError_t e = units >= 8 * p.num_ctas
                            ? launch_pdl(join_kernel<D, 1>, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, st, p)
                            : launch_pdl(join_kernel<D, 4>, dim3((unsigned)units), dim3(128), 0, st, p);
  return e == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}

}  // namespace prefix
}  // namespace cdb

extern "C" int64_t cdb_prefix_decode_workspace_floats(int num_items, int num_groups, int num_heads, int num_kv_heads,
                                                      int head_dim, int num_sms) {
  if (num_items < 0 || num_groups < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0 || num_sms <= 0)
    return 0;
  return cdb::prefix::layout(num_items, num_groups, num_heads, num_kv_heads, head_dim, num_sms).floats;
}

extern "C" int cdb_prefix_decode_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                           const void* kv_base, int num_cache_layers, int64_t kv_rows, int cache_layer,
                                           const int32_t* block_table, int64_t block_table_stride, int table_rows,
                                           int table_width, const int32_t* item_slot, const int32_t* item_pos,
                                           int num_items, const int32_t* group_start, const int32_t* prefix_len,
                                           int num_groups, int num_heads, int num_kv_heads, int head_dim, float scale,
                                           int num_sms, float* workspace, int64_t workspace_floats, int32_t* status,
                                           void* stream) {
  using namespace cdb;
  using namespace cdb::prefix;
  if (cache_layer < 0 || cache_layer >= num_cache_layers || kv_rows < kBlock || num_items < 0 || num_groups < 0 ||
      num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows < 0 || table_width < 0 ||
      num_sms <= 0 || !(scale > 0.f) || scale > 1e30f)
    return CDB_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  // cache rows, and the (row, head)s of a call, are counted in 32 bits
  if (2 * kv_rows > 0x7fffffff - 2 * kBlock || (int64_t)num_items * num_heads > 0x3fffffff) return CDB_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_stride & 7) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (out_stride & 7) || (reinterpret_cast<uintptr_t>(kv_base) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_items == 0) return CDB_OK;
  if (q == nullptr || out == nullptr || kv_base == nullptr || block_table == nullptr || item_slot == nullptr ||
      item_pos == nullptr || workspace == nullptr ||
      (num_groups > 0 && (group_start == nullptr || prefix_len == nullptr)))
    return CDB_ERR_INVALID_ARGUMENT;
  const Layout at = layout(num_items, num_groups, num_heads, num_kv_heads, head_dim, num_sms);
  if (workspace_floats < at.floats) return CDB_ERR_INVALID_ARGUMENT;
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.keys = static_cast<const __nv_bfloat16*>(kv_base) + 2 * (int64_t)cache_layer * kv_rows * num_kv_heads * head_dim;
  p.kv_rows = kv_rows;
  p.blocks = (int)(kv_rows / kBlock);
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.bt_rows = table_rows;
  p.bt_width = table_width;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.num_items = num_items;
  p.kv_heads = num_kv_heads;
  p.heads_per_kv = num_heads / num_kv_heads;
  p.head_groups = (p.heads_per_kv + kHeads - 1) / kHeads;
  p.stored_heads = p.heads_per_kv < kHeads ? p.heads_per_kv : kHeads;
  p.tile_items = TM / p.heads_per_kv;
  p.group_start = group_start;
  p.prefix_len = prefix_len;
  p.num_groups = num_groups;
  p.num_ctas = 2 * num_sms;
  p.scale_log2 = scale * kLog2e;
  p.header = reinterpret_cast<Header*>(workspace + at.header);
  p.items = reinterpret_cast<Item*>(workspace + at.items);
  p.before = reinterpret_cast<int64_t*>(workspace + at.before);
  p.groups = reinterpret_cast<Group*>(workspace + at.groups);
  p.state = reinterpret_cast<int2*>(workspace + at.state);
  p.shared_o = workspace + at.shared_o;
  p.shared_ml = reinterpret_cast<float2*>(workspace + at.shared_ml);
  p.single = workspace + at.single;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch<128>(p, st);
  if (head_dim == 96) return launch<96>(p, st);
  return launch<64>(p, st);
}
