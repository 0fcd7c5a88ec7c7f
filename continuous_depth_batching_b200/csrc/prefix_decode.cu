// Decode attention over the bf16 paged cache for requests that share a prompt.
//
// Rows of a group see the same blocks first. For those, Q K^T and P V are matrix products of all the group's
// rows, so a block is read once for up to 256 of them (row x query head of a kv head); behind them every row has pages of
// its own. Softmax parts (m a
// maximum of the logits, l the sum of 2^(x - m), o that of 2^(x - m) v) of any set of keys join by rescaling to
// one m, so the two kinds of work need not wait for each other: one launch does both side by side, and a
// last one joins. Three launches in all:
//   plan    a few CTAs: how many blocks each group shares, where every CTA and warp begins;
//   attend  a CTA an SM, of one kind: shared steps or pages of single rows;
//   join    a warp (or a CTA) per row and head adds up its parts. Rows with one part are written by attend.
// No counters and no atomics between CTAs: parts lie where the plan says, and are added in that order.
//
// Shared steps. Rows are request x query head of a kv head, 128 to a tile. The 64-key steps of all (group, kv head, two
// tiles) form one stream that is cut evenly. In a CTA two teams of four softmax warps, thread r owning row r, have
// accumulators of their own: S = Q K^T (tcgen05, 128 x 64 x D) and O += P V (128 x D x 64), P written over the S that it
// comes from in tensor memory, V as it lies in the cache (the product's inner index across its rows). Each team takes a
// tile through every step; a tile without a partner is taken by both teams, every other step to each. So one team's
// exponentials run beside the other's products, and a step's keys are read once for 256 rows. One warp issues
// each team's products, one brings the pages of K and one those of V (TMA, 128-byte swizzle; one warp for both was what
// bounded a step), five steps ahead.
//
// Pages of single rows. The pages of all (row, kv head, up to 8 query heads) form one stream that is cut into equal
// shares for the warps of the other CTAs. A warp brings its pages into a ring of its own (two pages of 8 KB at 128; with
// 12 warps 192 KB of an SM are on their way) and multiplies them by m16n8k16 products: S^T = K Q^T, O^T = V^T P^T.
//
// The weights P are rounded to bf16 for their product with V (2^-8 of each), V's type. l is their sum in fp32: single rows
// sum the rounded weights, so what is common to them cancels; shared steps, where that took 5 % longer, those before.
// m only moves when passed by 8, which bf16's range allows.
//
// What bounds it (16 to 32 heads of 128, B200 at 1.8 GHz). Single rows: memory, 256 x 2000 tokens on 8 kv heads 328 us from
// a graph of which 319 are their bytes at 6.6 TB/s; plan and join beside it where there is less, 64 x 600 tokens 41 us for 24. Shared steps of one tile: memory too, 32 KB in 0.6 us. Of two
// tiles: a warp's chain, 1700 cycles to a step: 220 until S is there, 100 to read it, 225 for the maximum, 1195 for the
// weights, the other team's on the same unit (1024 of them are 2 x 64 x 8 of the exponential unit). The tensor cores take
// 1024 (1280: at 64 keys S reads q from shared memory faster than that delivers). Measured against it: a quarter of the
// weights by a cubic on the other pipe, 4 % less time for another rounding and NaNs that it hides; more of them, none.
// The plan takes 5 us and the join 5 to 10, most of it waiting for what the launch before wrote.
#include <cuda.h>

#include "tcgen05.cuh"

namespace cdb {
namespace prefix {

constexpr int kBlock = 16;  // tokens of a page
constexpr int TM = 128;     // rows of a shared step
constexpr int TK = 64;      // keys of a shared step
constexpr int kStepPages = TK / kBlock;
constexpr int kWarps = 12;
constexpr int kThreads = kWarps * 32;
constexpr int kPlanThreads = 256;
constexpr int kPlanCtas = 8;
constexpr int kPlanItems = 1024;  // rows, and groups, whose state fits the plan's shared memory
constexpr int kHeads = 8;         // query heads of one single-row segment (n of an m16n8k16 product)
constexpr uint32_t kTmemCols = 256;  // of a team
constexpr uint32_t kAll = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
typedef unsigned long long u64;

// What the plan leaves for the others.
struct Header {
  int shared_ctas;  // CTAs of attend that take shared steps
  int64_t cost;     // of all of their steps
  int64_t share;    // pages of single rows that a warp takes
};
struct alignas(16) Item {
  int pos, slot;     // pos -1: skipped
  int shared;        // its first pages, which its group's steps cover
  int start;         // of the group: its first row,
  int rows, base;    // rows x query heads of a kv head, (row, head)s of the groups before it,
  int64_t cost;      // cost of the groups before it
};
struct alignas(16) Group {
  int pages;      // shared
  int start;      // its first row
  int rows;       // rows x query heads of a kv head
  int slot;       // of its first live row, whose block table is read
  int64_t steps, cost;  // of the groups before it
  int base;       // (row, head)s of the groups before it
};
// Where a CTA of shared steps begins: unit = (kv head, two tiles) of a group, step of the unit; and how many it takes.
struct alignas(16) Start {
  int group, unit, step, count;
  Group g;
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
  int64_t* before;    // [num_items + 1]: own pages of the rows before each
  Group* groups;      // [num_groups + 1]
  int2* state;        // [num_groups] and
  u64* leader;        // [num_groups]: the plan's, where they do not fit shared memory
  Start* starts;      // [num_ctas]
  int4* warps;        // [2][num_ctas * kWarps]: where a warp of single rows begins {row, (kv head, head group), page, how
                      // many pages}, and that row's {position, slot, shared pages}
  int64_t team_rows;  // of all parts of one of the two teams
  float* shared_o;    // parts of shared steps: part (unit, team, CTA) at row team * team_rows + unit's + 128 * CTA, [rows][D]
  float2* shared_ml;  // [rows of parts] {m, l}
  float* single;      // parts of single rows: [segment + warp][stored_heads][D + 4], m and l behind o
  int32_t* status;
};

// Two at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
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

__device__ __forceinline__ int steps_of(int pages) { return (pages + kStepPages - 1) / kStepPages; }
__device__ __forceinline__ int tiles_of(int items, int tile_items) { return (items + tile_items - 1) / tile_items; }

// The last of n places whose value, which never falls, is at most x; the first's is.
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int64_t x, F value) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (value(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// How a call's work is cut, in units of 1/64 us, measured at 16 and 32 heads of 128 as what divides a call best: a CTA
// takes 1 us to a step (HBM) and 1.3 where both teams have 128 rows (exponentials), 0.16 us to a page of single rows. Heads
// of 64 and 96 go by the same numbers, which were not measured for them. What a unit costs a CTA that enters it (q, an empty
// pipeline, O stored) is not counted, and a group's odd last tile counts as a pair: CTAs of equal cost end 45 to 62 us into a
// call of 5 groups.
// Sharing costs another 4 us (more parts, q, tensor memory), so few rows on a short prompt are faster each by itself: 4
// rows on 700 tokens, 16 heads, take 14 us so and 21 shared.
constexpr int kStepCost = 62, kPairCost = 83, kPageCost = 10, kSharedCost = 256;
// Of a step of a group of `rows` (row, head)s, `full` to a tile.
__device__ __forceinline__ int step_cost(int rows, int full) {
  return kStepCost + (kPairCost - kStepCost) * min(max(rows - full, 0), full) / full;
}

struct PlanShared {
  int start[kPlanItems + 1];
  int prefix[kPlanItems];
  int2 state[kPlanItems];  // {fewest whole pages that a row of the group sees, its rows}
  u64 leader[kPlanItems];  // {first live row, its slot}
  Group group[kPlanItems];
  int64_t before[kPlanItems + 1];
  int4 item[kPlanItems];  // {position, slot, shared pages, group}
  int64_t sum[2][32];
  int64_t steps, cost;  // of all groups
  unsigned best;
};

// A thread takes a stretch of the rows, the first warp the groups. Most of it is latencies: the bounds and positions, a
// row's group, the sums. Every CTA does that much for itself, and then takes a part of the rows' and groups' records and of
// the starts (one CTA of 1024 threads: 7.5 us for 64 rows, 2 of them the starts). What does not fit shared memory is left
// to the first CTA alone.
__global__ void __launch_bounds__(kPlanThreads, 1) plan_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t plan_smem[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(plan_smem);
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.best = ~0u;
  pdl_wait();
  int ng = p.tile_items > 0 ? p.num_groups : 0;
  const bool fits = ng <= kPlanItems, fits_items = p.num_items <= kPlanItems;
  if (!(fits && fits_items) && blockIdx.x > 0) return;
  const int ctas_here = fits && fits_items ? kPlanCtas : 1;
  int2* state = fits ? sh.state : p.state;
  u64* leader = fits ? sh.leader : p.leader;
  const int first_pos = tid < p.num_items ? p.item_pos[tid] : -1, first_slot = tid < p.num_items ? p.item_slot[tid] : -1;
  bool bad = false;
  for (int g = tid; g < p.num_groups; g += kPlanThreads) {
    const int a = p.group_start[g], b = p.group_start[g + 1];
    bad |= a < 0 || b < a || b > p.num_items;
    if (g < ng) {
      if (fits) {
        sh.start[g] = a;
        if (g + 1 == ng) sh.start[ng] = b;
        sh.prefix[g] = p.prefix_len[g];
      }
      state[g] = make_int2(INT32_MAX, 0);
      leader[g] = ~0ull;
    }
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) set_error(p.status, CDB_ERR_INDEX);
    ng = 0;
  }
  const int* start = fits ? sh.start : p.group_start;
  const int* prefix = fits ? sh.prefix : p.prefix_len;
  const int per_i = (p.num_items + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(p.num_items, tid * per_i), i1 = min(p.num_items, i0 + per_i);
  // rows {position, slot, -, group}: kept by their thread, or where it has several of them found again
  auto row = [&](int i, bool tell) {
    int4 it = make_int4(i == tid ? first_pos : p.item_pos[i], i == tid ? first_slot : p.item_slot[i], 0, -1);
    if (it.x < 0 || it.y < 0 || it.y >= p.bt_rows || it.x / kBlock >= p.bt_width) {
      if (it.x >= 0 && tell) set_error(p.status, CDB_ERR_INDEX);
      it.x = -1;
    } else if (ng > 0 && start[0] <= i && i < start[ng]) {
      it.w = last_at_most(ng, i, [&](int g) { return (int64_t)start[g]; });
    }
    return it;
  };
  int4 mine = make_int4(-1, -1, 0, -1);
  for (int i = i0; i < i1; ++i) {
    mine = row(i, true);
    if (mine.w >= 0) {
      atomicMin(&state[mine.w].x, (mine.x + 1) / kBlock);
      atomicAdd(&state[mine.w].y, 1);
      atomicMin(&leader[mine.w], (u64)i << 32 | (uint32_t)mine.y);
    }
  }
  __syncthreads();
  auto pages_of = [&](int g) {
    const int2 st = fits ? sh.state[g] : __ldcg(p.state + g);  // (atomics pass the first cache by)
    return st.y >= 2 ? min(max(prefix[g], 0) / kBlock, st.x) : 0;  // one row alone has nothing to share
  };
  auto share_row = [&](int4& it) {
    if (it.w >= 0) it.z = pages_of(it.w);
  };
  auto pages_in = [](const int4& it) { return it.x < 0 ? 0 : it.x / kBlock + 1; };
  // pages of the rows before this thread's: their own ones, and all
  int64_t own = 0, whole = 0;
  for (int i = i0; i < i1; ++i) {
    if (per_i > 1) mine = row(i, false);
    share_row(mine);
    whole += pages_in(mine);
    own += pages_in(mine) - mine.z;
  }
  int64_t x = own, y = whole;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(kAll, x, o), b = __shfl_up_sync(kAll, y, o);
    if (lane >= o) x += a, y += b;
  }
  if (lane == 31) sh.sum[0][warp] = x, sh.sum[1][warp] = y;
  if (warp == 0) {  // the groups: 32 at a time
    int64_t steps0 = 0, rows0 = 0, cost0 = 0;
    for (int base = 0; base < ng; base += 32) {
      const int g = base + lane;
      Group gr = {};
      int64_t steps = 0, rows = 0, cost = 0;
      if (g < ng) {
        gr.pages = pages_of(g);
        gr.start = start[g];
        const int n = start[g + 1] - start[g], tiles = tiles_of(n, p.tile_items);
        gr.rows = n * p.heads_per_kv;
        gr.slot = (int)(uint32_t)(fits ? sh.leader[g] : __ldcg(p.leader + g));
        steps = (int64_t)((tiles + 1) / 2) * p.kv_heads * steps_of(gr.pages);
        cost = steps * step_cost(gr.rows, p.tile_items * p.heads_per_kv);
        rows = (int64_t)gr.rows * p.kv_heads;
      }
      int64_t s = steps, t = rows, u = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = __shfl_up_sync(kAll, s, o), b = __shfl_up_sync(kAll, t, o), c = __shfl_up_sync(kAll, u, o);
        if (lane >= o) s += a, t += b, u += c;
      }
      gr.steps = steps0 + s - steps;
      gr.cost = cost0 + u - cost;
      gr.base = (int)(rows0 + t - rows);
      if (g < ng) {
        if (fits) sh.group[g] = gr;
        else p.groups[g] = gr;
      }
      steps0 += __shfl_sync(kAll, s, 31);
      rows0 += __shfl_sync(kAll, t, 31);
      cost0 += __shfl_sync(kAll, u, 31);
    }
    if (lane == 0) sh.steps = steps0, sh.cost = cost0;
  }
  __syncthreads();
  int64_t all_own, all_whole;
  {
    int64_t a = lane < kPlanThreads / 32 ? sh.sum[0][lane] : 0, b = lane < kPlanThreads / 32 ? sh.sum[1][lane] : 0;
#pragma unroll
    for (int o = 1; o < kPlanThreads / 32; o <<= 1) {
      const int64_t c = __shfl_up_sync(kAll, a, o), d = __shfl_up_sync(kAll, b, o);
      if (lane >= o) a += c, b += d;
    }
    all_own = __shfl_sync(kAll, a, kPlanThreads / 32 - 1), all_whole = __shfl_sync(kAll, b, kPlanThreads / 32 - 1);
    const int64_t c = __shfl_sync(kAll, a, (warp + 31) & 31), d = __shfl_sync(kAll, b, (warp + 31) & 31);
    if (warp > 0) x += c, y += d;
  }
  // the division of the CTAs that is done first, or none
  const int vheads = p.kv_heads * p.head_groups;
  const int64_t all_steps = sh.steps, all_cost = sh.cost;
  const int most_ctas = (int)min(all_cost / kPairCost, (int64_t)p.num_ctas);  // each of them has a step of every unit it is in
  int ctas = 0;
  if (most_ctas > 0) {
    unsigned mine_t = ~0u;
    const float cost = (float)all_cost, rest = (float)(all_own * vheads) * kPageCost;
    for (int c = tid; c <= p.num_ctas; c += kPlanThreads) {
      const float with = cost / (float)min(max(c, 1), most_ctas) + kSharedCost;
      const float time = c == 0             ? (float)(all_whole * vheads) * kPageCost / (float)p.num_ctas
                         : c < p.num_ctas   ? fmaxf(with, rest / (float)(p.num_ctas - c))
                         : rest == 0.f      ? with
                                            : 4e6f;
      mine_t = min(mine_t, (unsigned)fminf(time, 4e6f) << 10 | (unsigned)c);
    }
    mine_t = __reduce_min_sync(kAll, mine_t);
    if (lane == 0) atomicMin(&sh.best, mine_t);
    __syncthreads();
    ctas = min((int)(sh.best & 1023u), most_ctas);
  }
  const bool sharing = ctas > 0;
  const int64_t all_pages = sharing ? all_own : all_whole, vpages = all_pages * vheads;
  int64_t pages = sharing ? x - own : y - whole;
  for (int i = i0; i < i1; ++i) {
    if (per_i > 1) mine = row(i, false);
    if (sharing) share_row(mine);
    else mine.z = 0;
    if (blockIdx.x == 0) p.before[i] = pages;
    if (fits_items) sh.before[i] = pages, sh.item[i] = mine;
    pages += pages_in(mine) - mine.z;
  }
  const int64_t n_warps = (int64_t)(p.num_ctas - ctas) * kWarps;
  const int64_t share = n_warps ? max((int64_t)1, quotient(vpages + n_warps - 1, n_warps)) : 1;
  if (tid == 0) {
    if (blockIdx.x == 0) p.before[p.num_items] = all_pages;
    if (fits_items) sh.before[p.num_items] = all_pages;
    Header h;
    h.shared_ctas = ctas;
    h.cost = all_cost;
    h.share = share;
    if (blockIdx.x == 0) *p.header = h;
  }
  __syncthreads();  // rows and groups are read across threads from here on
  // records and starts, one to a thread
  const int64_t groups_end = (int64_t)p.num_items + (fits && sharing ? ng : 0), ctas_end = groups_end + ctas;
  for (int64_t n = (int64_t)blockIdx.x * kPlanThreads + tid; n < ctas_end + n_warps; n += ctas_here * kPlanThreads) {
    if (n < p.num_items) {
      const int i = (int)n;
      int4 it = fits_items ? sh.item[i] : row(i, false);
      if (!fits_items && sharing) share_row(it);
      Item to = {it.x, it.y, it.z, 0, 0, 0, 0};
      if (it.z > 0) {
        const Group gr = fits ? sh.group[it.w] : p.groups[it.w];
        to.start = gr.start;
        to.rows = gr.rows;
        to.base = gr.base;
        to.cost = gr.cost;
      }
      p.items[i] = to;
    } else if (n < groups_end) {
      const int g = (int)(n - p.num_items);
      p.groups[g] = sh.group[g];
    } else if (n < ctas_end) {
      const int c = (int)(n - groups_end);
      // the first step whose cost begins at or behind the CTA's share of the cost
      auto step_at = [&](int64_t cost, int& group, int64_t& local) {
        group = last_at_most(ng, cost, [&](int g) { return fits ? sh.group[g].cost : p.groups[g].cost; });
        const Group gr = fits ? sh.group[group] : p.groups[group];
        const int w = step_cost(gr.rows, p.tile_items * p.heads_per_kv);
        local = quotient(cost - gr.cost + w - 1, w);
        return gr.steps + local;
      };
      Start st;
      int next_group;
      int64_t local, next_local;
      const int64_t begin = step_at(quotient(all_cost * c, ctas), st.group, local);
      const int64_t end = c + 1 == ctas ? all_steps : step_at(quotient(all_cost * (c + 1), ctas), next_group, next_local);
      st.g = fits ? sh.group[st.group] : p.groups[st.group];
      const int tiles = tiles_of(st.g.rows, p.tile_items * p.heads_per_kv);
      if (local == (int64_t)((tiles + 1) / 2) * p.kv_heads * steps_of(st.g.pages)) {  // behind the group's last
        local = 0;
        do st.g = fits ? sh.group[++st.group] : p.groups[++st.group];
        while (st.g.pages == 0);
      }
      const int per = steps_of(st.g.pages);
      st.unit = (int)quotient(local, per);
      st.step = (int)(local - (int64_t)st.unit * per);
      st.count = (int)(end - begin);
      p.starts[c] = st;
    } else {
      const int64_t w = n - ctas_end;
      const int64_t begin = w * share, end = min(begin + share, vpages);
      int4 from = make_int4(0, 0, 0, 0), of = make_int4(-1, -1, 0, 0);
      if (begin < end) {  // its row is the last that begins at or before it, so one that has pages
        auto before = [&](int i) { return fits_items ? sh.before[i] : p.before[i]; };
        const int i = last_at_most(p.num_items, begin, [&](int j) { return before(j) * vheads; });
        of = fits_items ? sh.item[i] : row(i, false);
        if (!fits_items && sharing) share_row(of);
        const int64_t at = begin - before(i) * vheads;
        const int own_pages = pages_in(of) - of.z;
        from.x = i;
        from.y = (int)quotient(at, own_pages);
        from.z = of.z + (int)(at - (int64_t)from.y * own_pages);
        from.w = (int)min(end - begin, (int64_t)INT32_MAX);
      }
      const int64_t to = (int64_t)ctas * kWarps + w;
      p.warps[to] = from;
      p.warps[(int64_t)p.num_ctas * kWarps + to] = of;
    }
  }
}

// ---------------------------------------------------------------------------------------------- attend

template <int D>
struct Tile {
  static constexpr int ATOMS = (D + 63) / 64;  // 128-byte swizzle atoms of a row of D (96: the second one's end is zero)
  static constexpr int STAGES = D == 64 ? 12 : 5;  // steps in the ring
  static constexpr int STAGE = ATOMS * TK * 128;   // K or V of a step, [ATOMS][64][64]
  static constexpr int Q = ATOMS * TM * 128;       // q of a tile, [ATOMS][128][64]
  static constexpr int OFF_K = 2 * Q;
  static constexpr int OFF_V = OFF_K + STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_V + STAGES * STAGE;
  static constexpr int SMEM = OFF_BAR + 640;
  static_assert(SMEM <= 227 * 1024, "shared memory of an SM");
  // single rows
  static constexpr int BOX = kBlock * 128;        // 64 columns of a page
  static constexpr int PAGE = 2 * ATOMS * BOX;    // K and V of a page
  static constexpr int SLOTS = D == 64 ? 4 : 2;   // pages in a warp's ring
  static_assert(kWarps * SLOTS * PAGE <= OFF_BAR, "rings of all warps");
};

constexpr int kMaxStages = 12;
constexpr int kMissing = 16;  // steps whose missing pages are kept: more than the ring and three steps of either team

struct Shared {
  uint64_t kfull[kMaxStages], vfull[kMaxStages];  // a step's K, V have landed
  uint64_t kfree[kMaxStages], vfree[kMaxStages];  // and both teams have multiplied (or passed) it
  uint64_t qfull, qfree;                          // q of a piece written, and not needed any more
  struct Team {
    uint64_t sfull[2];  // S done, and the step's pages known
    uint64_t pfull[2];  // weights written
    uint64_t odone[2];  // O product done (S's place free)
    uint64_t drain;
  } team[2];
  int missing[kMissing];  // a step's pages that do not exist
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Shared) <= 640, "room behind the tiles");
static_assert(kMissing > kMaxStages + 3, "see Shared");

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

// One lane of a converged warp. (The compiler knows of this one, and not of a compared lane number, that what follows
// runs on a single lane: products, copies and commits then take their operands straight from uniform registers.)
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// The CTA's way through its share of the steps, one unit at a time.
struct Walk {
  Start at;
  Group g;
  int kvh, tile;  // the first of the unit's tiles
  bool both;      // it has two, one to a team
  int steps;      // of this unit that the CTA takes, from step at.step on
  __device__ __forceinline__ int rows(const Params& p, int team) const {
    const int full = p.tile_items * p.heads_per_kv;
    return min(full, g.rows - (both ? tile + team : tile) * full);
  }
  __device__ __forceinline__ void look(const Params& p) {
    const int tiles = tiles_of(g.rows, p.tile_items * p.heads_per_kv), pairs = (tiles + 1) / 2;
    kvh = at.unit / pairs;
    tile = 2 * (at.unit - kvh * pairs);
    both = tile + 1 < tiles;
    steps = min(at.count, steps_of(g.pages) - at.step);
  }
  __device__ __forceinline__ void begin(const Params& p, const Start& s) {
    at = s;
    g = s.g;
    if (at.count > 0) look(p);
  }
  __device__ __forceinline__ bool on() const { return at.count > 0; }
  __device__ __forceinline__ void next(const Params& p) {
    at.count -= steps;
    if (at.count <= 0) return;
    at.step = 0;
    ++at.unit;
    if (at.unit == (tiles_of(g.rows, p.tile_items * p.heads_per_kv) + 1) / 2 * p.kv_heads) {
      at.unit = 0;
      do g = p.groups[++at.group];
      while (g.pages == 0);
    }
    look(p);
  }
};

// (row, head)s of the parts before a unit's: one team's parts of the units in their order, as long as their first tiles.
__device__ __forceinline__ int64_t unit_base(const Params& p, const Group& g, int kvh, int tile) {
  const int full = p.tile_items * p.heads_per_kv, tiles = tiles_of(g.rows, full), pairs = (tiles + 1) / 2;
  const int of_head = (pairs - 1) * full + min(full, g.rows - 2 * (pairs - 1) * full);
  return g.base + (int64_t)kvh * of_head + (int64_t)(tile / 2) * full;
}

template <int D>
__device__ __forceinline__ void shared_steps(const CUtensorMap& map, const Params& p, const Start& start, uint8_t* smem,
                                             Shared& sh) {
  using T = Tile<D>;
  constexpr int R = T::STAGES;
  constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10);  // fp32 accumulators, bf16 operands
  constexpr uint32_t kIdescS = kBf16 | ((uint32_t)(TK >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  constexpr uint32_t kIdescO = kBf16 | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
  const uint32_t base = smem_u32(smem);
  const int warp = __shfl_sync(kAll, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort = &sh.abort;
  Walk w;

  // `t` counts the CTA's steps: step t lies in slot t % R of the ring. `j` counts a team's: its S lies in buffer j & 1. Every
  // barrier's phase follows.
  if (warp == 8 || warp == 11) {
    // ------------------------------------------------------------ pages, of K or of V
    const bool values = warp == 11;
    uint64_t *full = values ? sh.vfull : sh.kfull, *free = values ? sh.vfree : sh.kfree;
    const uint32_t tiles = base + (values ? T::OFF_V : T::OFF_K);
    int t = 0;
    bool ok = true;
    const int page_of = lane & 3;  // of the step
    for (w.begin(p, start); w.on() && ok; w.next(p)) {
      const int32_t* bt = p.block_table + (int64_t)w.g.slot * p.bt_stride;
      auto fetch = [&](int n) {
        const int page = (w.at.step + n) * kStepPages + page_of;
        return n < w.steps && page < w.g.pages ? bt[page] : INT32_MIN;
      };
      int id = fetch(0), next = fetch(1);
      for (int n = 0; n < w.steps; ++n, ++t) {
        const int after = fetch(n + 2), slot = t % R;
        const bool have = id >= 0 && id < p.blocks;
        const unsigned gone = __ballot_sync(kAll, !have) & 15u;
        // behind the cache's rows a box comes as zeros
        const int row = have ? id * kBlock + (values ? (int)p.kv_rows : 0) : 2 * (int)p.kv_rows;
        if (t >= R) ok = __all_sync(kAll, wait_for(&free[slot], (t / R + 1) & 1, p.status, abort));  // by step t - R
        if (!ok) break;
        int rows[kStepPages];
#pragma unroll
        for (int i = 0; i < kStepPages; ++i) rows[i] = __shfl_sync(kAll, row, i);
        if (elect()) {
          if (!values) sh.missing[t % kMissing] = (int)gone;
          mbar_arrive_expect_tx(&full[slot], T::STAGE);
#pragma unroll
          for (int i = 0; i < kStepPages * T::ATOMS; ++i)
            load_box(tiles + slot * T::STAGE + i / kStepPages * (TK * 128) + i % kStepPages * T::BOX, &map,
                     i / kStepPages * 64, w.kvh, rows[i % kStepPages], smem_u32(&full[slot]));
        }
        __syncwarp();
        if (!values && lane < kStepPages && !have && id != INT32_MIN) set_error(p.status, CDB_ERR_INDEX);
        id = next;
        next = after;
      }
    }
    // nothing may be on its way when the CTA ends
    for (int j = max(0, t - R); j < t; ++j) mbar_wait(&full[j % R], (j / R) & 1, p.status);
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------ products
    const int team = warp - 9;
    Shared::Team& tm = sh.team[team];
    const uint32_t tmem = sh.tmem + team * kTmemCols, tmem_o = tmem + 2 * TK;
    int t = 0, j = 0, c = 0;
    bool ok = true;
    auto weigh = [&](int step, int buffer, bool add) {  // O (+)= P V of a step, the team's last one
      ok = ok && wait_for(&sh.vfull[step % R], (step / R) & 1, p.status, abort) &&
           wait_for(&tm.pfull[buffer & 1], (buffer >> 1) & 1, p.status, abort);
      if (!ok) return;
      fence_after();
#pragma unroll
      for (int kk = 0; kk < TK / 16; ++kk)
        product_tmem(tmem_o, tmem + (buffer & 1) * TK + kk * 8,
                     operand(base + T::OFF_V + (step % R) * T::STAGE + kk * 2048, TK * 128), kIdescO, add || kk > 0);
      commit(&tm.odone[buffer & 1]);
      commit(&sh.vfree[step % R]);
    };
    if (elect()) {
      for (w.begin(p, start); w.on() && ok; w.next(p), ++c) {
        ok = wait_for(&sh.qfull, c & 1, p.status, abort);
        const uint32_t q = base + (w.both ? team * T::Q : 0);
        int done = -1;  // the team's last step, whose weights are still to come
        bool add = false;
        for (const int end = t + w.steps; t < end && ok; ++t) {
          const int slot = t % R;
          ok = wait_for(&sh.kfull[slot], (t / R) & 1, p.status, abort);
          if (!ok) break;
          if (!w.both && (t & 1) != team) {  // the other team's
            mbar_arrive(&sh.kfree[slot]);
            ok = wait_for(&sh.vfull[slot], (t / R) & 1, p.status, abort);
            if (ok) mbar_arrive(&sh.vfree[slot]);
            continue;
          }
          if (j >= 2) ok = wait_for(&tm.odone[j & 1], ((j - 2) >> 1) & 1, p.status, abort);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            product(tmem + (j & 1) * TK, operand(q + (kk >> 2) * (TM * 128) + (kk & 3) * 32),
                    operand(base + T::OFF_K + slot * T::STAGE + (kk >> 2) * (TK * 128) + (kk & 3) * 32), kIdescS, kk > 0);
          commit(&tm.sfull[j & 1]);
          commit(&sh.kfree[slot]);
          mbar_arrive(&tm.sfull[j & 1]);  // releases `missing` to whoever waits for S
          if (done >= 0) {
            weigh(done, j - 1, add);
            add = true;
          }
          done = t;
          ++j;
        }
        if (ok && done >= 0) weigh(done, j - 1, add);
      }
      // on every path: no product may run when the tensor memory is freed
      commit(&tm.drain);
      mbar_wait(&tm.drain, 0, p.status);
    }
    __syncwarp();
  } else if (warp < 8) {
    // ------------------------------------------------------------ softmax
    const int team = warp >> 2, quarter = warp & 3;  // of the tensor memory's lanes
    const int r = quarter * 32 + lane;               // row of the tile, and tensor-memory lane
    Shared::Team& tm = sh.team[team];
    const uint32_t tmem = sh.tmem + team * kTmemCols + ((uint32_t)(quarter * 32) << 16), tmem_o = tmem + 2 * TK;
    int t = 0, j = 0, c = 0;
    bool ok = true;
    for (w.begin(p, start); w.on() && ok; w.next(p)) {
      const int rows = w.rows(p, team);
      const bool mine = r < rows;
      const bool rows_here = quarter * 32 < rows;  // a warp without rows only keeps the barriers going
      if (c > 0) {  // both teams are done with the last piece's q
        mbar_arrive(&sh.qfree);
        ok = __all_sync(kAll, wait_for(&sh.qfree, (c - 1) & 1, p.status, abort));
        if (!ok) break;
      }
      ++c;
      {
        const int local = mine ? r / p.heads_per_kv : 0, tile = w.tile + (w.both ? team : 0);
        const __nv_bfloat16* src = p.q + (int64_t)(w.g.start + tile * p.tile_items + local) * p.q_stride +
                                   (int64_t)(w.kvh * p.heads_per_kv + (mine ? r - local * p.heads_per_kv : 0)) * D;
        uint8_t* dst = smem + (w.both ? team * T::Q : 0) + r * 128;
#pragma unroll 1
        for (int half = w.both ? 0 : team; half < (w.both ? 2 : team + 1); ++half) {  // one tile: a half to each team
          uint4 x[D / 16];
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            x[i] = mine ? *reinterpret_cast<const uint4*>(src + (half * (D / 16) + i) * 8) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int ch = half * (D / 16) + i;
            *reinterpret_cast<uint4*>(dst + (ch >> 3) * (TM * 128) + (((ch & 7) ^ (r & 7)) << 4)) = x[i];
          }
        }
      }
      fence_proxy_async_shared();
      mbar_arrive(&sh.qfull);
      float m = -INFINITY, l = 0.f;
      bool some = false;
      for (const int end = t + w.steps; t < end; ++t) {
        if (!w.both && (t & 1) != team) continue;
        ok = __all_sync(kAll, wait_for(&tm.sfull[j & 1], (j >> 1) & 1, p.status, abort));
        if (!ok) break;
        if (rows_here) {
          fence_after();
          uint32_t s[TK];
          tmem_load(tmem + (j & 1) * TK, s);
          tmem_load(tmem + (j & 1) * TK + 32, s + 32);
          wait_loads(s);
          wait_loads(s + 32);
          const int gone = sh.missing[t % kMissing];
          if (gone) {
#pragma unroll
            for (int k = 0; k < TK; ++k)
              if ((gone >> (k / kBlock)) & 1) s[k] = 0xff800000u;
          }
          float x0 = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
          float x1 = fmaxf(__uint_as_float(s[2]), __uint_as_float(s[3]));
#pragma unroll
          for (int k = 4; k < TK; k += 4) {  // (three operands to a maximum)
            x0 = fmaxf(fmaxf(x0, __uint_as_float(s[k])), __uint_as_float(s[k + 1]));
            x1 = fmaxf(fmaxf(x1, __uint_as_float(s[k + 2])), __uint_as_float(s[k + 3]));
          }
          const float mx = fmaxf(x0, x1) * p.scale_log2;
          const bool up = mx > m + 8.f;
          if (__any_sync(kAll, up)) {
            const float to = up ? mx : m;
            if (some) {  // the products so far have to be in O
              ok = __all_sync(kAll, wait_for(&tm.odone[(j - 1) & 1], ((j - 1) >> 1) & 1, p.status, abort));
              if (!ok) break;
              const float down = m == -INFINITY ? (up ? 0.f : 1.f) : ex2(m - to);
              l *= down;
              fence_after();
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                uint32_t o[16];
                tmem_load16(tmem_o + d, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
                tmem_store16(tmem_o + d, o);
              }
              wait_stores();
            }
            m = to;
          }
          const float off = m == -INFINITY ? 0.f : -m;  // (nothing seen yet)
          // (pairs take one instruction: 124 us of steps became 118)
          const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), off2 = make_float2(off, off);
          float2 sum = make_float2(0.f, 0.f), more = sum;
#pragma unroll
          for (int b = 0; b < TK / 16; ++b) {
            uint32_t x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 y = fma2(make_float2(__uint_as_float(s[b * 16 + 2 * k]), __uint_as_float(s[b * 16 + 2 * k + 1])),
                                    scale2, off2);
              const float2 e = make_float2(ex2(y.x), ex2(y.y));
              x[k] = pack_bf16x2(e.x, e.y);
              if (k & 1) more = add2(more, e);
              else sum = add2(sum, e);
            }
            tmem_store8(tmem + (j & 1) * TK + b * 8, x);
          }
          sum = add2(sum, more);
          l += sum.x + sum.y;
          wait_stores();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tm.pfull[j & 1]);
        some = true;
        ++j;
      }
      if (!ok) break;
      if (some) ok = __all_sync(kAll, wait_for(&tm.odone[(j - 1) & 1], ((j - 1) >> 1) & 1, p.status, abort));
      if (!ok) break;
      if (rows_here) {
        const int64_t part =
            team * p.team_rows + unit_base(p, w.g, w.kvh, w.tile) + (int64_t)blockIdx.x * TM;
        if (some) {
          fence_after();
          // O by CH columns through shared memory (q's of this tile, or of the tile that there is not), so that rows
          // leave in whole lines
          constexpr int CH = D == 64 ? 16 : 32, V = CH / 4;
          const uint32_t stage = base + (w.both ? team * T::Q : T::Q + team * (T::Q / 2)) + quarter * (32 * CH * 4);
          float* dst = p.shared_o + (part + quarter * 32) * D;
#pragma unroll 1
          for (int d = 0; d < D; d += CH) {
            uint32_t o[32];
            if constexpr (CH == 32) {
              tmem_load(tmem_o + d, o);
              wait_loads(o);
            } else {
              tmem_load16(tmem_o + d, *reinterpret_cast<uint32_t(*)[16]>(o));
            }
#pragma unroll
            for (int k = 0; k < V; ++k)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * (CH * 4) + ((k ^ (lane & (V - 1))) << 4)),
                           "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3])
                           : "memory");
            __syncwarp();
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const int at = k * (32 / V) + lane / V, ch = lane % V;
              float4 v;
              asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                           : "r"(stage + at * (CH * 4) + ((ch ^ (at & (V - 1))) << 4))
                           : "memory");
              if (quarter * 32 + at < rows) __stcg(reinterpret_cast<float4*>(dst + at * D + d + ch * 4), v);
            }
            __syncwarp();
          }
          fence_before();
        }
        if (mine) __stcg(p.shared_ml + part + r, make_float2(m, l));  // (-inf, 0) where the team had no step
      }
    }
  }
}

// ---------------------------------------------------------------- pages of single rows

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

// Four 8 x 8 matrices of 16-bit values, a row to each lane's address (quarter warps in turn).
__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&m)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_transposed(uint32_t at, uint32_t (&m)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
               : "r"(at)
               : "memory");
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
__device__ __forceinline__ void single_rows(const CUtensorMap& map, const Params& p, const Header& h, uint8_t* smem,
                                            uint64_t* bars) {
  using T = Tile<D>;
  constexpr int MT = D / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, in_cta = threadIdx.x >> 5;
  const int64_t warp = (int64_t)((int)blockIdx.x - h.shared_ctas) * kWarps + in_cta;
  const int4 start = p.warps[(int64_t)blockIdx.x * kWarps + in_cta];
  const int4 first = p.warps[(int64_t)(gridDim.x + blockIdx.x) * kWarps + in_cta];
  const int count = start.w;
  if (count <= 0) return;
  uint64_t* full = bars + in_cta * T::SLOTS;  // a page has landed
  if (lane == 0) {
    for (int i = 0; i < T::SLOTS; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int vheads = p.kv_heads * p.head_groups;
  Cursor c;
  c.row = start.x;
  c.it.pos = first.x;
  c.it.slot = first.y;
  c.it.shared = first.z;
  c.kvh = start.y / p.head_groups;
  c.grp = start.y - c.kvh * p.head_groups;
  c.page = start.z;
  const uint32_t ring = smem_u32(smem) + in_cta * (T::SLOTS * T::PAGE);
  // lane i holds the block id of page i of a window of 32 pages of the row that is being brought
  int win_row = -1, win_first = 0, win_id = -1;
  Cursor ahead = c;
  int issued = 0, put = 0;
  unsigned gone = 0;  // slots whose page does not exist
  auto issue = [&]() {
    const int first = ahead.page & ~31;
    if (ahead.row != win_row || first != win_first) {
      win_row = ahead.row;
      win_first = first;
      win_id = first + lane <= last_page(ahead) ? p.block_table[(int64_t)ahead.it.slot * p.bt_stride + first + lane] : -1;
    }
    const int id = __shfl_sync(kAll, win_id, ahead.page & 31);
    const bool have = id >= 0 && id < p.blocks;
    gone = have ? gone & ~(1u << put) : gone | 1u << put;
    if (lane == 0) {
      if (!have) set_error(p.status, CDB_ERR_INDEX);
      mbar_arrive_expect_tx(&full[put], T::PAGE);
    }
    __syncwarp();
    if (lane < 2 * T::ATOMS) {  // K's columns, then V's; behind the cache's rows a box comes as zeros
      const bool value = lane >= T::ATOMS;
      const int row = have ? id * kBlock + (value ? (int)p.kv_rows : 0) : 2 * (int)p.kv_rows;
      load_box(ring + put * T::PAGE + lane * T::BOX, &map, (lane - (value ? T::ATOMS : 0)) * 64, ahead.kvh, row,
               smem_u32(&full[put]));
    }
    put = put + 1 == T::SLOTS ? 0 : put + 1;
    if (++issued < count) advance(p, ahead);
  };
  for (int i = 0; i < T::SLOTS && issued < count; ++i) issue();

  uint32_t qf[MT][2];
  float acc[MT][4], m[2], l[2];
  bool fresh = true, whole = false;
  int get = 0;
  uint32_t phase = 0;
  // where this lane's row of the four matrices of a product's operand lies: K's 16 tokens x 16 dims, V's transposed
  const int krow = (lane & 7) + (lane & 8), kch = lane >> 4, vrow = (lane & 7) + ((lane >> 4) << 3), vch = (lane >> 3) & 1;
  for (int i = 0; i < count; ++i) {
    if (fresh) {
      const int in_kv = c.grp * kHeads + g;
      const bool on = in_kv < p.heads_per_kv;
      const __nv_bfloat16* src =
          p.q + (int64_t)c.row * p.q_stride + (int64_t)(c.kvh * p.heads_per_kv + (on ? in_kv : 0)) * D + 2 * t;
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        qf[k][0] = on ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        qf[k][1] = on ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
      whole = c.page == c.it.shared;
#pragma unroll
      for (int k = 0; k < MT; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    const bool seg_end = c.page == last_page(c), more = i + 1 < count;
    if (!__all_sync(kAll, mbar_wait(&full[get], phase, p.status))) {
      for (int k = i + 1; k < issued; ++k) {  // a copy that never came: the error is recorded; wait for the others
        get = get + 1 == T::SLOTS ? (phase ^= 1u, 0) : get + 1;
        mbar_wait(&full[get], phase, p.status);
      }
      return;
    }
    if (!((gone >> get) & 1u)) {
      const uint32_t k_at = ring + get * T::PAGE, v_at = k_at + T::ATOMS * T::BOX;
      float s[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) s[k][0] = s[k][1] = s[k][2] = s[k][3] = 0.f;
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        uint32_t a[4];
        load_matrices(k_at + (k >> 2) * T::BOX + krow * 128 + ((((k & 3) * 2 + kch) ^ (krow & 7)) << 4), a);
        mma_bf16(s[k & 1], a[0], a[1], a[2], a[3], qf[k][0], qf[k][1]);
      }
      // y[hd][j]: token g + 8 j, head 2t + hd
      float y[2][2];
#pragma unroll
      for (int hd = 0; hd < 2; ++hd)
#pragma unroll
        for (int j = 0; j < 2; ++j) y[hd][j] = (s[0][2 * j + hd] + s[1][2 * j + hd]) * p.scale_log2;
      // what lies behind the row's end may be anything, NaN too
      const int live = seg_end ? c.it.pos % kBlock + 1 : kBlock;
      if (seg_end) {
#pragma unroll
        for (int hd = 0; hd < 2; ++hd)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (g + 8 * j >= live) y[hd][j] = -INFINITY;
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
      const uint32_t seen0 = (2 * t < live ? 0xffffu : 0u) | (2 * t + 1 < live ? 0xffff0000u : 0u);
      const uint32_t seen1 = (2 * t + 8 < live ? 0xffffu : 0u) | (2 * t + 9 < live ? 0xffff0000u : 0u);
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        uint32_t a[4];
        load_transposed(v_at + (k >> 2) * T::BOX + vrow * 128 + ((((k & 3) * 2 + vch) ^ (vrow & 7)) << 4), a);
        if (seg_end) a[0] &= seen0, a[1] &= seen0, a[2] &= seen1, a[3] &= seen1;
        mma_bf16(acc[k], a[0], a[1], a[2], a[3], pw[0], pw[1]);
      }
    }
    get = get + 1 == T::SLOTS ? (phase ^= 1u, 0) : get + 1;
    __syncwarp();  // every lane has read the page
    if (issued < count) issue();
    if (seg_end || !more) {
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        l[hd] += __shfl_xor_sync(kAll, l[hd], 4);
        l[hd] += __shfl_xor_sync(kAll, l[hd], 8);
        l[hd] += __shfl_xor_sync(kAll, l[hd], 16);
      }
      const bool direct = seg_end && whole && c.it.shared == 0;
      const int64_t seg = (int64_t)c.row * vheads + c.kvh * p.head_groups + c.grp;
      // o of head 2t + hd: dims 16 k + g in acc[k][hd], 16 k + 8 + g in acc[k][2 + hd]
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        const int head = 2 * t + hd, in_kv = c.grp * kHeads + head;
        if (in_kv >= p.heads_per_kv) continue;
        if (direct) {
          const float f = l[hd] == 0.f ? 0.f : 1.f / l[hd];
          __nv_bfloat16* dst =
              p.out + (int64_t)c.row * p.out_stride + (int64_t)(c.kvh * p.heads_per_kv + in_kv) * D + g;
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            dst[k * 16] = f_to_bf16(acc[k][hd] * f);
            dst[k * 16 + 8] = f_to_bf16(acc[k][2 + hd] * f);
          }
        } else {
          float* dst = p.single + ((seg + warp) * p.stored_heads + head) * (D + 4) + g;
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            __stcg(dst + k * 16, acc[k][hd]);
            __stcg(dst + k * 16 + 8, acc[k][2 + hd]);
          }
          if (g == 0) __stcg(reinterpret_cast<float2*>(dst + D), make_float2(m[hd], l[hd]));
        }
      }
    }
    fresh = seg_end;
    if (more) advance(p, c);
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  const Header h = *p.header;
  const int warp = threadIdx.x >> 5;
  if ((int)blockIdx.x >= h.shared_ctas) {
    pdl_trigger();
    single_rows<D>(map, p, h, smem, reinterpret_cast<uint64_t*>(smem + Tile<D>::OFF_BAR));
    return;
  }
  const Start start = p.starts[blockIdx.x];
  Shared& sh = *reinterpret_cast<Shared*>(smem + Tile<D>::OFF_BAR);
  if (threadIdx.x == 0) {
    for (int i = 0; i < Tile<D>::STAGES; ++i) {
      mbar_init(&sh.kfull[i], 1);
      mbar_init(&sh.vfull[i], 1);
      mbar_init(&sh.kfree[i], 2);
      mbar_init(&sh.vfree[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      Shared::Team& tm = sh.team[i >> 1];
      mbar_init(&tm.sfull[i & 1], 2);
      mbar_init(&tm.pfull[i & 1], TM / 32);
      mbar_init(&tm.odone[i & 1], 1);
      if (i & 1) mbar_init(&tm.drain, 1);
    }
    mbar_init(&sh.qfull, 2 * TM);
    mbar_init(&sh.qfree, 2 * TM);
    sh.abort = (smem_u32(smem) & 1023u) != 0u;  // the swizzle counts on it
    if (sh.abort) set_error(p.status, CDB_ERR_INVALID_ARGUMENT);
    fence_barrier_init();
  }
  if (warp == 11) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(2 * kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // Only now may the next kernel's CTAs come: one that holds tensor memory and waits for this kernel could otherwise
  // be what the allocation above waits for.
  pdl_trigger();
  shared_steps<D>(map, p, start, smem, sh);
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 11)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(2 * kTmemCols) : "memory");
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
  int shared = 0;            // parts of shared steps
  bool both = false;         // a CTA has one of this tile's, not two
  int64_t part = 0;          // its row in the first of them
  const float* shared_o = nullptr;
  if (it.shared > 0) {
    Group gr;
    gr.rows = it.rows;
    gr.base = it.base;
    const int local = item - it.start, tile = local / p.tile_items, in_tile = local - tile * p.tile_items;
    const int n = steps_of(it.shared), full = p.tile_items * p.heads_per_kv, tiles = tiles_of(gr.rows, full);
    both = (tile | 1) < tiles;
    // the CTAs that hold the unit's steps: CTA c takes those that begin at costs [cost c / ctas, cost (c + 1) / ctas)
    const int w = step_cost(it.rows, full);
    const int64_t s0 = it.cost + ((int64_t)kvh * ((tiles + 1) / 2) + tile / 2) * n * w, s1 = s0 + (int64_t)(n - 1) * w;
    const int64_t b0 = quotient((s0 + 1) * h.shared_ctas - 1, h.cost), b1 = quotient((s1 + 1) * h.shared_ctas - 1, h.cost);
    shared = (both ? 1 : 2) * (int)(b1 - b0 + 1);
    const int64_t base = unit_base(p, gr, kvh, tile) + b0 * TM + (both ? (tile & 1) * p.team_rows : 0);
    part = base + in_tile * p.heads_per_kv + in_kv;
    shared_o = p.shared_o + part * D;
  }
  // part j of the shared ones: a CTA's, or one of its two teams'
  auto place = [&](int j) { return both ? (int64_t)j * TM : (j & 1) * p.team_rows + (int64_t)(j >> 1) * TM; };
  if (shared == 0 && c0 == c1) return;  // written already
  const int parts = shared + (int)(c1 - c0 + 1);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const int in_warp = WARPS == 1 ? 0 : warp;
  // Eight parts of a warp at a time, {m, l} and o of all of them requested at once.
  for (int j0 = in_warp; j0 < parts; j0 += 8 * WARPS) {
    auto single_part = [&](int j) {
      return p.single + ((seg + c0 + j - shared) * p.stored_heads + in_kv - grp * kHeads) * (D + 4);
    };
    float2 ml = make_float2(-INFINITY, 0.f);
    const int j = j0 + lane * WARPS;
    if (lane < 8 && j < parts)
      ml = __ldcg(j < shared ? p.shared_ml + part + place(j) : reinterpret_cast<const float2*>(single_part(j) + D));
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int jj = j0 + k * WARPS;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane < D / 4 && jj < parts)
        v[k] = __ldcg(reinterpret_cast<const float4*>(
            (jj < shared ? shared_o + place(jj) * D : single_part(jj)) + lane * 4));
    }
    const float to = fmaxf(m, warp_max(ml.x));
    const float down = m == -INFINITY ? 0.f : ex2(m - to), f = ml.x == -INFINITY ? 0.f : ex2(ml.x - to);
    m = to;
    l = l * down + warp_sum(ml.y * f);
    o.x *= down, o.y *= down, o.z *= down, o.w *= down;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float fk = __shfl_sync(kAll, f, k);
      if (fk == 0.f) continue;  // (a part without keys has no o)
      o.x = fmaf(v[k].x, fk, o.x), o.y = fmaf(v[k].y, fk, o.y), o.z = fmaf(v[k].z, fk, o.z), o.w = fmaf(v[k].w, fk, o.w);
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
  int64_t header, items, before, groups, state, leader, starts, warps, shared_o, shared_ml, single, floats;
};

static int64_t padded(int64_t floats) { return (floats + 3) / 4 * 4; }

static Layout layout(int64_t items, int64_t groups, int64_t heads, int64_t kv_heads, int64_t dim, int64_t sms) {
  const int64_t ratio = heads / kv_heads, head_groups = (ratio + kHeads - 1) / kHeads;
  const int64_t stored = ratio < kHeads ? ratio : kHeads;
  const int64_t rows = groups > 0 ? 2 * (sms * TM + items * heads) : 0;  // of both teams' parts
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
  l.leader = take(groups * sizeof(u64));
  l.starts = take(sms * sizeof(Start));
  l.warps = take(2 * sms * kWarps * sizeof(int4));
  l.shared_o = take(rows * dim * 4);
  l.shared_ml = take(rows * 8);
  l.single = take((items * kv_heads * head_groups + sms * kWarps) * stored * (dim + 4) * 4);
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
  if (allow_shared(reinterpret_cast<const void*>(plan_kernel), sizeof(PlanShared)) != cudaSuccess ||
      launch_pdl(plan_kernel, dim3(kPlanCtas), dim3(kPlanThreads), sizeof(PlanShared), st, p) != cudaSuccess)
    return CDB_ERR_CUDA;
  if (launch_pdl(attend, dim3(p.num_ctas), dim3(kThreads), Tile<D>::SMEM, st, map, p) != cudaSuccess)
    return CDB_ERR_CUDA;
  const int64_t units = (int64_t)p.num_items * p.kv_heads * p.heads_per_kv;
  const cudaError_t e = units >= 16 * p.num_ctas
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
      num_sms < 2 || num_sms > 1023 || !(scale > 0.f) || scale > 1e30f)
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
  p.num_ctas = num_sms;
  p.scale_log2 = scale * kLog2e;
  p.header = reinterpret_cast<Header*>(workspace + at.header);
  p.items = reinterpret_cast<Item*>(workspace + at.items);
  p.before = reinterpret_cast<int64_t*>(workspace + at.before);
  p.groups = reinterpret_cast<Group*>(workspace + at.groups);
  p.state = reinterpret_cast<int2*>(workspace + at.state);
  p.leader = reinterpret_cast<u64*>(workspace + at.leader);
  p.starts = reinterpret_cast<Start*>(workspace + at.starts);
  p.warps = reinterpret_cast<int4*>(workspace + at.warps);
  p.team_rows = (int64_t)num_sms * TM + (int64_t)num_items * num_heads;
  p.shared_o = workspace + at.shared_o;
  p.shared_ml = reinterpret_cast<float2*>(workspace + at.shared_ml);
  p.single = workspace + at.single;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch<128>(p, st);
  if (head_dim == 96) return launch<96>(p, st);
  return launch<64>(p, st);
}
