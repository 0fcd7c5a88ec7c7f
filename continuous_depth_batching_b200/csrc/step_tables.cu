// A step's metadata from its requests' lengths, on the device: blocks taken from the FIFO ring for the
// tokens to come, block tables, cumulative lengths, and for every new token its slot, position and
// cache row, plus the prefill tiles.
//
// Integer work on a few bytes per request and token, bound by latency: one launch, one CTA or one cluster of
// them (256 requests of one token 5.7 us, 64 of 256 tokens 7.2 us, from a graph of the same call again and again; 7.0
// and 8.4 us as a step makes them, between other work and with other inputs each; an empty launch takes some 2.5).
// Every CTA reads the requests (two dependent loads) and scans them in shared memory, each for itself:
// that costs less than handing the scans round. After one cluster barrier (every read of the allocator's
// state lies before it, every write behind) each CTA writes its share of tokens, tiles and new blocks;
// a token finds its request by bisection in shared memory and its block in the ring or in the request's
// table row, so nobody waits for the table to be written.
#include "cdb_common.cuh"

namespace cdb {
namespace step {

constexpr int kThreads = 1024;
constexpr int kBlock = 16;
constexpr int kTile = 64;
constexpr int kMaxRequests = 8192;

struct Params {
  const int32_t* slots;
  const int32_t* seq_len;  // [table_rows] cached tokens per slot
  const int32_t* new_len;  // [n]
  const int32_t* row_len;  // [table_rows] blocks held per slot
  int32_t* table;
  int64_t table_stride;
  int table_rows, table_width;
  const int32_t* ring;
  int ring_size;
  const int32_t* state;  // {head, free, size, peak}
  int32_t* row_len_out;
  int32_t* state_out;
  int32_t* granted;
  int32_t* cu_q;
  int32_t* cu_k;
  int32_t* item_slot;
  int32_t* item_pos;
  int64_t* slot_map;
  int cap;
  int4* tiles;
  int tile_cap;
  int n;
  int32_t* status;
};

// What is summed over the requests: blocks taken, new tokens, keys, tiles.
constexpr int kSums = 4;
struct Sums {
  int64_t v[kSums];
  __device__ __forceinline__ void add(const Sums& o) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) v[i] += o.v[i];
  }
};

// Block-wide exclusive scan of one Sums per thread; total receives the sum.
__device__ __forceinline__ Sums scan(const Sums& mine, Sums* s_warp, Sums& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  Sums x = mine, y, before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) {
      const int64_t t = __shfl_up_sync(0xffffffffu, x.v[i], o);
      if (lane >= o) x.v[i] += t;
    }
  }
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  y = s_warp[lane];  // every warp sums the warps before it
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) {
      const int64_t t = __shfl_up_sync(0xffffffffu, y.v[i], o);
      if (lane >= o) y.v[i] += t;
    }
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    total.v[i] = __shfl_sync(0xffffffffu, y.v[i], 31);
    const int64_t base = __shfl_sync(0xffffffffu, y.v[i], w > 0 ? w - 1 : 0);
    before.v[i] = x.v[i] - mine.v[i] + (w > 0 ? base : 0);
  }
  return before;
}

// Largest j with first[j] <= i, first ascending from 0 over n entries.
__device__ __forceinline__ int find(const int32_t* first, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) step_tables_kernel(const Params p, int ctas) {
  pdl_trigger();
  extern __shared__ int32_t smem[];
  __shared__ Sums s_warp[2][32];
  const int n = p.n, rank = blockIdx.x;
  int32_t* s_slot = smem;           // [n] -1: no such slot
  int32_t* s_ctx = s_slot + n;      // cached tokens
  int32_t* s_held = s_ctx + n;      // blocks held before
  int32_t* s_need = s_held + n;     // blocks taken now; -1: refused
  int32_t* s_block = s_need + n;    // [n] blocks taken before this request
  int32_t* s_q = s_block + n;       // tokens before this request (its own tokens until they are scanned)
  int32_t* s_t = s_q + n;           // tiles before this request
  pdl_wait();

  const int head = p.state[0], avail = p.state[1], peak = p.state[3];
  const int nb = p.ring_size;
  const bool sane = head >= 0 && head < nb && avail >= 0 && avail <= nb;
  const int per = (n + kThreads - 1) / kThreads;
  const int j0 = min(n, (int)threadIdx.x * per), j1 = min(n, j0 + per);
  constexpr int64_t kMost = 0x7fffffff;  // positions and sums are given in 32 bits
  bool bad = !sane;
  for (int j = j0; j < j1; ++j) {
    const int slot = p.slots[j], fresh = p.new_len[j];
    int ctx = 0, held = 0, need = -1;
    const bool known = slot >= 0 && slot < p.table_rows;
    if (known) {
      ctx = p.seq_len[slot];
      held = p.row_len[slot];
      if (fresh >= 0 && ctx >= 0 && held >= 0) {
        const int64_t total = ((int64_t)ctx + fresh + kBlock - 1) / kBlock;
        if (total <= p.table_width && held <= p.table_width && sane && (int64_t)ctx + fresh <= kMost)
          need = (int)(total > held ? total - held : 0);
      }
    }
    bad = bad || !known || fresh < 0 || ctx < 0 || held < 0 || (int64_t)ctx + fresh > kMost;
    s_slot[j] = known ? slot : -1;
    s_ctx[j] = ctx;
    s_held[j] = held;
    s_need[j] = need;
    s_q[j] = fresh;
  }
  // What a request adds to the sums, and where they begin for this thread's requests.
  auto adds = [&](int j) {
    Sums a = {{0, 0, 0, 0}};
    if (s_need[j] >= 0) a = {{s_need[j], s_q[j], (int64_t)s_ctx[j] + s_q[j], ((int64_t)s_q[j] + kTile - 1) / kTile}};
    return a;
  };
  Sums all;
  auto begin = [&](int which) {
    Sums mine = {{0, 0, 0, 0}};
    for (int j = j0; j < j1; ++j) mine.add(adds(j));
    return scan(mine, s_warp[which], all);
  };
  Sums at = begin(0);
  if (all.v[0] > avail) {  // not enough for everybody: in order, whoever still fits
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = avail;
      for (int j = 0; j < n; ++j)
        if (s_need[j] > left) s_need[j] = -1;
        else if (s_need[j] > 0) left -= s_need[j];
    }
    __syncthreads();
    at = begin(1);
  }
  const int64_t all_b = all.v[0], all_q = all.v[1], all_k = all.v[2], all_t = all.v[3];
  const bool fits = all_q <= p.cap && all_k <= 0x7fffffff && (p.tiles == nullptr || all_t <= p.tile_cap);
  if (ctas > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // Nothing was written so far: every CTA has read slots, lengths and state. Sums past 32 bits stay at the largest
  // number, so that those in shared memory ascend, as the searches below need.
  auto cut = [](int64_t v) { return (int)(v < kMost ? v : kMost); };
  for (int j = j0; j < j1; ++j) {
    const Sums add = adds(j);
    if (rank == 0) {
      p.granted[j] = s_need[j] >= 0 ? 1 : 0;
      p.cu_q[j] = cut(at.v[1]);
      p.cu_k[j] = cut(at.v[2]);
      if (s_need[j] >= 0) p.row_len_out[s_slot[j]] = s_held[j] + s_need[j];
    }
    s_block[j] = (int)at.v[0];
    s_q[j] = cut(at.v[1]);
    s_t[j] = cut(at.v[3]);
    at.add(add);
  }
  if (rank == 0) {
    if (bad || !fits) set_error(p.status, CDB_ERR_INDEX);
    if (threadIdx.x == 0) {
      p.cu_q[n] = cut(all_q);
      p.cu_k[n] = cut(all_k);
      const int taken = (int)all_b;
      p.state_out[0] = sane && nb > 0 ? (int)(((int64_t)head + taken) % nb) : head;
      p.state_out[1] = avail - taken;
      p.state_out[2] = nb;
      p.state_out[3] = max(peak, nb - avail + taken);
    }
  }
  __syncthreads();

  const int first = rank * kThreads + threadIdx.x, step = ctas * kThreads;
  // new blocks into the tables
  for (int i = first; i < (int)all_b; i += step) {
    const int j = find(s_block, n, i);  // the last request that starts at or before i: requests without blocks sort before
    p.table[(int64_t)s_slot[j] * p.table_stride + s_held[j] + i - s_block[j]] = p.ring[(int)(((int64_t)head + i) % nb)];
  }
  // tokens
  const int live = (int)(all_q < p.cap ? all_q : p.cap);
  for (int i = first; i < p.cap; i += step) {
    int slot = -1, pos = -1;
    int64_t row = -1;
    if (i < live) {
      const int j = find(s_q, n, i);
      slot = s_slot[j];
      pos = s_ctx[j] + i - s_q[j];
      const int page = pos / kBlock;
      const int blk = page < s_held[j] ? p.table[(int64_t)slot * p.table_stride + page]
                                       : p.ring[(int)(((int64_t)head + s_block[j] + page - s_held[j]) % nb)];
      row = blk < 0 ? -1 : (int64_t)blk * kBlock + pos % kBlock;
      if (blk < 0) set_error(p.status, CDB_ERR_INDEX);
    }
    p.item_slot[i] = slot;
    p.item_pos[i] = pos;
    p.slot_map[i] = row;
  }
  // tiles of up to 64 rows, in request order
  if (p.tiles != nullptr) {
    const int live_t = (int)(all_t < p.tile_cap ? all_t : p.tile_cap);
    for (int i = first; i < p.tile_cap; i += step) {
      int4 tile = make_int4(0, 0, 0, 0);
      if (i < live_t && fits) {
        const int j = find(s_t, n, i);
        const int at = (i - s_t[j]) * kTile;
        const int rows = (j + 1 < n ? s_q[j + 1] : (int)all_q) - s_q[j];
        tile = make_int4(s_q[j] + at, min(kTile, rows - at), s_slot[j], s_ctx[j] + at);
      }
      p.tiles[i] = tile;
    }
  }
}

}  // namespace step
}  // namespace cdb

extern "C" int cdb_step_tables(const int32_t* slots, const int32_t* seq_len, const int32_t* new_len,
                               const int32_t* row_len, int num_requests, int32_t* block_table,
                               int64_t block_table_stride, int table_rows, int table_width, const int32_t* ring,
                               int ring_size, const int32_t* state, int32_t* row_len_out, int32_t* state_out,
                               int32_t* granted, int32_t* cu_seq_lens_q, int32_t* cu_seq_lens_k, int32_t* item_slot,
                               int32_t* item_pos, int64_t* slot_map, int capacity, void* tiles, int tile_capacity,
                               int32_t* status, void* stream) {
  using namespace cdb;
  using namespace cdb::step;
  if (num_requests < 0 || capacity < 0 || capacity > (1 << 30) || tile_capacity < 0 || tile_capacity > (1 << 30) ||
      table_rows < 0 || table_width < 0 || ring_size < 0 ||
      row_len == nullptr || block_table == nullptr || ring == nullptr || state == nullptr || row_len_out == nullptr ||
      state_out == nullptr || cu_seq_lens_q == nullptr || cu_seq_lens_k == nullptr ||
      (num_requests > 0 && (slots == nullptr || seq_len == nullptr || new_len == nullptr || granted == nullptr)) ||
      (capacity > 0 && (item_slot == nullptr || item_pos == nullptr || slot_map == nullptr)) ||
      (reinterpret_cast<uintptr_t>(tiles) & 15) || (reinterpret_cast<uintptr_t>(slot_map) & 7))
    return CDB_ERR_INVALID_ARGUMENT;
  if (num_requests > kMaxRequests) return CDB_ERR_UNSUPPORTED;
  Params p;
  p.slots = slots;
  p.seq_len = seq_len;
  p.new_len = new_len;
  p.row_len = row_len;
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.table_rows = table_rows;
  p.table_width = table_width;
  p.ring = ring;
  p.ring_size = ring_size;
  p.state = state;
  p.row_len_out = row_len_out;
  p.state_out = state_out;
  p.granted = granted;
  p.cu_q = cu_seq_lens_q;
  p.cu_k = cu_seq_lens_k;
  p.item_slot = item_slot;
  p.item_pos = item_pos;
  p.slot_map = slot_map;
  p.cap = capacity;
  p.tiles = static_cast<int4*>(tiles);
  p.tile_cap = tile_capacity;
  p.n = num_requests;
  p.status = status;
  // One CTA covers a decode step; more tokens are worth a cluster's launch and barrier. One against eight: 256
  // requests of one token 5.1 us (5.5), 1024 tokens 5.4 (5.8), 2048 6.8 (6.2), 16384 20 (7.4).
  const int ctas = capacity <= kThreads ? 1 : 8;
  const size_t smem = (size_t)7 * num_requests * 4;
  if (allow_shared(reinterpret_cast<const void*>(step_tables_kernel), 7 * kMaxRequests * 4) != cudaSuccess)
    return CDB_ERR_CUDA;
  prefer_max_shared(reinterpret_cast<const void*>(step_tables_kernel));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, step_tables_kernel, p, ctas) == cudaSuccess ? CDB_OK : CDB_ERR_CUDA;
}
