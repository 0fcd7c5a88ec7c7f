// torch.ops.cdb.* of the low-bit decode step and of many continuations of one prompt: argument checks (types and shapes
// first, then the device,
// so that a call with CPU tensors is told what else is wrong with it), workspaces and the launch on the current
// stream, over the C ABI. In C++ because a decode step makes hundreds of these calls and each kernel
// takes a few microseconds: the same checks cost 17 us of host time a call in Python.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <limits>
#include <map>
#include <mutex>
#include <optional>
#include <tuple>
#include <utility>

#include "../../include/cdb_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 16;  // tokens of one block of the 8-bit cache

void same_device(const Tensor& t, std::optional<c10::Device>& dev) {
  TORCH_CHECK(t.is_cuda(), "torch.ops.cdb kernels run on CUDA tensors only (sm_100a); there is no CPU path");
  if (!dev) dev = t.device();
  TORCH_CHECK_VALUE(t.device() == *dev, "all tensors must be on one device, got ", *dev, " and ", t.device());
}
void same_device(const OptTensor& t, std::optional<c10::Device>& dev) {
  if (t) same_device(*t, dev);
}
template <typename... T>
c10::Device one_device(const T&... ts) {
  std::optional<c10::Device> dev;
  (same_device(ts, dev), ...);
  return *dev;
}

// The C ABI counts in 32 bits; cut to them, a larger number would pass for another.
int as_int(const char* name, int64_t v) {
  TORCH_CHECK_VALUE(v <= std::numeric_limits<int>::max(), name, " must be below 2^31, got ", v);
  return (int)v;
}

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// A 2-D bf16 tensor of at least rows x cols whose rows may be accessed 16 bytes at a time.
void check_rows(const char* name, const Tensor& t, int64_t rows, int64_t cols) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) >= rows && t.size(1) >= cols, name,
                    " must be a 2-D bf16 tensor of at least ", rows, " x ", cols, ", got ", t.scalar_type(), " ",
                    t.sizes());
  TORCH_CHECK_VALUE(t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= cols) && t.stride(0) % 8 == 0 && aligned16(t),
                    name, " needs unit column stride, a row stride that is a multiple of 8 and 16-byte alignment");
}

void check_ints(const char* name, const Tensor& t, int64_t n, at::ScalarType type = at::kInt) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 1 && t.size(0) >= n && t.is_contiguous(), name,
                    " must be a contiguous 1-D ", type, " tensor of at least ", n, " entries, got ", t.scalar_type(),
                    " ", t.sizes());
}

void check_table(const Tensor& t) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&
                        (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
                    "block_table must be a 2-D int32 tensor with unit column stride, got ", t.scalar_type(), " ",
                    t.sizes());
  as_int("block_table's rows", t.size(0));
  as_int("block_table's columns", t.size(1));
}

void check_tiles(const Tensor& t) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) == 4 && t.is_contiguous() && aligned16(t),
                    "tiles must be a contiguous 16-byte aligned int32 tensor [n, 4], got ", t.scalar_type(), " ",
                    t.sizes());
}

struct Cache {
  int layers, blocks, heads, dim;
};

Cache check_cache(const Tensor& codes, const Tensor& scales, int64_t layer) {
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kFloat8_e4m3fn && codes.dim() == 6 && codes.is_contiguous() &&
                        codes.size(1) == 2 && codes.size(4) == kBlock && codes.size(2) > 0 && codes.size(3) > 0,
                    "codes must be a contiguous float8_e4m3fn tensor [layers, 2, blocks, kv heads, 16, head dim], got ",
                    codes.scalar_type(), " ", codes.sizes());
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat && scales.sizes() == codes.sizes().slice(0, 4) &&
                        scales.is_contiguous(),
                    "scales must be a contiguous fp32 tensor ", codes.sizes().slice(0, 4), ", got ",
                    scales.scalar_type(), " ", scales.sizes());
  const int64_t dim = codes.size(5);
  TORCH_CHECK_VALUE(dim == 64 || dim == 96 || dim == 128, "the 8-bit cache takes head dims 64, 96 and 128, got ", dim);
  TORCH_CHECK_VALUE(layer >= 0 && layer < codes.size(0), "cache_layer must be in [0, ", codes.size(0), "), got ", layer);
  TORCH_CHECK_VALUE(aligned16(codes), "codes must be 16-byte aligned");
  return {as_int("layers", codes.size(0)), as_int("blocks", codes.size(2)), as_int("kv heads", codes.size(3)), (int)dim};
}

void check_heads(int64_t heads, int64_t kv_heads) {
  TORCH_CHECK_VALUE(heads > 0 && heads % kv_heads == 0, "num_heads must be a positive multiple of the cache's ", kv_heads,
                    " kv heads, got ", heads);
  as_int("num_heads", heads);
}

template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(const_cast<void*>(t.const_data_ptr()));
}
template <typename T>
T* ptr(const OptTensor& t) {
  return t ? ptr<T>(*t) : nullptr;
}

std::mutex g_mutex;

// The device-side status word that all ops of a device share; allocated by the first call.
const Tensor& status_word(c10::Device dev) {
  static auto& words = *new std::map<int, Tensor>;  // never destroyed: the device may be gone by then
  std::lock_guard<std::mutex> lock(g_mutex);
  Tensor& word = words[dev.index()];
  if (!word.defined()) {
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
                "torch.ops.cdb: the first call on a device allocates the shared status word; make one call before "
                "capturing a CUDA graph");
    word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(dev));
    c10::cuda::getCurrentCUDAStream(dev.index()).synchronize();  // calls on other streams may write it next
  }
  return word;
}

int sm_count(c10::Device dev) {
  static std::map<int, int> counts;
  std::lock_guard<std::mutex> lock(g_mutex);
  int& n = counts[dev.index()];
  if (n == 0) C10_CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev.index()));
  return n;
}

void check(int rc, const char* what) { TORCH_CHECK(rc == CDB_OK, what, " failed: ", cdb_status_string(rc), " (status ", rc, ")"); }

// Piece buffer and arrival counters of a decode attention (`op` tells them apart). Eager calls keep one per stream, so
// that calls on two streams never share one, and hold its lock until all their launches are on the stream: what a call's
// launches hand on to one another must not be overwritten by those of another host thread's call on that stream. A captured
// call takes its own from the graph's memory and zeroes the counters inside the graph, so that two graphs may be replayed
// at once.
enum Op { kKv8Decode, kPrefixDecode };
struct Workspace {
  Tensor floats, counters;
  std::unique_lock<std::mutex> lock;
};
Workspace workspace(Op op, c10::Device dev, c10::cuda::CUDAStream stream, int64_t floats, int64_t counters) {
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  const auto i32 = at::TensorOptions().dtype(at::kInt).device(dev);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return {at::empty({floats}, f32), at::zeros({counters}, i32), {}};
  struct Kept {
    std::mutex launches;
    Tensor floats, counters;
  };
  static auto& kept = *new std::map<std::tuple<Op, int, cudaStream_t>, Kept>;  // (whose places never move)
  Kept* ws;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    ws = &kept[{op, dev.index(), stream.stream()}];
  }
  std::unique_lock<std::mutex> lock(ws->launches);
  if (!ws->floats.defined() || ws->floats.numel() < floats || ws->counters.numel() < counters)
    ws->floats = at::empty({floats}, f32), ws->counters = at::zeros({counters}, i32);
  return {ws->floats, ws->counters, std::move(lock)};
}

// The rotation's tables; returns their positions.
int check_rope(const OptTensor& rope_cos, const OptTensor& rope_sin, int64_t rope_mode, int64_t dim) {
  TORCH_CHECK_VALUE(rope_mode >= 0 && rope_mode <= 2,
                    "rope_mode must be 0 (none), 1 (split halves) or 2 (interleaved pairs), got ", rope_mode);
  if (rope_mode == 0) return 0;
  TORCH_CHECK_VALUE(rope_cos && rope_sin && rope_cos->sizes() == rope_sin->sizes(),
                    "rope_cos and rope_sin must be given, with one shape, when rope_mode is not 0");
  const auto type = rope_mode == 1 ? at::kBFloat16 : at::kFloat;
  const int64_t cols = rope_mode == 1 ? dim : dim / 2;
  for (const Tensor* t : {&*rope_cos, &*rope_sin})
    TORCH_CHECK_VALUE(t->scalar_type() == type && t->dim() == 2 && t->size(1) == cols && t->is_contiguous() &&
                          aligned16(*t),
                      "rope_cos and rope_sin must be contiguous 16-byte aligned ", type, " tensors [positions, ", cols,
                      "] in rope_mode ", rope_mode);
  return as_int("rope_cos's positions", rope_cos->size(0));
}

void kv8_append(const Tensor& qkv, const OptTensor& q_out, const Tensor& codes, const Tensor& scales,
                int64_t cache_layer, const Tensor& block_table, const Tensor& item_slot, const Tensor& item_pos,
                const OptTensor& rope_cos, const OptTensor& rope_sin, const OptTensor& qk_bias, int64_t rope_mode,
                int64_t num_heads) {
  const Cache c = check_cache(codes, scales, cache_layer);
  const int64_t n = as_int("item_pos's entries", item_pos.numel());
  TORCH_CHECK_VALUE(num_heads > 0, "num_heads must be positive, got ", num_heads);
  as_int("num_heads", num_heads);
  check_rows("qkv", qkv, n, (num_heads + 2 * c.heads) * c.dim);
  if (q_out) check_rows("q_out", *q_out, n, num_heads * c.dim);
  check_ints("item_pos", item_pos, n);
  check_ints("item_slot", item_slot, n);
  check_table(block_table);
  const int rope_rows = check_rope(rope_cos, rope_sin, rope_mode, c.dim);
  TORCH_CHECK_VALUE(!qk_bias || (qk_bias->scalar_type() == at::kBFloat16 &&
                                 qk_bias->numel() == (num_heads + c.heads) * c.dim && qk_bias->is_contiguous() &&
                                 aligned16(*qk_bias)),
                    "qk_bias must be a contiguous 16-byte aligned bf16 tensor of ", num_heads, " + ", c.heads,
                    " heads of ", c.dim);
  const auto dev = one_device(qkv, q_out, codes, scales, block_table, item_slot, item_pos, rope_cos, rope_sin, qk_bias);
  const c10::cuda::CUDAGuard guard(dev);
  const bool rope = rope_mode != 0;
  check(cdb_kv8_append(ptr<void>(qkv), qkv.stride(0), ptr<void>(q_out), q_out ? q_out->stride(0) : 0, ptr<void>(codes),
                       ptr<float>(scales), c.layers, (int)cache_layer, c.blocks, ptr<int32_t>(block_table),
                       block_table.stride(0), (int)block_table.size(0), (int)block_table.size(1),
                       ptr<int32_t>(item_slot), ptr<int32_t>(item_pos), (int)rope_mode,
                       rope ? ptr<void>(rope_cos) : nullptr, rope ? ptr<void>(rope_sin) : nullptr, rope_rows,
                       ptr<void>(qk_bias), (int)n, (int)num_heads, c.heads, c.dim, ptr<int32_t>(status_word(dev)),
                       c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_kv8_append");
}

void kv8_gather(const Tensor& codes, const Tensor& scales, int64_t cache_layer, const Tensor& blocks,
                const Tensor& out) {
  const Cache c = check_cache(codes, scales, cache_layer);
  const int64_t n = as_int("blocks' entries", blocks.numel());
  check_ints("blocks", blocks, n);
  TORCH_CHECK_VALUE(out.scalar_type() == at::kBFloat16 && out.dim() == 5 && out.size(0) == n && out.size(1) == 2 &&
                        out.size(2) == c.heads && out.size(3) == kBlock && out.size(4) == c.dim &&
                        out.is_contiguous() && aligned16(out),
                    "out must be a contiguous 16-byte aligned bf16 tensor [", n, ", 2, ", c.heads, ", 16, ", c.dim,
                    "], got ", out.scalar_type(), " ", out.sizes());
  const auto dev = one_device(codes, scales, blocks, out);
  const c10::cuda::CUDAGuard guard(dev);
  check(cdb_kv8_gather(ptr<void>(codes), ptr<float>(scales), c.layers, (int)cache_layer, c.blocks, c.heads, c.dim,
                       ptr<int32_t>(blocks), (int)n, ptr<void>(out), ptr<int32_t>(status_word(dev)),
                       c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_kv8_gather");
}

void check_scale(double scale) {
  TORCH_CHECK_VALUE(scale > 0 && scale <= 1e30, "scale must be positive and finite, got ", scale);
}

void kv8_decode_attention(const Tensor& q, const Tensor& out, const Tensor& codes, const Tensor& scales,
                          int64_t cache_layer, const Tensor& block_table, const Tensor& item_slot,
                          const Tensor& item_pos, int64_t num_heads, double scale) {
  const Cache c = check_cache(codes, scales, cache_layer);
  check_heads(num_heads, c.heads);
  check_scale(scale);
  const int64_t n = as_int("item_pos's entries", item_pos.numel());
  check_rows("q", q, n, num_heads * c.dim);
  check_rows("out", out, n, num_heads * c.dim);
  check_ints("item_pos", item_pos, n);
  check_ints("item_slot", item_slot, n);
  check_table(block_table);
  const auto dev = one_device(q, out, codes, scales, block_table, item_slot, item_pos);
  const c10::cuda::CUDAGuard guard(dev);
  const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const int ctas = sm_count(dev);
  const Tensor& status = status_word(dev);
  const Workspace ws = workspace(kKv8Decode, dev, stream, cdb_kv8_decode_workspace_floats(ctas, c.dim),
                                 cdb_kv8_decode_counters(ctas));
  check(cdb_kv8_decode_attention(ptr<void>(q), q.stride(0), ptr<void>(out), out.stride(0), ptr<void>(codes),
                                 ptr<float>(scales), c.layers, (int)cache_layer, c.blocks, ptr<int32_t>(block_table),
                                 block_table.stride(0), (int)block_table.size(0), (int)block_table.size(1),
                                 ptr<int32_t>(item_slot), ptr<int32_t>(item_pos), (int)n, (int)num_heads, c.heads,
                                 c.dim, (float)scale, ctas, ptr<float>(ws.floats), ws.floats.numel(),
                                 ptr<int32_t>(ws.counters), ptr<int32_t>(status), stream.stream()),
        "cdb_kv8_decode_attention");
}

void kv8_prefill_attention(const Tensor& q, const Tensor& out, const Tensor& codes, const Tensor& scales,
                           int64_t cache_layer, const Tensor& block_table, const Tensor& tiles, int64_t num_heads,
                           double scale) {
  const Cache c = check_cache(codes, scales, cache_layer);
  check_heads(num_heads, c.heads);
  check_scale(scale);
  check_rows("q", q, 0, num_heads * c.dim);
  as_int("q's rows", q.size(0));
  check_rows("out", out, q.size(0), num_heads * c.dim);
  check_table(block_table);
  check_tiles(tiles);
  TORCH_CHECK_VALUE(tiles.size(0) <= 65535, "one call takes at most 65535 tiles, got ", tiles.size(0));
  const auto dev = one_device(q, out, codes, scales, block_table, tiles);
  const c10::cuda::CUDAGuard guard(dev);
  check(cdb_kv8_prefill_attention(ptr<void>(q), q.stride(0), ptr<void>(out), out.stride(0), (int)q.size(0),
                                  ptr<void>(codes), ptr<float>(scales), c.layers, (int)cache_layer, c.blocks,
                                  ptr<int32_t>(block_table), block_table.stride(0), (int)block_table.size(0),
                                  (int)block_table.size(1), ptr<void>(tiles), (int)tiles.size(0), (int)num_heads,
                                  c.heads, c.dim, (float)scale, ptr<int32_t>(status_word(dev)),
                                  c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_kv8_prefill_attention");
}

void step_tables(const Tensor& slots, const Tensor& seq_len, const Tensor& new_len, const Tensor& row_len,
                 const Tensor& block_table, const Tensor& ring, const Tensor& state, const Tensor& row_len_out,
                 const Tensor& state_out, const Tensor& granted, const Tensor& cu_q, const Tensor& cu_k,
                 const Tensor& item_slot, const Tensor& item_pos, const Tensor& slot_map, const OptTensor& tiles) {
  const int64_t n = slots.numel(), rows = as_int("row_len's entries", row_len.numel()), cap = item_pos.numel();
  TORCH_CHECK_VALUE(cap <= 1 << 30, "one call takes at most 2^30 tokens, got ", cap);
  as_int("ring's entries", ring.numel());
  check_ints("slots", slots, n);
  check_ints("new_len", new_len, n);
  check_ints("granted", granted, n);
  check_ints("cu_seq_lens_q", cu_q, n + 1);
  check_ints("cu_seq_lens_k", cu_k, n + 1);
  check_ints("row_len", row_len, rows);
  check_ints("row_len_out", row_len_out, rows);
  check_ints("seq_len", seq_len, rows);
  check_ints("ring", ring, 0);
  check_ints("state", state, 4);
  check_ints("state_out", state_out, 4);
  check_ints("item_pos", item_pos, cap);
  check_ints("item_slot", item_slot, cap);
  check_ints("slot_map", slot_map, cap, at::kLong);
  check_table(block_table);
  TORCH_CHECK_VALUE(block_table.size(0) >= rows, "block_table needs a row for each of the ", rows, " slots, got ",
                    block_table.size(0));
  TORCH_CHECK_VALUE(n <= 8192, "one call takes at most 8192 requests, got ", n);
  if (tiles) check_tiles(*tiles);
  TORCH_CHECK_VALUE(!tiles || tiles->size(0) <= 1 << 30, "one call takes at most 2^30 tiles, got ", tiles->size(0));
  const auto dev = one_device(slots, seq_len, new_len, row_len, block_table, ring, state, row_len_out, state_out,
                              granted, cu_q, cu_k, item_slot, item_pos, slot_map, tiles);
  const c10::cuda::CUDAGuard guard(dev);
  check(cdb_step_tables(ptr<int32_t>(slots), ptr<int32_t>(seq_len), ptr<int32_t>(new_len), ptr<int32_t>(row_len), (int)n,
                        ptr<int32_t>(block_table), block_table.stride(0), (int)rows, (int)block_table.size(1),
                        ptr<int32_t>(ring), (int)ring.numel(), ptr<int32_t>(state), ptr<int32_t>(row_len_out),
                        ptr<int32_t>(state_out), ptr<int32_t>(granted), ptr<int32_t>(cu_q), ptr<int32_t>(cu_k),
                        ptr<int32_t>(item_slot), ptr<int32_t>(item_pos), ptr<int64_t>(slot_map), (int)cap,
                        ptr<void>(tiles), tiles ? (int)tiles->size(0) : 0, ptr<int32_t>(status_word(dev)),
                        c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_step_tables");
}

void gemv_w4(const Tensor& x, const Tensor& w, const Tensor& scales, const OptTensor& zeros, const Tensor& out) {
  TORCH_CHECK_VALUE(w.scalar_type() == at::kByte && w.dim() == 2 && w.size(0) > 0 && w.size(1) > 0 && w.stride(1) == 1,
                    "w must be a 2-D uint8 tensor [N, K / 2] with unit column stride, got ", w.scalar_type(), " ",
                    w.sizes());
  const int64_t n = w.size(0), k = 2 * w.size(1), m = x.dim() == 2 ? x.size(0) : 0;
  as_int("w's rows", n + 15);  // in whole tiles of 16
  as_int("K", k);
  const int64_t ldw = n > 1 ? w.stride(0) : (w.size(1) + 15) / 16 * 16;
  TORCH_CHECK_VALUE(k % 32 == 0 && ldw % 16 == 0 && ldw >= w.size(1) && aligned16(w),
                    "w needs K a multiple of 32, a row stride that is a multiple of 16 bytes and 16-byte alignment, got K ",
                    k);
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kBFloat16 && scales.dim() == 2 && scales.size(0) == n &&
                        scales.size(1) > 0 && k % scales.size(1) == 0 && scales.is_contiguous(),
                    "scales must be a contiguous bf16 tensor [", n, ", K / group], got ", scales.scalar_type(), " ",
                    scales.sizes(), " for K ", k);
  const int64_t group = k / scales.size(1);
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group % 128 == 0,
                    "groups of 32, 64 or a multiple of 128 are taken, got ", group);
  TORCH_CHECK_VALUE(!zeros || (zeros->scalar_type() == at::kByte && zeros->sizes() == scales.sizes() &&
                               zeros->is_contiguous()),
                    "zeros must be a contiguous uint8 tensor ", scales.sizes());
  check_rows("x", x, 0, k);
  TORCH_CHECK_VALUE(m <= 65535, "one call takes at most 65535 token rows, got ", m);
  TORCH_CHECK_VALUE(x.size(1) == k, "x has ", x.size(1), " columns, the weights ", k);
  TORCH_CHECK_VALUE(out.scalar_type() == at::kBFloat16 && out.dim() == 2 && out.size(0) == m && out.size(1) == n &&
                        (n == 1 || out.stride(1) == 1) && (m <= 1 || out.stride(0) >= n),
                    "out must be a bf16 tensor [", m, ", ", n, "] with unit column stride, got ", out.scalar_type(), " ",
                    out.sizes());
  const auto dev = one_device(x, w, scales, zeros, out);
  const c10::cuda::CUDAGuard guard(dev);
  check(cdb_gemv_w4(ptr<void>(x), std::max(x.stride(0), k), ptr<void>(w), ldw, ptr<void>(scales), ptr<void>(zeros),
                    ptr<void>(out), std::max(out.stride(0), n), (int)m, (int)n, (int)k, (int)group, sm_count(dev),
                    ptr<int32_t>(status_word(dev)), c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_gemv_w4");
}

struct Pool {
  int layers, heads, dim;
  int64_t rows;
};

Pool check_pool(const Tensor& pool, int64_t layer) {
  TORCH_CHECK_VALUE(pool.scalar_type() == at::kBFloat16 && pool.dim() == 5 && pool.is_contiguous() &&
                        pool.size(1) == 2 && pool.size(2) >= kBlock && pool.size(3) > 0,
                    "kv_pool must be a contiguous bf16 tensor [layers, 2, rows, kv heads, head dim] of at least ", kBlock,
                    " rows, got ", pool.scalar_type(), " ", pool.sizes());
  const int64_t dim = pool.size(4);
  TORCH_CHECK_VALUE(dim == 64 || dim == 96 || dim == 128, "head dims 64, 96 and 128 are taken, got ", dim);
  TORCH_CHECK_VALUE(layer >= 0 && layer < pool.size(0), "cache_layer must be in [0, ", pool.size(0), "), got ", layer);
  TORCH_CHECK_VALUE(aligned16(pool), "kv_pool must be 16-byte aligned");
  return {as_int("layers", pool.size(0)), as_int("kv heads", pool.size(3)), (int)dim, pool.size(2)};
}

// Bytes from a 2-D tensor's first element to behind its last.
std::pair<uintptr_t, uintptr_t> extent(const Tensor& t, int64_t rows, int64_t cols) {
  const auto at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {at, at + (uintptr_t)(((rows - 1) * t.stride(0) + cols) * t.element_size())};
}

// Whether n rows of `cols` columns of two tensors of one type share memory without being the same rows.
bool partly_overlap(const Tensor& a, const Tensor& b, int64_t n, int64_t cols) {
  if (n == 0) return false;
  const bool alike = n == 1 || a.stride(0) == b.stride(0);
  const auto x = extent(a, n, cols), y = extent(b, n, cols);
  if (x.second <= y.first || y.second <= x.first || (alike && x.first == y.first)) return false;
  if (n == 1 || !alike) return true;
  // columns of one buffer
  const int64_t pitch = a.stride(0) * (int64_t)a.element_size(), width = cols * (int64_t)a.element_size();
  const int64_t off = (((int64_t)(y.first - x.first)) % pitch + pitch) % pitch;
  return off < width || pitch - off < width;
}

void qk_norm_rope_append(const Tensor& qkv, const OptTensor& q_out, const Tensor& kv_pool, int64_t cache_layer,
                         const Tensor& block_table, const Tensor& item_slot, const Tensor& item_pos,
                         const Tensor& q_weight, const Tensor& k_weight, const OptTensor& rope_cos,
                         const OptTensor& rope_sin, int64_t rope_mode, int64_t num_heads, double eps) {
  const Pool c = check_pool(kv_pool, cache_layer);
  const int64_t n = as_int("item_pos's entries", item_pos.numel());
  TORCH_CHECK_VALUE(num_heads > 0, "num_heads must be positive, got ", num_heads);
  as_int("num_heads", num_heads);
  const int64_t all = num_heads + 2 * (int64_t)c.heads;
  TORCH_CHECK_VALUE(all <= 1 << 20, "one call takes at most 2^20 heads, got ", all);
  check_rows("qkv", qkv, n, all * c.dim);
  if (q_out) {
    check_rows("q_out", *q_out, n, num_heads * c.dim);
    if (n > 0 && !(q_out->const_data_ptr() == qkv.const_data_ptr() && (n == 1 || q_out->stride(0) == qkv.stride(0)))) {
      const auto a = extent(qkv, n, all * c.dim), b = extent(*q_out, n, num_heads * c.dim);
      TORCH_CHECK_VALUE(a.second <= b.first || b.second <= a.first,
                        "q_out may be q's columns of qkv, but may not overlap qkv otherwise");
    }
  }
  check_ints("item_pos", item_pos, n);
  check_ints("item_slot", item_slot, n);
  check_table(block_table);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("q_weight", q_weight), {"k_weight", k_weight}})
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.dim() == 1 && t.size(0) == c.dim && t.is_contiguous() &&
                          aligned16(t),
                      name, " must be a contiguous 16-byte aligned bf16 tensor of ", c.dim, ", got ", t.scalar_type(), " ",
                      t.sizes());
  TORCH_CHECK_VALUE(eps >= 0 && eps <= 1e30, "eps must be finite and not negative, got ", eps);
  const int rope_rows = check_rope(rope_cos, rope_sin, rope_mode, c.dim);
  const auto dev = one_device(qkv, q_out, kv_pool, block_table, item_slot, item_pos, q_weight, k_weight, rope_cos, rope_sin);
  const c10::cuda::CUDAGuard guard(dev);
  const bool rope = rope_mode != 0;
  check(cdb_qk_norm_rope_append(
            ptr<void>(qkv), qkv.stride(0), ptr<void>(q_out), q_out ? q_out->stride(0) : 0, ptr<void>(kv_pool), c.layers,
            c.rows, (int)cache_layer, ptr<int32_t>(block_table), block_table.stride(0), (int)block_table.size(0),
            (int)block_table.size(1), ptr<int32_t>(item_slot), ptr<int32_t>(item_pos), ptr<void>(q_weight),
            ptr<void>(k_weight), (int)rope_mode, rope ? ptr<void>(rope_cos) : nullptr,
            rope ? ptr<void>(rope_sin) : nullptr, rope_rows, (float)eps, (int)n, (int)num_heads, c.heads, c.dim,
            ptr<int32_t>(status_word(dev)), c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_qk_norm_rope_append");
}

void prefix_decode_attention(const Tensor& q, const Tensor& out, const Tensor& kv_pool, int64_t cache_layer,
                             const Tensor& block_table, const Tensor& item_slot, const Tensor& item_pos,
                             const Tensor& group_start, const Tensor& prefix_len, int64_t num_heads, double scale) {
  const Pool c = check_pool(kv_pool, cache_layer);
  check_heads(num_heads, c.heads);
  check_scale(scale);
  const int64_t n = as_int("item_pos's entries", item_pos.numel());
  const int64_t groups = as_int("prefix_len's entries", prefix_len.numel());
  check_rows("q", q, n, num_heads * c.dim);
  check_rows("out", out, n, num_heads * c.dim);
  TORCH_CHECK_VALUE(!partly_overlap(q, out, n, num_heads * c.dim),
                    "out may be q's own columns, but may not overlap them otherwise");
  check_ints("item_pos", item_pos, n);
  check_ints("item_slot", item_slot, n);
  check_ints("prefix_len", prefix_len, groups);
  check_ints("group_start", group_start, groups > 0 ? groups + 1 : 0);
  check_table(block_table);
  const auto dev = one_device(q, out, kv_pool, block_table, item_slot, item_pos, group_start, prefix_len);
  const c10::cuda::CUDAGuard guard(dev);
  const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const int sms = sm_count(dev);
  const Tensor& status = status_word(dev);
  const Workspace ws =
      workspace(kPrefixDecode, dev, stream,
                cdb_prefix_decode_workspace_floats((int)n, (int)groups, (int)num_heads, c.heads, c.dim, sms), 0);
  check(cdb_prefix_decode_attention(
            ptr<void>(q), q.stride(0), ptr<void>(out), out.stride(0), ptr<void>(kv_pool), c.layers, c.rows,
            (int)cache_layer, ptr<int32_t>(block_table), block_table.stride(0), (int)block_table.size(0),
            (int)block_table.size(1), ptr<int32_t>(item_slot), ptr<int32_t>(item_pos), (int)n,
            ptr<int32_t>(group_start), ptr<int32_t>(prefix_len), (int)groups, (int)num_heads, c.heads, c.dim,
            (float)scale, sms, ptr<float>(ws.floats), ws.floats.numel(), ptr<int32_t>(status),
            stream.stream()),
        "cdb_prefix_decode_attention");
}

void sample_tokens(const Tensor& logits, const Tensor& uniform, const Tensor& temperature, const OptTensor& top_k,
                   const OptTensor& top_p, const OptTensor& min_p, const Tensor& out_ids, const OptTensor& out_logprobs) {
  const bool wide = logits.scalar_type() == at::kFloat;
  TORCH_CHECK_VALUE((wide || logits.scalar_type() == at::kBFloat16) && logits.dim() == 2 && logits.size(1) > 0,
                    "logits must be a 2-D bf16 or fp32 tensor [rows, vocabulary], got ", logits.scalar_type(), " ",
                    logits.sizes());
  const int64_t n = as_int("logits' rows", logits.size(0)), v = logits.size(1);
  TORCH_CHECK_VALUE(v <= 1 << 24, "vocabularies of up to 2^24 are taken, got ", v);
  TORCH_CHECK_VALUE((v == 1 || logits.stride(1) == 1) && (n <= 1 || logits.stride(0) >= v),
                    "logits need unit column stride and rows that do not overlap, got strides ", logits.strides());
  check_ints("uniform", uniform, n, at::kFloat);
  check_ints("temperature", temperature, n, at::kFloat);
  if (top_k) check_ints("top_k", *top_k, n);
  if (top_p) check_ints("top_p", *top_p, n, at::kFloat);
  if (min_p) check_ints("min_p", *min_p, n, at::kFloat);
  check_ints("out_ids", out_ids, n, at::kLong);
  if (out_logprobs) check_ints("out_logprobs", *out_logprobs, n, at::kFloat);
  const auto dev = one_device(logits, uniform, temperature, top_k, top_p, min_p, out_ids, out_logprobs);
  const c10::cuda::CUDAGuard guard(dev);
  check(cdb_sample_tokens(ptr<void>(logits), wide, n > 1 ? logits.stride(0) : v, (int)n, (int)v, ptr<float>(uniform),
                          ptr<float>(temperature), ptr<int32_t>(top_k), ptr<float>(top_p), ptr<float>(min_p),
                          ptr<int64_t>(out_ids), ptr<float>(out_logprobs),
                          c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "cdb_sample_tokens");
}

Tensor status(const Tensor& like) {
  const auto dev = one_device(like);
  const c10::cuda::CUDAGuard guard(dev);
  return status_word(dev);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cdb, m) {
  m.def(
      "kv8_append(Tensor qkv, Tensor(a!)? q_out, Tensor(b!) codes, Tensor(c!) scales, int cache_layer, Tensor "
      "block_table, Tensor item_slot, Tensor item_pos, Tensor? rope_cos, Tensor? rope_sin, Tensor? qk_bias, int "
      "rope_mode, int num_heads) -> ()");
  m.def("kv8_gather(Tensor codes, Tensor scales, int cache_layer, Tensor blocks, Tensor(a!) out) -> ()");
  m.def(
      "kv8_decode_attention(Tensor q, Tensor(a!) out, Tensor codes, Tensor scales, int cache_layer, Tensor block_table, "
      "Tensor item_slot, Tensor item_pos, int num_heads, float scale) -> ()");
  m.def(
      "kv8_prefill_attention(Tensor q, Tensor(a!) out, Tensor codes, Tensor scales, int cache_layer, Tensor block_table, "
      "Tensor tiles, int num_heads, float scale) -> ()");
  m.def(
      "step_tables(Tensor slots, Tensor seq_len, Tensor new_len, Tensor row_len, Tensor(a!) block_table, Tensor ring, "
      "Tensor state, Tensor(b!) row_len_out, Tensor(c!) state_out, Tensor(d!) granted, Tensor(e!) cu_seq_lens_q, "
      "Tensor(f!) cu_seq_lens_k, Tensor(g!) item_slot, Tensor(h!) item_pos, Tensor(i!) slot_map, Tensor(j!)? tiles) -> ()");
  m.def("gemv_w4(Tensor x, Tensor w, Tensor scales, Tensor? zeros, Tensor(a!) out) -> ()");
  m.def(
      "qk_norm_rope_append(Tensor qkv, Tensor(a!)? q_out, Tensor(b!) kv_pool, int cache_layer, Tensor block_table, Tensor "
      "item_slot, Tensor item_pos, Tensor q_weight, Tensor k_weight, Tensor? rope_cos, Tensor? rope_sin, int rope_mode, "
      "int num_heads, float eps) -> ()");
  m.def(
      "prefix_decode_attention(Tensor q, Tensor(a!) out, Tensor kv_pool, int cache_layer, Tensor block_table, Tensor "
      "item_slot, Tensor item_pos, Tensor group_start, Tensor prefix_len, int num_heads, float scale) -> ()");
  m.def(
      "sample_tokens(Tensor logits, Tensor uniform, Tensor temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, "
      "Tensor(a!) out_ids, Tensor(b!)? out_logprobs) -> ()");
  m.def("_status_word(Tensor like) -> Tensor");
}

// For every backend, so that CPU tensors reach the check that refuses them.
TORCH_LIBRARY_IMPL(cdb, CompositeExplicitAutograd, m) {
  m.impl("kv8_append", &kv8_append);
  m.impl("kv8_gather", &kv8_gather);
  m.impl("kv8_decode_attention", &kv8_decode_attention);
  m.impl("kv8_prefill_attention", &kv8_prefill_attention);
  m.impl("step_tables", &step_tables);
  m.impl("gemv_w4", &gemv_w4);
  m.impl("qk_norm_rope_append", &qk_norm_rope_append);
  m.impl("prefix_decode_attention", &prefix_decode_attention);
  m.impl("sample_tokens", &sample_tokens);
  m.impl("_status_word", &status);
}
