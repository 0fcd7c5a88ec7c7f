// 16-bit [rows][D] tiles in shared memory for the prefill attention kernels: row pitch, swizzle and
// matrix loads.
#pragma once

#include <stdint.h>

namespace cdb {
namespace prefill {

// Shared-memory row pitch of a [rows][D] 16-bit tile. D = 64/128: rows of D*2 bytes with the
// 16-byte chunk index XOR-swizzled by r % 8 (rows hold whole groups of 8 chunks). D = 96: 12
// chunks per row do not form whole groups, so rows are padded to 13 chunks (208 bytes) instead;
// the 8 rows one ldmatrix phase reads then start in distinct bank groups ((13 r + c) mod 8).
template <int D>
struct RowPitch {
  static constexpr int BYTES = (D == 96) ? 208 : D * 2;
  static constexpr bool XOR = (D != 96);
};

template <int D>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return (uint32_t)(r * RowPitch<D>::BYTES + ((RowPitch<D>::XOR ? (c ^ (r & 7)) : c) << 4));
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

}  // namespace prefill
}  // namespace cdb
