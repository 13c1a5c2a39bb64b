// What the kernels over packed rows and the paged KV cache share: which sequence a
// row belongs to, where the rows that no sequence has are read from, scans over a wave,
// direct loads into LDS and the waits for them.
#pragma once

#include "device_common.hpp"
#include "kernels.hpp"

namespace mi {
namespace dev {

// A key row of zeros (the largest head_dim). Rows of a decode tile past its last key, and
// those of a page that is not there, are read from here: a masked weight is 0, and 0
// times what a recycled page holds (infinities, NaN) would be NaN in the products.
static __device__ __attribute__((aligned(512))) uint16_t zero_row[256];

// Sequence `b`'s packed rows [begin, end) of the call's `rows`, whatever the
// offsets hold (they are device data: out-of-order ones make an empty sequence).
struct RowRange {
  uint32_t begin, end;
};
__device__ __forceinline__ RowRange sequence_rows(const uint32_t *row_starts, uint32_t b, uint32_t rows) {
  if (row_starts == nullptr) return {min(b, rows), min(b + 1, rows)};
  const uint32_t end = min(row_starts[b + 1], rows);
  return {min(row_starts[b], end), end};
}

// The last sequence that starts at or before `row` (uniform over the wave), which is
// the one that holds it if any does: sequences without rows start where the next one
// does.
__device__ __forceinline__ uint32_t sequence_of_row(const uint32_t *row_starts, uint32_t batch, uint32_t row,
                                                    int lane) {
  if (row_starts == nullptr) return min(row, batch - 1);
  uint32_t count = 0;
  for (uint32_t c0 = 1; c0 < batch; c0 += 64) {
    const uint32_t b = c0 + lane;
    count += (uint32_t)__popcll(__ballot(b < batch && row_starts[b] <= row));
  }
  return count;
}

// Keys of sequence `b`: its length, within what its table row can name.
__device__ __forceinline__ uint32_t paged_length(const kernels::PagedKv &kv, uint32_t b) {
  return min(kv.lengths[b], kv.table_width << kv.page_shift);
}

// Sum of x over the lanes up to this one (row shifts, then the rows' last lanes).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t scan64(uint32_t x) {
  x = dpp_add<0x118, 0xf>(dpp_add<0x114, 0xf>(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(x))));
  return dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(x));
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
// Sum and largest value over the 64 lanes, to every lane.
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) { return last_lane(scan64(x)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(x))));
  return last_lane(dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(x)));
}

// The parameters of a kernel of one parameter, read again: what is used only before and
// after a loop then takes none of its scalar registers (the compiler would keep every
// parameter from the first read to the last use, and spill).
template <typename Params>
__device__ __forceinline__ const Params __attribute__((address_space(4))) *params_again() {
  auto at = (const Params __attribute__((address_space(4))) *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return at;
}

__device__ __forceinline__ uint32_t divide(uint32_t x, kernels::Divisor d) {
  return (uint32_t)(((uint64_t)x * d.magic) >> d.shift);
}

// Of the eight f16 of `v`: bit 2 e where element e is an infinity or NaN and not negative, bit
// 2 e + 1 where it is a negative one; NaN has both.
__device__ __forceinline__ uint32_t not_finite_columns(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t x = w[e >> 1] >> (16 * (e & 1)) & 0xffffu, kind = (x & 0x7fffu) > 0x7c00u ? 3u : x >> 15 ? 2u : 1u;
    bits |= (x & 0x7c00u) == 0x7c00u ? kind << 2 * e : 0u;
  }
  return bits;
}

// s_waitcnt vmcnt(N), the other counters left at their maxima.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is six bits");
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0 | (N & 15) | ((N >> 4) << 14));
}

// A direct global -> LDS load of 16 bytes per lane, as load_lds16, from the uniform address
// `base` plus a byte offset per lane; an offset of kBufferEnd or more loads zeros.
constexpr uint32_t kBufferEnd = 0x80000000u;
__device__ __forceinline__ void load_lds16_buffer(const uint16_t *base, uint32_t offset, uint16_t *lds) {
  // Raw 32-bit data, no stride, no swizzle.
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(base), 0, (int)kBufferEnd, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) uint16_t *)lds, 16, (int)offset, 0, 0, 0);
}

// s_waitcnt lgkmcnt(0): the wave's LDS accesses are done.
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

}  // namespace dev
}  // namespace mi
