// QK-norm, RoPE and the K/V append of packed rows into a paged cache.
//
// Per head row x of a token at position p (f32, one rounding to f16 at the store):
// x' = x / sqrt(mean(x^2) + eps) * w where there are norm weights, then the pairs
// (x'_i, x'_{i + D/2}) turned by p theta^(-2i/D). The turn is counted in whole
// revolutions in 64 bits and only its fraction goes to 32: an angle of 10^5 radians
// in f32 is off by 4e-3. Bound by bytes: every row is read and written once.
#include "kernels.hpp"
#include "paged_tile.hpp"

namespace mi {
namespace kernels {
namespace {

using namespace mi::dev;

// cos and sin of `position` theta^(-2 pair / D).
__device__ __forceinline__ void turn(const PagedAppendParams &p, uint32_t position, uint32_t pair, uint32_t head_dim,
                                     float *c, float *s) {
  const double frequency = exp2(-(double)(2 * pair) / (double)head_dim * p.log2_theta) * 0.15915494309189533577;
  const double turns = (double)position * frequency;
  sincospif(2.0f * (float)(turns - rint(turns)), s, c);
}

// One wave per (row, head): query heads, then key heads, then value heads.
template <int D>
__global__ __launch_bounds__(64) void paged_append_kernel(PagedAppendParams p) {
  const uint32_t heads = p.q_heads + 2 * p.kv_heads;
  const uint32_t row = blockIdx.x / heads, head = blockIdx.x % heads;
  const int lane = threadIdx.x;
  const uint32_t b = sequence_of_row(p.row_starts, p.batch, row, lane);
  const RowRange range = sequence_rows(p.row_starts, b, p.rows);
  if (row < range.begin || row >= range.end) return;  // no sequence has this row
  const uint32_t len = paged_length(p.kv, b), behind = range.end - row;
  if (len < behind) return;  // more rows than keys: this one has no position
  const uint32_t position = len - behind;
  const bool is_query = head < p.q_heads, is_value = head >= p.q_heads + p.kv_heads;
  const uint32_t kvh = is_value ? head - p.q_heads - p.kv_heads : head - p.q_heads;
  uint16_t *dst;
  if (is_query) {
    dst = p.q_out + (int64_t)row * p.qo_tok + (int64_t)head * p.qo_head;
  } else {
    const uint32_t page = p.kv.table[(int64_t)b * p.kv.table_seq + (position >> p.kv.page_shift)];
    if (page >= p.kv.pages) return;  // the sequence has no page there
    const uint32_t slot = position & ((1u << p.kv.page_shift) - 1);
    dst = is_value ? p.value_pages + (int64_t)page * p.kv.v_page + (int64_t)slot * p.kv.v_pos + (int64_t)kvh * p.kv.v_head
                   : p.key_pages + (int64_t)page * p.kv.k_page + (int64_t)slot * p.kv.k_pos + (int64_t)kvh * p.kv.k_head;
  }
  if (is_value) {
    const uint16_t *src = p.v + (int64_t)row * p.v_tok + (int64_t)kvh * p.v_head;
    for (int i = lane; i < D; i += 64) dst[i] = src[i];
    return;
  }
  const uint16_t *src = is_query ? p.q + (int64_t)row * p.q_tok + (int64_t)head * p.q_head
                                 : p.k + (int64_t)row * p.k_tok + (int64_t)kvh * p.k_head;
  const uint16_t *weight = is_query ? p.q_weight : p.k_weight;
  constexpr int HALF = D / 2, PAIRS = (HALF + 63) / 64;
  float x[PAIRS], y[PAIRS], sum = 0.0f;
#pragma unroll
  for (int a = 0; a < PAIRS; ++a) {
    const int pair = lane + 64 * a;
    x[a] = pair < HALF ? f16_to_f32(src[pair]) : 0.0f;
    y[a] = pair < HALF ? f16_to_f32(src[pair + HALF]) : 0.0f;
    sum += x[a] * x[a] + y[a] * y[a];
  }
  sum = group_sum<64>(sum);
  const float scale = weight != nullptr ? 1.0f / sqrtf(sum / (float)D + p.epsilon) : 1.0f;
#pragma unroll
  for (int a = 0; a < PAIRS; ++a) {
    const int pair = lane + 64 * a;
    if (pair >= HALF) continue;
    const float wx = weight != nullptr ? f16_to_f32(weight[pair]) : 1.0f;
    const float wy = weight != nullptr ? f16_to_f32(weight[pair + HALF]) : 1.0f;
    const float nx = x[a] * scale * wx, ny = y[a] * scale * wy;
    float c, s;
    turn(p, position, pair, D, &c, &s);
    dst[pair] = f32_to_f16(nx * c - ny * s);
    dst[pair + HALF] = f32_to_f16(nx * s + ny * c);
  }
}

template <int D>
hipError_t launch_d(const PagedAppendParams &p, const Launch &l) {
  const uint32_t heads = p.q_heads + 2 * p.kv_heads;
  return dispatch(paged_append_kernel<D>, dim3(p.rows * heads), dim3(64), 0, l, p);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams &p, uint32_t head_dim, const Launch &l) {
  switch (head_dim) {
    case 32: return launch_d<32>(p, l);
    case 64: return launch_d<64>(p, l);
    case 128: return launch_d<128>(p, l);
    case 256: return launch_d<256>(p, l);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace kernels
}  // namespace mi
