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

// A wave takes kSteps steps of a packed row, ROWS heads of Q, K or V a step: D / 16
// lanes per head, each with 8 values of its first half and the 8 that they pair with, so
// that a turn stays in the lane and every access is 16 bytes. The angles depend on the
// row and pair only: each is computed once per wave and shared through LDS, while all of
// the wave's rows are in flight. Two steps share the angles at no cost in waves: 4 sequences
// of 2048 rows, 64 heads on 8 of 128, take 62 us (5.4 TB/s, more than a large copy) with one
// step, 64 with two and 67 with four; 9 prompts of 3 to 900 rows at D = 64 13, 10 and 10.5 us.
constexpr uint32_t kSteps = 2;
template <int D>
__global__ __launch_bounds__(64) void paged_append_kernel(PagedAppendParams p) {
  constexpr int LPR = D / 16, ROWS = 64 / LPR, HALF = D / 2;
  __shared__ __attribute__((aligned(16))) float s_cos[HALF], s_sin[HALF];
  const int lane = threadIdx.x, l = lane % LPR;
  const uint32_t q_steps = (p.q_heads + ROWS - 1) / ROWS, k_steps = (p.kv_heads + ROWS - 1) / ROWS;
  const uint32_t total = q_steps + 2 * k_steps, chunks = (total + kSteps - 1) / kSteps;
  const uint32_t row = blockIdx.x / chunks, first = blockIdx.x % chunks * kSteps;
  // Step i of the wave: which heads, and this lane's.
  auto is_query = [&](int i) { return first + i < q_steps; };
  auto is_value = [&](int i) { return first + i >= q_steps + k_steps; };
  auto head_of = [&](int i) -> uint32_t {
    const uint32_t step = first + i;
    return (is_query(i) ? step : is_value(i) ? step - q_steps - k_steps : step - q_steps) * ROWS + lane / LPR;
  };
  auto mine = [&](int i) { return first + i < total && head_of(i) < (is_query(i) ? p.q_heads : p.kv_heads); };
  uint4 x[kSteps][2];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
    if (!mine(i)) continue;
    const uint16_t *src = is_query(i)   ? p.q + (int64_t)row * p.q_tok + (int64_t)head_of(i) * p.q_head
                          : is_value(i) ? p.v + (int64_t)row * p.v_tok + (int64_t)head_of(i) * p.v_head
                                        : p.k + (int64_t)row * p.k_tok + (int64_t)head_of(i) * p.k_head;
    x[i][0] = *reinterpret_cast<const uint4 *>(src + 8 * l);
    x[i][1] = *reinterpret_cast<const uint4 *>(src + HALF + 8 * l);
  }
  const uint32_t b = sequence_of_row(p.row_starts, p.batch, row, lane);
  const RowRange range = sequence_rows(p.row_starts, b, p.rows);
  if (row < range.begin || row >= range.end) return;  // no sequence has this row
  const uint32_t len = p.kv.lengths[b], behind = range.end - row;
  if (len < behind) return;  // more rows than keys: this one has no position
  const uint32_t position = len - behind, slot = position & ((1u << p.kv.page_shift) - 1);
  const uint32_t at = position >> p.kv.page_shift;  // past the table: no page
  const uint32_t page = at < p.kv.table_width ? p.kv.table[(int64_t)b * p.kv.table_seq + at] : ~0u;
  float c[8], s[8];
  if (!is_value(0)) {
#pragma unroll
    for (int a = 0; a < (HALF + 63) / 64; ++a)
      if (lane + 64 * a < HALF) turn(p, position, lane + 64 * a, D, &s_cos[lane + 64 * a], &s_sin[lane + 64 * a]);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = s_cos[8 * l + e], s[e] = s_sin[8 * l + e];
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (first + i >= total) break;
    uint16_t *dst;
    if (is_query(i))
      dst = p.q_out + (int64_t)row * p.qo_tok + (int64_t)head_of(i) * p.qo_head;
    else if (is_value(i))
      dst = p.value_pages + (int64_t)page * p.kv.v_page + (int64_t)slot * p.kv.v_pos + (int64_t)head_of(i) * p.kv.v_head;
    else
      dst = p.key_pages + (int64_t)page * p.kv.k_page + (int64_t)slot * p.kv.k_pos + (int64_t)head_of(i) * p.kv.k_head;
    uint4 y[2] = {x[i][0], x[i][1]};
    if (!is_value(i)) {
      const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
      float v[2][8];
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float f = (e & 1) ? hi_f16(w[e >> 1]) : lo_f16(w[e >> 1]);
        v[e >> 3][e & 7] = f;
        sum = fmaf(f, f, sum);
      }
      const uint16_t *weight = is_query(i) ? p.q_weight : p.k_weight;
      if (weight != nullptr) {
        sum = group_sum<LPR>(sum);
        const float scale = 1.0f / sqrtf(sum / (float)D + p.epsilon);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint4 g = *reinterpret_cast<const uint4 *>(weight + hf * HALF + 8 * l);
          const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) v[hf][e] *= scale * ((e & 1) ? hi_f16(gw[e >> 1]) : lo_f16(gw[e >> 1]));
        }
      }
      uint32_t r[2][4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        r[0][e >> 1] = pack_f16x2(v[0][e] * c[e] - v[1][e] * s[e], v[0][e + 1] * c[e + 1] - v[1][e + 1] * s[e + 1]);
        r[1][e >> 1] = pack_f16x2(v[0][e] * s[e] + v[1][e] * c[e], v[0][e + 1] * s[e + 1] + v[1][e + 1] * c[e + 1]);
      }
      y[0] = make_uint4(r[0][0], r[0][1], r[0][2], r[0][3]);
      y[1] = make_uint4(r[1][0], r[1][1], r[1][2], r[1][3]);
    }
    if (!mine(i) || (!is_query(i) && page >= p.kv.pages)) continue;  // the sequence has no page there
    *reinterpret_cast<uint4 *>(dst + 8 * l) = y[0];
    *reinterpret_cast<uint4 *>(dst + HALF + 8 * l) = y[1];
  }
}

template <int D>
hipError_t launch_d(const PagedAppendParams &p, const Launch &l) {
  constexpr uint32_t ROWS = 1024 / D;
  const uint32_t total = (p.q_heads + ROWS - 1) / ROWS + 2 * ((p.kv_heads + ROWS - 1) / ROWS);
  return dispatch(paged_append_kernel<D>, dim3(p.rows * ((total + kSteps - 1) / kSteps)), dim3(64), 0, l, p);
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
