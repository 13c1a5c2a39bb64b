// Attention of packed rows: the new tokens of many sequences of different lengths in one
// call, over their own rows of K and V or over the pages of a cache (head_dim 32, 64,
// 128, 256).
//
// A workgroup owns 128 rows (32 per wave) of one sequence's (token, head in group) rows
// for ONE KV head, so each 64-key tile is staged into LDS once for all query heads that
// share it, and walks that sequence's keys with an online softmax:
//  - S^T = K Q^T on v_mfma_f32_32x32x16_f16, Q^T kept in registers: a lane holds 32
//    keys' scores of one row, so the softmax is lane-local (its f32 max and sum);
//  - O^T += V^T P^T on the same MFMA, P^T being the S^T accumulator rounded to f16 in
//    place (2^-12 of each weight on average, the size of the output's own rounding; the
//    row sum takes the rounded weights) and V^T read transposed from LDS
//    (ds_read_b64_tr_b16);
//  - the next tile's direct global -> LDS loads are in flight while one is computed. A
//    wave loads 16 (or 8) consecutive rows of a tile, so they lie in one page.
// Bound by the matrix instructions with the exponentials beside them for long prompts,
// by the bytes of K and V for a few rows on a long cache.
#include <type_traits>

#include "paged_tile.hpp"
#include "prefill_tile.hpp"

namespace mi {
namespace kernels {
namespace {

using namespace mi::dev;

constexpr int BN = kPrefillBlockN;  // keys per tile
constexpr int BM = kPrefillBlockM;  // rows per workgroup
// Added to every weight's exponent, so that f16 holds weights down to 2^-32 of the
// reference's (a long tail of them counts); it cancels against the row sum.
constexpr float kBias = 8.0f;
constexpr int kReadAhead = 4;       // LDS operand reads in flight ahead of the MFMAs
constexpr int kSchedMfma = 0x008, kSchedDsRead = 0x100;

__device__ __forceinline__ uint32_t row_tiles_of(RowRange r, uint32_t group) {
  return ((r.end - r.begin) * group + BM - 1) / BM;
}

// Nonzero if an f16 of `w` is infinite or NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
// `w` with such values replaced by zero.
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  uint32_t m = 0;
  if ((w & 0x7c00u) != 0x7c00u) m |= 0xffffu;
  if ((w & 0x7c000000u) != 0x7c000000u) m |= 0xffff0000u;
  return w & m;
}

template <int D, bool PAGED>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_packed_kernel(const PackedParams p) {
  constexpr int CPR = D / 8;           // 16-byte chunks per tile row
  constexpr int RPB = 512 / D;         // tile rows per 1 KB direct load
  constexpr int BPW = 16 / RPB;        // direct loads of K (and V) per wave and tile
  constexpr int DC = D / 16, DT = D / 32;
  constexpr int TILE = BN * D;
  // One array per stage, and the stage a compile-time choice, so that the compiler can
  // tell the loads into one from the reads of the other.
  __shared__ __attribute__((aligned(16))) uint16_t k_lds_a[TILE], k_lds_b[TILE];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds_a[TILE], v_lds_b[TILE];
  // s_bad[st] = ti + 1: V of the masked tile ti in stage st holds a value that is not finite.
  __shared__ uint32_t s_bad[2];
  auto k_stage = [&](int st) __attribute__((always_inline)) -> uint16_t * { return st ? k_lds_b : k_lds_a; };
  auto v_stage = [&](int st) __attribute__((always_inline)) -> uint16_t * { return st ? v_lds_b : v_lds_a; };

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const uint32_t G = p.group;

  // Workgroups go round-robin over the 8 XCDs: where the KV heads divide evenly, each
  // XCD takes whole heads, whose K and V stay in its L2.
  uint32_t kvh, rest;
  {
    const uint32_t id = blockIdx.x, H = p.kv_heads;
    if (H % 8 == 0) {
      const uint32_t xcd = id % 8, k = id / 8, per = H / 8;
      kvh = xcd * per + k % per;
      rest = k / per;
    } else {
      kvh = id % H;
      rest = id / H;
    }
  }
  // The sequence and row tile of `rest`, by the prefix sums of the sequences' tiles.
  uint32_t b = 0, tile = 0;
  {
    uint32_t before = 0;
    bool found = false;
    for (uint32_t c0 = 0; c0 < p.batch && !found; c0 += 64) {
      const uint32_t bb = c0 + lane;
      uint32_t x = bb < p.batch ? row_tiles_of(sequence_rows(p.row_starts, bb, p.rows), G) : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
      }
      const uint64_t le = __ballot(before + x <= rest);
      if (le != ~0ull) {
        const int at = __popcll(le);  // x is nondecreasing
        const uint32_t below = at == 0 ? 0 : (uint32_t)__builtin_amdgcn_readlane((int)x, at - 1);
        b = c0 + at;
        tile = rest - before - below;
        found = b < p.batch;
        break;
      }
      before += (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
    }
    if (!found) return;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const RowRange range = sequence_rows(p.row_starts, b, p.rows);
  const uint32_t tokens = range.end - range.begin;
  const uint32_t L = PAGED ? paged_length(p.kv, b) : tokens;
  const int64_t off = (int64_t)L - tokens;  // position of the first row (negative: more rows than keys)

  const uint32_t row0 = tile * BM, my_row = row0 + wave * 32 + n;
  const uint32_t my_t = my_row / G, my_g = my_row % G;
  const bool row_ok = my_t < tokens;
  const uint32_t t_first = row0 / G, t_last = min(tokens - 1, (row0 + BM - 1) / G);
  const uint32_t kmax = p.causal != 0 ? (uint32_t)max((int64_t)0, off + t_last + 1) : L;  // at most L
  const uint32_t n_tiles = (kmax + BN - 1) / BN;
  // Last key that this lane's row sees, and that the tile's first row does.
  const int64_t lim = p.causal != 0 ? off + min(my_t, tokens - 1) : (int64_t)L - 1;
  const int64_t full_lim = p.causal != 0 ? off + t_first : (int64_t)L - 1;

  // Q^T as the B operand: lane (h, n) holds Q[row n][16 c + 8 h .. + 8].
  h8_t qop[DC];
  {
    const uint16_t *qrow = p.q + (int64_t)(range.begin + min(my_t, tokens - 1)) * p.q_tok +
                           (int64_t)(kvh * G + my_g) * p.q_head + 8 * h;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      qop[c] = row_ok ? as_h8(*reinterpret_cast<const uint4 *>(qrow + 16 * c)) : as_h8(make_uint4(0, 0, 0, 0));
  }

  // Page ids of the tiles' 16-key groups: lane l holds group l of the 64 (16 tiles)
  // since tile 16 k. `absent` has a bit for each group without a page, gone_a / gone_b
  // those of the tiles in the stages.
  uint32_t ids = 0, gone_a = 0, gone_b = 0;
  uint64_t absent = 0;
  const uint32_t shift = PAGED ? p.kv.page_shift : 0, in_page = (1u << shift) - 1;
  auto load_ids = [&](uint32_t ti) {
    if constexpr (PAGED) {
      const uint32_t key = ti * BN + 16 * lane;
      ids = key < kmax ? p.kv.table[(int64_t)b * p.kv.table_seq + (key >> shift)] : 0;
      absent = __ballot(key < kmax && ids >= p.kv.pages);
    }
  };

  // Direct loads of tile ti into a stage: each wave fills 16 rows, lane L writing bytes
  // 16 L .. 16 L + 15 of a 1 KB block, so it fetches the 16 bytes that belong at that
  // swizzled position. A scalar base and loop-invariant offsets.
  uint32_t k_off[BPW], v_off[BPW];
#pragma unroll
  for (int i = 0; i < BPW; ++i) {
    const int r = i * RPB + lane / CPR, row = wave * 16 + r, pc = lane % CPR;
    k_off[i] = ((uint32_t)r * (uint32_t)p.kv.k_pos + ((pc ^ k_swizzle<D>(row)) * 8)) * 2u;
    v_off[i] = ((uint32_t)r * (uint32_t)p.kv.v_pos + ((pc ^ v_swizzle<D>(row)) * 8)) * 2u;
  }
  auto issue_tile = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    if (PAGED && (ti & 15) == 0) load_ids(ti);
    const uint32_t key = ti * BN + wave * 16;
    const char *kt, *vt;
    bool there = key < kmax;
    if constexpr (PAGED) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(4 * (ti & 15) + wave));
      there = there && page < p.kv.pages;
      (stage ? gone_b : gone_a) = (uint32_t)(absent >> (4 * (ti & 15))) & 15u;
      kt = reinterpret_cast<const char *>(p.kv.k + (int64_t)page * p.kv.k_page + (int64_t)(key & in_page) * p.kv.k_pos +
                                          (int64_t)kvh * p.kv.k_head);
      vt = reinterpret_cast<const char *>(p.kv.v + (int64_t)page * p.kv.v_page + (int64_t)(key & in_page) * p.kv.v_pos +
                                          (int64_t)kvh * p.kv.v_head);
    } else {
      kt = reinterpret_cast<const char *>(p.kv.k + (int64_t)(range.begin + key) * p.kv.k_pos + (int64_t)kvh * p.kv.k_head);
      vt = reinterpret_cast<const char *>(p.kv.v + (int64_t)(range.begin + key) * p.kv.v_pos + (int64_t)kvh * p.kv.v_head);
    }
    uint16_t *kd = k_stage(stage) + wave * 16 * D, *vd = v_stage(stage) + wave * 16 * D;
    if (there && key + 16 <= kmax) {
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        load_lds16(reinterpret_cast<const uint16_t *>(kt + k_off[i]), kd + i * 512);
        load_lds16(reinterpret_cast<const uint16_t *>(vt + v_off[i]), vd + i * 512);
      }
      return;
    }
    // Rows past the last key that any row sees, or without a page, are zeros.
    const char *zero = reinterpret_cast<const char *>(zero_row) + 16 * (lane % CPR);
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const bool ok = there && key + i * RPB + lane / CPR < kmax;
      load_lds16(reinterpret_cast<const uint16_t *>(ok ? kt + k_off[i] : zero), kd + i * 512);
      load_lds16(reinterpret_cast<const uint16_t *>(ok ? vt + v_off[i] : zero), vd + i * 512);
    }
  };
  // Tiles wholly inside the first row's window need no mask.
  const uint32_t n_full = full_lim < 0 ? 0 : (uint32_t)min((int64_t)n_tiles, (full_lim + 1) / BN);
  // A masked tile's V may hold values that some of its rows must not see and that are
  // not finite, and 0 times those is NaN: each wave looks at the 16 rows it has loaded.
  auto look = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    if (ti < n_full) return;
    const uint16_t *mine = v_stage(stage) + wave * 16 * D;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const uint4 v = *reinterpret_cast<const uint4 *>(mine + i * 512 + lane * 8);
      bad |= not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w);
    }
    if (__any(bad != 0)) s_bad[stage] = ti + 1;
  };

  float16_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;  // raw-score reference max, this half-wave's share of the row sum
  const float c2 = p.scale_log2;
  // Roles in the V^T reads (ds_read_b64_tr_b16): within each 16-lane group g, output
  // lane 4a + b, element j receives element b of the 8 bytes addressed by lane a + 4j.
  const int tr_g = lane >> 4, tr_a = lane & 3, tr_j = (lane >> 2) & 3;
  const int tr_key = 4 * (tr_g >> 1) + tr_j;
  const int tr_off = tr_key * D + 4 * (tr_a & 1);
  const int tr_chunk = 2 * (tr_g & 1) + (tr_a >> 1);

  auto step = [&](uint32_t it, auto mask_tag, auto stage_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    constexpr int ST = decltype(stage_tag)::value;
    const uint32_t j0 = it * BN;
    const uint16_t *k_lds = ST ? k_lds_b : k_lds_a;
    const uint16_t *v_lds = ST ? v_lds_b : v_lds_a;
    const uint32_t gone = ST ? gone_b : gone_a;
    // S^T[key][row]: two 32-key halves, at raised wave priority.
    __builtin_amdgcn_s_setprio(1);
    float16_t s[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mt][r] = 0.0f;
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const uint16_t *kp = k_lds + (32 * mt + n) * D + (((2 * c + h) ^ k_swizzle<D>(n)) * 8);
        s[mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(*reinterpret_cast<const uint4 *>(kp)), qop[c], s[mt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_group_barrier(kSchedDsRead, kReadAhead, 0);
#pragma unroll
    for (int k = 0; k < 2 * DC - kReadAhead; ++k) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kSchedMfma, kReadAhead, 0);
    __builtin_amdgcn_s_setprio(0);
    // Key 32 mt + 8 (r >> 2) + 4 h + (r & 3) of the tile is seen when it is at most
    // lim_rel; the lane's 4 h moves to the limit, so each compare is with a constant.
    int lim_lane = BN;
    if constexpr (MASK) {
      lim_lane = (int)max(min(lim - (int64_t)j0, (int64_t)BN), (int64_t)-1) - 4 * h;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mt][r] = 32 * mt + 8 * (r >> 2) + (r & 3) > lim_lane ? -INFINITY : s[mt][r];
    }
    if (PAGED && gone != 0) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (gone >> (2 * mt + (r >> 3)) & 1) s[mt][r] = -INFINITY;
    }
    // P = 2^(s c2 - m c2 + kBias) against the row's reference max m_run, as f16 pairs
    // in accumulator order.
    uint32_t pw[2][8];
    float psum;
    auto weights = [&](float mc) __attribute__((always_inline)) {
      float ps0 = 0.0f, ps1 = 0.0f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const uint32_t w = pack_f16x2(exp2_raw(fmaf(s[mt][r], c2, -mc)), exp2_raw(fmaf(s[mt][r + 1], c2, -mc)));
          pw[mt][r >> 1] = w;
          if (r & 2)
            ps1 = dot2(w, 0x3c003c00u, ps1);
          else
            ps0 = dot2(w, 0x3c003c00u, ps0);
        }
      psum = ps0 + ps1;
    };
    // The reference moves only when a weight leaves f16's range: the sum is then +inf
    // or NaN, as it is for a row without a reference yet (m_run = -inf).
    weights(m_run * c2 - kBias);
    if (__any(!(psum <= __FLT_MAX__))) {
      float mx = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m_run, mx);
      // A row that has seen no key yet keeps m = -inf and nothing to rescale.
      const float alpha = m_new == -INFINITY ? 1.0f : exp2_raw((m_run - m_new) * c2);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m_run = m_new;
      weights(m_run == -INFINITY ? 0.0f : m_run * c2 - kBias);
    }
    l_run += psum;
    // O^T[d][row] += V^T[d][keys] P^T[keys][row], four 16-key chunks.
    auto pv = [&](auto bad_tag) __attribute__((always_inline)) {
      constexpr bool BAD = decltype(bad_tag)::value;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int mt = c >> 1, base = (c & 1) * 4;
        const h8_t pb = as_h8(make_uint4(pw[mt][base], pw[mt][base + 1], pw[mt][base + 2], pw[mt][base + 3]));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint16_t *v0 = v_lds + 16 * c * D + tr_off + ((4 * dt + tr_chunk) ^ v_swizzle<D>(tr_key)) * 8;
          uint2 lo = read_tr16(v0), hi = read_tr16(v0 + 8 * D);
          if constexpr (BAD) {
            lo = make_uint2(finite_part(lo.x), finite_part(lo.y));
            hi = make_uint2(finite_part(hi.x), finite_part(hi.y));
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, o[dt], 0, 0, 0);
        }
      }
    };
    bool bad = false;
    if constexpr (MASK) bad = s_bad[ST] == it + 1;
    if (!bad) {
      __builtin_amdgcn_s_setprio(1);
      pv(std::false_type{});
      __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2 * kReadAhead, 1);
#pragma unroll
      for (int k = 0; k < 4 * DT - kReadAhead; ++k) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 1);
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 1);
      }
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, kReadAhead, 1);
      __builtin_amdgcn_s_setprio(0);
    } else {
      // The finite values by the products, the others added to the rows that see their
      // key (a positive weight leaves an infinity or NaN what it is).
      pv(std::true_type{});
#pragma unroll 1
      for (int key = 0; key < BN; ++key) {
        const bool seen = key - 4 * h <= lim_lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // d = 32 dt + 8 q + 4 h + e of this lane's row.
            const int chunk = (4 * dt + q) ^ v_swizzle<D>(key);
            const uint2 v = *reinterpret_cast<const uint2 *>(v_lds + key * D + chunk * 8 + 4 * h);
            const uint32_t w[2] = {v.x, v.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint16_t x = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
              if (seen && (x & 0x7c00u) == 0x7c00u) o[dt][4 * q + e] += f16_to_f32(x);
            }
          }
      }
    }
    // Tile it + 1 (issued a tile ago) has landed in this wave's part of the other stage;
    // after the barrier nobody reads this stage, which then receives tile it + 2.
    wait_vmcnt<0>();
    if (it + 1 < n_tiles) look(it + 1, ST ^ 1);
    __syncthreads();
    if (it + 2 < n_tiles) issue_tile(it + 2, ST);
  };

  if (n_tiles > 0) {
    if (tid < 2) s_bad[tid] = 0;
    __syncthreads();
    // The first tile is computed once it has landed; the second stays in flight. Loads
    // complete in issue order, so vmcnt(2 BPW) leaves only the second tile's pending. The
    // barrier is a bare s_barrier (a workgroup fence would wait for every load); each
    // wave has waited for its own part, and the memory clobber keeps LDS reads below it.
    issue_tile(0, 0);
    if (n_tiles > 1) {
      issue_tile(1, 1);
      wait_vmcnt<2 * BPW>();
    } else {
      wait_vmcnt<0>();
    }
    look(0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    uint32_t it = 0;
    for (; it + 1 < n_full; it += 2) {
      step(it, std::false_type{}, S0{});
      step(it + 1, std::false_type{}, S1{});
    }
    if (it < n_full) {
      step(it, std::false_type{}, S0{});
      ++it;
    }
    if ((it & 1) != 0 && it < n_tiles) {
      step(it, std::true_type{}, S1{});
      ++it;
    }
    for (; it + 1 < n_tiles; it += 2) {
      step(it, std::true_type{}, S0{});
      step(it + 1, std::true_type{}, S1{});
    }
    if (it < n_tiles) step(it, std::true_type{}, S0{});
  }

  const float l_total = l_run + __shfl_xor(l_run, 32, 64);
  // Normalise (a row that saw no key: 0 / 0), then store through LDS: each wave writes
  // its 32 rows as f16 into a region of the idle stages and stores them back as whole
  // 16-byte chunks, D / 8 consecutive lanes per row.
  const float inv = 1.0f / l_total;
  constexpr int RPI = 64 / CPR;  // rows per store instruction
  static_assert(2 * 32 * D <= TILE, "output staging");
  __syncthreads();  // every wave is past its last LDS operand read
  uint16_t *rows_lds = (wave < 2 ? k_lds_a : k_lds_b) + (wave & 1) * 32 * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint2 v;
      v.x = pack_f16x2(o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv);
      v.y = pack_f16x2(o[dt][4 * q + 2] * inv, o[dt][4 * q + 3] * inv);
      const int chunk = (4 * dt + q) ^ out_swizzle<D>(n);
      *reinterpret_cast<uint2 *>(rows_lds + n * D + chunk * 8 + 4 * h) = v;
    }
  __syncthreads();
  const int lane_o = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const int c_out = lane_o % CPR;
#pragma unroll
  for (int i = 0; i < 32 / RPI; ++i) {
    const int r = i * RPI + lane_o / CPR;
    const uint4 v = *reinterpret_cast<const uint4 *>(rows_lds + r * D + (c_out ^ out_swizzle<D>(r)) * 8);
    const uint32_t prow = row0 + wave * 32 + r, t = prow / G, g = prow % G;
    if (t < tokens)
      *reinterpret_cast<uint4 *>(p.out + (int64_t)(range.begin + t) * p.o_tok + (int64_t)(kvh * G + g) * p.o_head +
                                 c_out * 8) = v;
  }
}

template <int D>
hipError_t launch_d(const PackedParams &p, const Launch &l) {
  const dim3 grid(p.row_tiles * p.kv_heads);
  return p.kv.table != nullptr ? dispatch(attn_packed_kernel<D, true>, grid, dim3(256), 0, l, p)
                               : dispatch(attn_packed_kernel<D, false>, grid, dim3(256), 0, l, p);
}

}  // namespace

uint64_t packed_row_tiles(uint64_t rows, uint32_t batch, uint32_t group) {
  return rows * group / BM + (batch < rows ? batch : rows);
}

hipError_t launch_packed(const PackedParams &p, uint32_t head_dim, const Launch &l) {
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
