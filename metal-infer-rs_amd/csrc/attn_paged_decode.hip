// Attention of one new token per sequence over its pages (head_dim 32, 64, 128, 256).
//
// One workgroup per (sequence, KV head, chunk of up to 16 query heads); its 4 waves
// take interleaved 32-key tiles with an online softmax and merge through LDS.
//  - S^T[key][head] = K Q^T on v_mfma_f32_16x16x32_f16: lane (g, c) loads key c's
//    halves 8 g + 32 j straight into the A operand, and holds 8 keys' scores of head c.
//  - O^T[d][head] += V^T P^T on the same MFMA: V rows land in the wave's LDS stage by
//    direct loads, in the key order of the S accumulator, and are read transposed. P
//    goes in two f16 terms (22 bits down to 2^-8 of the largest weight): one term adds
//    an error of the output's own rounding, and the MFMAs hide behind the loads.
//  - Pages hold at least 16 positions, so a half tile lies in one page: its address is
//    a scalar base (page id from the table) and an offset per lane that does not change.
#include <type_traits>

#include "decode_tile.hpp"
#include "paged_tile.hpp"

namespace mi {
namespace kernels {
namespace {

using namespace mi::dev;

constexpr int kWaves = 4;
typedef float f4_t __attribute__((ext_vector_type(4)));

template <int D>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) void attn_decode_paged_kernel(const PagedDecodeParams p) {
  constexpr int WAVES = kWaves, KT = kDecodeTile, DC = D / 32, DB = D / 16;
  constexpr int CPR = D / 8, VL = KT * CPR / 64;  // 16-byte chunks per V row, 1 KB V loads per tile
  constexpr int THREADS = WAVES * 64, STAGE = KT * D, GM = kDecodeRows;
  // Added to every weight's exponent, so that the low terms stay above f16's smallest
  // values; it cancels between the weighted sum and the row sum.
  constexpr float kBias = 6.0f;
  // One array per V stage, so that the compiler can tell the loads into one from the
  // reads of the other. After the tile loop stage a holds the waves' partial rows.
  __shared__ __attribute__((aligned(16))) uint16_t v_lds_a[WAVES * STAGE];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds_b[WAVES * STAGE];
  __shared__ float s_m[WAVES][GM], s_l[WAVES][GM];
  static_assert(WAVES * GM * D * 4 <= WAVES * STAGE * 2, "wave merge must fit a stage");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const float c2 = p.scale_log2;
  const uint32_t upb = p.kv_heads * p.head_chunks;  // units per sequence
  const uint32_t b = blockIdx.x / upb, j = blockIdx.x % upb;
  const uint32_t kvh = j / p.head_chunks, hc = j % p.head_chunks;
  const uint32_t GC = min(p.chunk, p.group - hc * p.chunk);  // heads of this chunk
  const uint32_t h0 = kvh * p.group + hc * p.chunk;
  const uint32_t len = paged_length(p.kv, b);
  const uint32_t shift = p.kv.page_shift, in_page = (1u << shift) - 1;
  const uint32_t *table = p.kv.table + (int64_t)b * p.kv.table_seq;
  const uint32_t t1 = (len + KT - 1) / KT;

  h8_t qop[DC];
  {
    const uint16_t *qb = p.q + (int64_t)b * p.q_seq + (int64_t)(h0 + min((uint32_t)col, GC - 1)) * p.q_head + 8 * grp;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      qop[c] = (uint32_t)col < GC ? as_h8(*reinterpret_cast<const uint4 *>(qb + 32 * c)) : as_h8(make_uint4(0, 0, 0, 0));
  }
  // Offsets of a lane within a half tile (bytes). V: direct-load instruction i writes
  // 1 KB of LDS rows, lane L row (64 i + L) / CPR and 16-byte chunk L % CPR.
  uint32_t v_off[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int r = (64 * i + lane) / CPR, pc = lane % CPR;
    const int chunk = 2 * ((pc >> 1) ^ decode_v_swizzle<D>(r)) + (pc & 1);
    v_off[i] = ((uint32_t)(decode_slot_key(r) & 15) * (uint32_t)p.kv.v_pos + chunk * 8) * 2u;
  }
  const uint32_t k_off = ((uint32_t)col * (uint32_t)p.kv.k_pos + 8 * grp) * 2u;
  const int mu = lane & 15, tr_row = 8 * grp + (mu >> 2);
  const int tr_base = tr_row * D + 4 * (mu & 1), tr_hi = (mu & 3) >> 1, tr_f = decode_v_swizzle<D>(tr_row);

  f4_t o[DB];
#pragma unroll
  for (int dt = 0; dt < DB; ++dt) o[dt] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m_run = -INFINITY, l_run = 0.0f;  // raw-score reference max, row sum

  // Page ids of the wave's tiles, two per tile: lane l holds the half l & 1 of the
  // wave's tile l / 2 of the 32 since `ids_from`.
  uint32_t ids = 0, ids_from = 0;
  auto load_ids = [&](uint32_t n) {
    const uint32_t key = (wave + WAVES * (n + (lane >> 1))) * KT + 16 * (lane & 1);
    ids = key < len ? table[key >> shift] : ~0u;
    ids_from = n;
  };
  // Page ids of the halves of the wave's n-th tile.
  auto page_of = [&](uint32_t n, int hf) -> uint32_t {
    return (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (n - ids_from) + hf));
  };
  auto k_base = [&](uint32_t page, uint32_t key) {
    return reinterpret_cast<const char *>(p.kv.k + (int64_t)page * p.kv.k_page + (int64_t)kvh * p.kv.k_head +
                                          (int64_t)(key & in_page) * p.kv.k_pos);
  };
  auto v_base = [&](uint32_t page, uint32_t key) {
    return reinterpret_cast<const char *>(p.kv.v + (int64_t)page * p.kv.v_page + (int64_t)kvh * p.kv.v_head +
                                          (int64_t)(key & in_page) * p.kv.v_pos);
  };
  auto issue = [&](uint32_t n, uint4 *kr, uint16_t *vst) __attribute__((always_inline)) {
    if (n - ids_from >= 32) load_ids(n);
    const uint32_t base = (wave + WAVES * n) * KT;
    uint16_t *vdst = vst + wave * STAGE;
    const uint32_t p0 = page_of(n, 0), p1 = page_of(n, 1);
    const bool whole = base + KT <= len && p0 < p.kv.pages && p1 < p.kv.pages;
    const char *zero = reinterpret_cast<const char *>(zero_row);
    const char *k0 = p0 < p.kv.pages ? k_base(p0, base) : zero, *k1 = p1 < p.kv.pages ? k_base(p1, base + 16) : zero;
    const char *v0 = p0 < p.kv.pages ? v_base(p0, base) : zero, *v1 = p1 < p.kv.pages ? v_base(p1, base + 16) : zero;
    if (whole) {
#pragma unroll
      for (int c = 0; c < DC; ++c) kr[c] = load16_nt(reinterpret_cast<const uint16_t *>(k0 + k_off + 64 * c));
#pragma unroll
      for (int c = 0; c < DC; ++c) kr[DC + c] = load16_nt(reinterpret_cast<const uint16_t *>(k1 + k_off + 64 * c));
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int r = (64 * i + lane) / CPR;
        load_lds16_nt(reinterpret_cast<const uint16_t *>(((r >> 2) & 1 ? v1 : v0) + v_off[i]), vdst + i * 512);
      }
    } else {
      // Keys past the last one, and those of a page that is not there, are rows of zeros.
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const bool there = base + 16 * hf + col < len && (hf ? p1 : p0) < p.kv.pages;
        const char *row = there ? (hf ? k1 : k0) + k_off : zero + 16 * grp;
#pragma unroll
        for (int c = 0; c < DC; ++c) kr[hf * DC + c] = load16_nt(reinterpret_cast<const uint16_t *>(row + 64 * c));
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int r = (64 * i + lane) / CPR, hf = (r >> 2) & 1;
        const bool there = base + (uint32_t)decode_slot_key(r) < len && (hf ? p1 : p0) < p.kv.pages;
        const char *row = there ? (hf ? v1 : v0) + v_off[i] : zero + 16 * (lane % CPR);
        load_lds16_nt(reinterpret_cast<const uint16_t *>(row), vdst + i * 512);
      }
    }
  };
  // `finite`: every value of the tile is (a constant of the main loop).
  auto compute = [&](uint32_t n, const uint4 *kr, const uint16_t *vst, bool finite) __attribute__((always_inline)) {
    const uint32_t base = (wave + WAVES * n) * KT;
    f4_t s[2];  // s[hf][e]: head col, key 16 hf + 4 grp + e
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      s[hf] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < DC; ++c)
        s[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(kr[hf * DC + c]), qop[c], s[hf], 0, 0, 0);
    }
    const bool there[2] = {page_of(n, 0) < p.kv.pages, page_of(n, 1) < p.kv.pages};
    if (base + KT > len || !there[0] || !there[1]) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!there[hf] || base + 16 * hf + 4 * grp + e >= len) s[hf][e] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // The reference max moves only when some head outgrows it by 2^8 (always on the
    // first tile), which keeps P at 2^14 or less.
    if (__any((mx - m_run) * c2 > 8.0f)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_new == -INFINITY ? 1.0f : exp2_raw((m_run - m_new) * c2);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DB; ++dt) o[dt] *= alpha;
      m_run = m_new;
    }
    const float mc = m_run == -INFINITY ? 0.0f : m_run * c2 - kBias;
    if (!finite) {
      float w[2][4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[hf][e] = exp2_raw(fmaf(s[hf][e], c2, -mc));
      weigh_tile<D>(o, w, vst + wave * STAGE, v_lds_b + wave * STAGE, grp, col, (int)min(len - base, (uint32_t)KT));
      return;
    }
    uint32_t pw[4], pl[4];  // P as f16 pairs in the PV operand's key order, and its low terms
    float ps = 0.0f;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float w0 = exp2_raw(fmaf(s[hf][e], c2, -mc)), w1 = exp2_raw(fmaf(s[hf][e + 1], c2, -mc));
        const uint32_t wv = pack_f16x2(w0, w1);
        pw[2 * hf + e / 2] = wv;
        pl[2 * hf + e / 2] = pack_f16x2(w0 - lo_f16(wv), w1 - hi_f16(wv));
        ps += w0 + w1;
      }
    l_run += ps;
    const h8_t ph = as_h8(make_uint4(pw[0], pw[1], pw[2], pw[3])), pll = as_h8(make_uint4(pl[0], pl[1], pl[2], pl[3]));
    const uint16_t *vw = vst + wave * STAGE;
#pragma unroll
    for (int dt = 0; dt < DB; ++dt) {
      const uint16_t *a0 = vw + tr_base + (2 * (dt ^ tr_f) + tr_hi) * 8;
      const uint2 lo = read_tr16(a0), hi = read_tr16(a0 + 4 * D);
      const h8_t va = as_h8(make_uint4(lo.x, lo.y, hi.x, hi.y));
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pll, o[dt], 0, 0, 0);
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph, o[dt], 0, 0, 0);
    }
  };

  // The wave's tiles are wave, wave + 4, ...: tile n of them is wave + 4 n.
  const uint32_t mine = t1 > (uint32_t)wave ? (t1 - wave + WAVES - 1) / WAVES : 0;
  uint4 kra[2 * DC], krb[2 * DC];
  if (mine > 0) {
    load_ids(0);
    issue(0, kra, v_lds_a);
  }
  for (uint32_t n = 0; n < mine; n += 2) {
    // compute() reads its tile's ids, so the ids move on only after both tiles.
    if (n + 1 < mine) issue(n + 1, krb, v_lds_b);
    compute(n, kra, v_lds_a, true);
    if (n + 1 >= mine) break;
    if (n + 2 < mine && n + 2 - ids_from < 32) {
      issue(n + 2, kra, v_lds_a);
      compute(n + 1, krb, v_lds_b, true);
    } else {
      compute(n + 1, krb, v_lds_b, true);
      if (n + 2 < mine) issue(n + 2, kra, v_lds_a);
    }
  }
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  // An infinite or NaN value times a low term of zero is NaN in the products above. If
  // any accumulator is not finite, the wave takes its tiles again, those that hold such
  // a value on the vector units with whole f32 weights.
  float bad = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DB; ++dt) bad += (o[dt][0] + o[dt][1] + o[dt][2] + o[dt][3]) * 0.0f;
  if (__any(!(bad == 0.0f))) {
    const float l_sum = l_run;
#pragma unroll
    for (int dt = 0; dt < DB; ++dt) o[dt] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (uint32_t n = 0; n < mine; ++n) {
      if (n % 32 == 0) load_ids(n);
      issue(n, kra, v_lds_a);
      wait_vmcnt<0>();
      compute(n, kra, v_lds_a, !any_not_finite<2 * STAGE>(v_lds_a + wave * STAGE, lane));
    }
    l_run = l_sum;
  }

  __syncthreads();
  float *s_o = reinterpret_cast<float *>(v_lds_a);  // [WAVES][GM][D]
  if ((uint32_t)col < GC) {
    if (grp == 0) {
      s_m[wave][col] = m_run;
      s_l[wave][col] = l_run;
    }
#pragma unroll
    for (int dt = 0; dt < DB; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_o[(wave * GM + col) * D + 16 * dt + 4 * grp + e] = o[dt][e];
  }
  __syncthreads();
  uint16_t *out = p.out + (int64_t)b * p.o_seq + (int64_t)h0 * p.o_head;
  for (int idx = tid; idx < (int)GC * D; idx += THREADS) {
    const int g = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, s_m[w][g]);
    float L = 0.0f, A = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = s_m[w][g] == -INFINITY ? 0.0f : exp2_raw((s_m[w][g] - M) * c2);
      L += s_l[w][g] * f;
      A += s_o[(w * GM + g) * D + d] * f;
    }
    out[g * p.o_head + d] = f32_to_f16(A / L);  // no key: 0 / 0
  }
}

template <int D>
hipError_t launch_d(const PagedDecodeParams &p, const Launch &l) {
  return dispatch(attn_decode_paged_kernel<D>, dim3(p.batch * p.kv_heads * p.head_chunks), dim3(kWaves * 64), 0, l, p);
}

}  // namespace

hipError_t launch_paged_decode(const PagedDecodeParams &p, uint32_t head_dim, const Launch &l) {
  if (p.chunk == 0 || p.chunk > kDecodeRows) return hipErrorInvalidValue;
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
