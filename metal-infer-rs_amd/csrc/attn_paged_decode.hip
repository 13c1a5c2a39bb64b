// Attention of one new token per sequence over its pages (head_dim 32, 64, 128, 256).
//
// Bound by the bytes of K and V, each read once per chunk of up to 16 query heads.
//  - Split: a unit is (sequence, KV head, chunk). The launch's workgroups divide the
//    (unit, 32-key tile) space of all sequences equally, as the lengths on the device
//    say, so the bytes are even whatever they are; with few keys each takes one piece
//    of one unit instead. A piece that is not its whole unit leaves its max, sum and
//    weighted values (f32), and the last of a unit's pieces to finish joins them in
//    piece order, so the result does not depend on which one that is.
//  - In a piece the waves take interleaved tiles with an online softmax each, and merge
//    through LDS.
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

// Workgroups per CU (two stages of V: 64 KB of LDS at head_dim 128, 128 KB at 256).
constexpr uint32_t per_cu(uint32_t head_dim) { return head_dim == 256 ? 1 : 2; }
// Tiles of a piece where there are few keys: one or two per wave.
constexpr uint32_t kPiece = kWaves, kPieceMost = 2 * kWaves;

// How a launch divides its work, the same in every workgroup. A position is a tile of a
// unit, or with `piece` a piece of that many tiles; each workgroup takes `seg` of them.
struct Share {
  uint32_t piece, seg, total;
};

template <int THREADS>
__device__ __forceinline__ Share share_work(const PagedDecodeParams &p, uint32_t upb, uint32_t *s_tiles,
                                            uint32_t *s_pre, uint32_t (*s_sum)[4]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int WAVES = THREADS / 64;
  uint32_t sum[4] = {0, 0, 0, 0};  // tiles, pieces of kPiece and kPieceMost, sequences longer than one
  for (uint32_t b = tid; b < p.batch; b += THREADS) {
    const uint32_t t = (paged_length(p.kv, b) + kDecodeTile - 1) / kDecodeTile;
    s_tiles[b] = t;
    sum[0] += t;
    sum[1] += (t + kPiece - 1) / kPiece;
    sum[2] += (t + kPieceMost - 1) / kPieceMost;
    sum[3] += t > kPiece;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum[i] += __shfl_xor(sum[i], d, 64);
    if (lane == 0) s_sum[wave][i] = sum[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[i] = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum[i] += s_sum[w][i];
  }
  const uint32_t W = gridDim.x;
  Share sh{0, 0, 0};
  if (sum[1] * upb <= W || sum[3] == 0)
    sh.piece = kPiece;
  else if (sum[2] * upb <= W)
    sh.piece = kPieceMost;
  sh.total = (sh.piece == 0 ? sum[0] : sh.piece == kPiece ? sum[1] : sum[2]) * upb;
  sh.seg = max((sh.total + W - 1) / W, sh.piece == 0 ? kPiece : 1u);
  // s_pre[b]: positions of the units of all sequences before b.
  uint32_t carry = 0;
  for (uint32_t c0 = 0; c0 < p.batch; c0 += THREADS) {
    const uint32_t b = c0 + tid;
    uint32_t x = b < p.batch ? s_tiles[b] : 0;
    if (sh.piece != 0) x = (x + sh.piece - 1) / sh.piece;
    x *= upb;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    __syncthreads();  // s_sum is read by every wave of the step before
    if (lane == 63) s_sum[wave][0] = x;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) x += s_sum[w][0];
      all += s_sum[w][0];
    }
    if (b < p.batch) s_pre[b + 1] = carry + x;
    carry += all;
  }
  if (tid == 0) s_pre[0] = 0;
  __syncthreads();
  return sh;
}

// The output rows of a unit from its pieces' partials, in piece order.
template <int D, int THREADS>
__device__ void join_pieces(const PagedDecodeParams &p, const float *partial, uint32_t pieces, uint32_t heads,
                            uint16_t *out) {
  constexpr uint32_t ROW = D + 2, FEW = 16;
  const size_t stride = (size_t)p.chunk * ROW;
  for (uint32_t i = threadIdx.x; i < heads * (D / 2); i += THREADS) {
    const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
    const float *row = partial + g * ROW;
    float M = -INFINITY, L = 0.0f, A0 = 0.0f, A1 = 0.0f;
    for (uint32_t s0 = 0; s0 < pieces; s0 += FEW) {
      float2 ml[FEW], a[FEW];  // one memory round trip
#pragma unroll
      for (uint32_t k = 0; k < FEW; ++k) {
        const float *part = row + min(s0 + k, pieces - 1) * stride;
        ml[k] = load_partial2(part);
        a[k] = load_partial2(part + 2 + d);
      }
      float m = M;
#pragma unroll
      for (uint32_t k = 0; k < FEW; ++k) m = s0 + k < pieces ? fmaxf(m, ml[k].x) : m;
      const float r = M == -INFINITY ? 0.0f : exp2_raw((M - m) * p.scale_log2);
      L *= r, A0 *= r, A1 *= r, M = m;
#pragma unroll
      for (uint32_t k = 0; k < FEW; ++k) {
        if (s0 + k >= pieces || ml[k].x == -INFINITY) continue;
        const float f = exp2_raw((ml[k].x - M) * p.scale_log2);
        L = fmaf(ml[k].y, f, L);
        A0 = fmaf(a[k].x, f, A0);
        A1 = fmaf(a[k].y, f, A1);
      }
    }
    *reinterpret_cast<uint32_t *>(out + g * p.o_head + d) = pack_f16x2(A0 / L, A1 / L);
  }
}

template <int D>
__global__ __launch_bounds__(kWaves * 64, per_cu(D)) void attn_decode_paged_kernel(const PagedDecodeParams p) {
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
  __shared__ uint32_t s_tiles[kPagedMaxBatch], s_pre[kPagedMaxBatch + 1], s_sum[WAVES][4], s_last;
  static_assert(WAVES * GM * D * 4 <= WAVES * STAGE * 2, "wave merge must fit a stage");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const float c2 = p.scale_log2;
  const uint32_t upb = p.kv_heads * p.head_chunks;  // units per sequence
  const uint32_t shift = p.kv.page_shift, in_page = (1u << shift) - 1;
  const Share sh = share_work<THREADS>(p, upb, s_tiles, s_pre, s_sum);
  // Sequences without a key: 0 / 0.
  for (uint32_t b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (s_tiles[b] == 0)
      for (uint32_t i = tid; i < p.q_heads * D; i += THREADS)
        p.out[(int64_t)b * p.o_seq + (int64_t)(i / D) * p.o_head + i % D] = 0x7e00;
  const uint32_t w = blockIdx.x;
  uint32_t pos = w * sh.seg;
  if (pos >= sh.total) return;
  const uint32_t end = min(pos + sh.seg, sh.total);
  // The sequence of a position: the last one whose first position is at or before it.
  auto sequence_at = [&](uint32_t at) -> uint32_t {
    uint32_t count = 0;
    for (uint32_t c0 = 1; c0 < p.batch; c0 += 64)
      count += (uint32_t)__popcll(__ballot(c0 + lane < p.batch && s_pre[c0 + lane] <= at));
    return count;
  };
  uint32_t b = sequence_at(pos);

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

  while (pos < end) {
    b = __builtin_amdgcn_readfirstlane(b);
    // This piece: tiles [t0, t1) of unit j of sequence b, and the unit's pieces.
    const uint32_t tiles = s_tiles[b], rel = pos - s_pre[b];
    uint32_t j, t0, t1, piece, pieces, slot;
    const uint32_t units_before = b * upb;
    if (sh.piece != 0) {
      pieces = (tiles + sh.piece - 1) / sh.piece;
      j = rel / pieces;
      piece = rel - j * pieces;
      t0 = piece * sh.piece;
      t1 = min(tiles, t0 + sh.piece);
      slot = pos;
    } else {
      j = rel / tiles;
      t0 = rel - j * tiles;
      t1 = min(tiles, t0 + (end - pos));
      const uint32_t start = pos - t0, first = start / sh.seg;  // the unit's first position and workgroup
      pieces = (start + tiles - 1) / sh.seg - first + 1;
      piece = w - first;
      slot = w + units_before + j;  // consecutive for a unit's pieces
    }
    const uint32_t kvh = j / p.head_chunks, hc = j % p.head_chunks;
    const uint32_t GC = min(p.chunk, p.group - hc * p.chunk);  // heads of this chunk
    const uint32_t h0 = kvh * p.group + hc * p.chunk;
    const uint32_t len = paged_length(p.kv, b);
    const uint32_t *table = p.kv.table + (int64_t)b * p.kv.table_seq;
    h8_t qop[DC];
    {
      const uint16_t *qb = p.q + (int64_t)b * p.q_seq + (int64_t)(h0 + min((uint32_t)col, GC - 1)) * p.q_head + 8 * grp;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        qop[c] = (uint32_t)col < GC ? as_h8(*reinterpret_cast<const uint4 *>(qb + 32 * c)) : as_h8(make_uint4(0, 0, 0, 0));
    }
    f4_t o[DB];
#pragma unroll
    for (int dt = 0; dt < DB; ++dt) o[dt] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;  // raw-score reference max, row sum

    // Page ids of the wave's tiles, two per tile: lane l holds the half l & 1 of the
    // wave's tile l / 2 of the 32 since `ids_from`.
    uint32_t ids = 0, ids_from = 0;
    auto load_ids = [&](uint32_t n) {
      const uint32_t key = (t0 + wave + WAVES * (n + (lane >> 1))) * KT + 16 * (lane & 1);
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
      const uint32_t base = (t0 + wave + WAVES * n) * KT;
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
      const uint32_t base = (t0 + wave + WAVES * n) * KT;
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

    // The wave's tiles are t0 + wave, t0 + wave + 4, ...
    const uint32_t mine = t1 - t0 > (uint32_t)wave ? (t1 - t0 - wave + WAVES - 1) / WAVES : 0;
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

    // The waves' rows through LDS: the unit's output, or this piece's partial.
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
    constexpr uint32_t ROW = D + 2;
    float *partial = p.partial + (size_t)slot * p.chunk * ROW;
    for (uint32_t i = tid; i < GC * (D / 2); i += THREADS) {
      const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
      float M = -INFINITY;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) M = fmaxf(M, s_m[v][g]);
      float L = 0.0f, A0 = 0.0f, A1 = 0.0f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        const float f = s_m[v][g] == -INFINITY ? 0.0f : exp2_raw((s_m[v][g] - M) * c2);
        L += s_l[v][g] * f;
        A0 += s_o[(v * GM + g) * D + d] * f;
        A1 += s_o[(v * GM + g) * D + d + 1] * f;
      }
      if (pieces == 1) {
        // No key with a page: 0 / 0.
        *reinterpret_cast<uint32_t *>(out + g * p.o_head + d) = pack_f16x2(A0 / L, A1 / L);
      } else {
        store_partial2(partial + g * ROW + 2 + d, A0, A1);
        if (d == 0) store_partial2(partial + g * ROW, M, L);
      }
    }
    if (pieces > 1) {
      wait_vmcnt<0>();
      __syncthreads();
      uint32_t *counter = p.counters + (size_t)(units_before + j) * p.counter_stride;
      if (tid == 0) {
        const bool last = arrive(counter) == pieces - 1;
        if (last) {
          acquire_partials();
          __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        s_last = last;
      }
      __syncthreads();
      if (s_last != 0) join_pieces<D, THREADS>(p, p.partial + (size_t)(slot - piece) * p.chunk * ROW, pieces, GC, out);
    }
    __syncthreads();  // the next piece's loads overwrite the stages
    pos += sh.piece != 0 ? 1 : t1 - t0;
    if (pos < end && pos >= s_pre[b + 1]) b = sequence_at(pos);
  }
}

template <int D>
hipError_t launch_d(const PagedDecodeParams &p, const Launch &l) {
  return dispatch(attn_decode_paged_kernel<D>, dim3(p.workgroups), dim3(kWaves * 64), 0, l, p);
}

}  // namespace

uint32_t paged_decode_workgroups(uint32_t compute_units, uint32_t head_dim) {
  return per_cu(head_dim) * (compute_units > 1 ? compute_units : 1);
}

hipError_t launch_paged_decode(const PagedDecodeParams &p, uint32_t head_dim, const Launch &l) {
  if (p.chunk == 0 || p.chunk > kDecodeRows || p.batch > kPagedMaxBatch) return hipErrorInvalidValue;
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
