// Attention of one new token per sequence over its pages (head_dim 32, 64, 128, 256).
//
// Bound by the bytes of K and V, each read once per chunk of up to 16 query heads.
//  - Split: a unit is (sequence, KV head, chunk). Where pieces of one length divide all
//    units about evenly over the workgroups, each workgroup takes one piece and its waves,
//    on interleaved tiles, merge through LDS. Many units of about equal length are a wave's
//    each. Else every wave takes an equal share of the (unit, 32-key tile) space of all
//    sequences, as the lengths on the device say, and goes through it by itself with an
//    online softmax: no barriers, and while one wave ends a part the others keep loading.
//  - A part that is not its whole unit leaves its max, sum and weighted values (f32), and
//    the last of a unit's parts to finish joins them in order, so the result does not
//    depend on which one that is.
//  - S^T[key][head] = K Q^T on v_mfma_f32_16x16x32_f16: lane (g, c) loads key c's
//    halves 8 g + 32 j straight into the A operand, and holds 8 keys' scores of head c.
//  - O^T[d][head] += V^T P^T on the same MFMA: V rows land in the wave's LDS stage by
//    direct loads, in the key order of the S accumulator, and are read transposed. P
//    goes in two f16 terms (22 bits and more down to 2^-14 of the largest weight): one
//    term adds an error of the output's own rounding, and the MFMAs hide behind the loads.
//  - One tile of K (registers) and V (LDS) per wave: the next K is loaded once the scores
//    have taken this one, the next V after the products, and the CU's other waves cover
//    what is left of the latency. A second stage would halve the waves and double a loop
//    whose instructions a short call fetches for the first time.
//  - Pages hold at least 16 positions, so a half tile lies in one page: its address is
//    a scalar base (page id from the table) and an offset per lane that does not change.
#include "decode_tile.hpp"
#include "paged_tile.hpp"

namespace mi {
namespace kernels {
namespace {

using namespace mi::dev;

constexpr int kWaves = kPagedWaves;
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kPerCu = 2;  // workgroups per CU, by the registers of a wave at head_dim 256
// Fewest tiles of a workgroup's piece (one per wave) and of a wave's share.
constexpr uint32_t kPiece = kWaves, kShare = 2;
// Pieces may be longer than an even share by this many eighths; more than twice kJoin of a
// unit's are joined in steps of kJoin.
constexpr uint32_t kUneven = 2, kJoin = 16;
constexpr uint32_t kJoinTiles = 12;  // tiles that take as long as shares' partials and joins
// The least weight of a part in a join, and the least rescaling factor: nothing beside finite
// sums, but not 0, so that an infinity far below the other keys stays one.
constexpr float kSmallest = 0x1p-126f;

// Two f16 that are not negative, or f16's smallest value where one is zero.
__device__ __forceinline__ uint32_t above_zero(uint32_t w) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, w), u16x2_t{1, 1}));
}
// The two values of a pair over the row's sum: of a row without a weight above zero 0 / 0.
__device__ __forceinline__ uint32_t over_sum(float a, float b, float sum) {
  return sum == 0.0f ? 0x7e007e00u : pack_f16x2(a / sum, b / sum);
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), lane));
}
// The largest value and the sum of lanes 0 to 31, to every lane.
__device__ __forceinline__ float max32(float x) {
  x = fmaxf(x, dpp_f32<kDppQuadXor1>(x));
  x = fmaxf(x, dpp_f32<kDppQuadXor2>(x));
  x = fmaxf(x, dpp_f32<kDppRowRor4>(x));
  x = fmaxf(x, dpp_f32<kDppRowRor8>(x));
  return fmaxf(lane_value(x, 0), lane_value(x, 16));
}
__device__ __forceinline__ float sum32(float x) {
  x = row16_sum(x);
  return lane_value(x, 0) + lane_value(x, 16);
}

// How a launch divides its work, the same in every wave. With `piece` a position is a
// piece of that many tiles of a unit, for a workgroup, which takes one at most; else it is
// a tile, or with `whole` a unit, for a wave, which takes `seg` of them. s_tiles[b] gets the
// sequences' tiles, s_pre[b] the positions of all units before b's. Every wave computes all
// of it and reads back what it wrote itself, so no barrier is needed (the waves write the
// same values).
struct Share {
  uint32_t piece, seg, total;
  bool whole;
};
__device__ __forceinline__ Share share_work(const PagedDecodeParams &p, uint32_t upb, uint32_t *s_tiles,
                                            uint32_t *s_pre, int lane) {
  uint32_t tiles = 0, few = 0, used = 0, longest = 0;  // tiles, pieces of kPiece, sequences with a key
  for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
    const uint32_t b = c0 + lane;
    const uint32_t t = b < p.batch ? (paged_length(p.kv, b) + kDecodeTile - 1) / kDecodeTile : 0;
    if (b < p.batch) s_tiles[b] = t;
    tiles += t;
    few += (t + kPiece - 1) / kPiece;
    used += (uint32_t)__popcll(__ballot(t != 0));
    longest = max(longest, t);
  }
  tiles = wave_sum(tiles), few = wave_sum(few), longest = wave_max(longest);
  const uint32_t W = gridDim.x;
  Share sh{0, 0, tiles * upb, false};
  if (few * upb <= W) {
    sh.piece = kPiece, sh.total = few * upb;
  } else if (const uint32_t units = used * upb, waves = W * kWaves;
             longest <= kPiece ||
             (2 * units >= waves && (units + waves - 1) / waves * longest <= tiles * upb / waves + kJoinTiles)) {
    // More units than workgroups, of a piece at most: a wave each (808 of one tile, D = 128:
    // 7.5 us, by workgroups 11.7). The same where that keeps half of the waves busy and the
    // longest is not far from an even share (1024 of 400 to 511 keys: 48 us, in shares 60;
    // 512 of 300 to 400 at D = 256 59 and 42).
    sh.whole = true, sh.total = units;
  } else {
    // The smallest pieces that give each workgroup one at most, if they are near an even
    // share: a workgroup's four waves on one piece need no joins but that piece's, but the
    // longest piece sets the time. 32 equal sequences of 4096 keys (8 KV heads of 128) take 89
    // us so and 93 by shares of waves; 32 of 500 to 8000 keys 116 and 103.
    const uint32_t even = (tiles * upb + W - 1) / W, most = used * upb > W ? 0 : even + even * kUneven / 8;
    for (uint32_t piece = even; piece <= most; piece += (piece + 7) / 8) {
      uint32_t pieces = 0;
      for (uint32_t c0 = 0; c0 < p.batch; c0 += 64)
        if (c0 + lane < p.batch) pieces += (s_tiles[c0 + lane] + piece - 1) / piece;
      sh.total = last_lane(scan64(pieces)) * upb;
      if (sh.total <= W) {
        sh.piece = piece;
        break;
      }
    }
    if (sh.piece == 0) sh.total = tiles * upb;
  }
  const uint32_t takers = sh.piece != 0 ? W : W * kWaves;
  sh.seg = max((sh.total + takers - 1) / takers, sh.piece != 0 || sh.whole ? 1u : kShare);
  uint32_t carry = 0;
  for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
    const uint32_t b = c0 + lane;
    uint32_t x = b < p.batch ? s_tiles[b] : 0;
    if (sh.whole) x = min(x, 1u);
    if (sh.piece != 0) x = (x + sh.piece - 1) / sh.piece;
    x = scan64(x * upb);
    if (b < p.batch) s_pre[b + 1] = carry + x;
    carry += last_lane(x);
  }
  if (lane == 0) s_pre[0] = 0;
  return sh;
}

// One partial from several (row_stride floats apart), in order: to `out` as the unit's
// rows, or in place of the first one (out null). Of every `step` blocks of value pairs
// this wave takes the `first`; a block is of whole heads, so no other wave reads what this
// one writes. 32 parts at a time: the weights of the block's heads (a lane per part; kept
// in 2 KB of the wave's own LDS) and the first parts' values are one round trip to
// memory, the other parts' values the next ones.
template <int D>
__device__ __forceinline__ void join_parts(float *partial, size_t row_stride, uint32_t parts, uint32_t heads,
                                           float scale_log2, uint16_t *out, int64_t o_head, uint32_t first,
                                           uint32_t step, float *s_f, int lane) {
  constexpr uint32_t ROW = D + 2, MOST = 32, KU = 2, PU = 8;
  constexpr uint32_t BLOCK = 64 * KU, HEADS = BLOCK / (D / 2), FROW = MOST + 2;
  static_assert(HEADS * FROW * 4 <= 2048 && BLOCK % (D / 2) == 0, "a block is of whole heads");
  const uint32_t pairs = heads * (D / 2);
  for (uint32_t i0 = first * BLOCK; i0 < pairs; i0 += step * BLOCK) {
    const uint32_t g0 = i0 / (D / 2);
    uint32_t at[KU], hd[KU];  // this lane's pairs: offset in a partial, head within the block
    float2 A[KU];
#pragma unroll
    for (uint32_t u = 0; u < KU; ++u) {
      const uint32_t i = min(i0 + 64 * u + lane, pairs - 1), g = i / (D / 2);
      at[u] = g * ROW + 2 + i % (D / 2) * 2;
      hd[u] = g - g0;
      A[u] = make_float2(0.0f, 0.0f);
    }
    float M[HEADS], L[HEADS];
#pragma unroll
    for (uint32_t h = 0; h < HEADS; ++h) M[h] = -INFINITY, L[h] = 0.0f;
    for (uint32_t s0 = 0; s0 < parts; s0 += MOST) {
      const uint32_t n = min(MOST, parts - s0);
      const float *base = partial + (size_t)s0 * row_stride;
      float2 ml[HEADS], a[KU][PU];
#pragma unroll
      for (uint32_t h = 0; h < HEADS; ++h)
        ml[h] = load_partial2(base + min((uint32_t)lane, n - 1) * row_stride + min(g0 + h, heads - 1) * ROW);
      auto load_values = [&](uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t k = 0; k < PU; ++k)
#pragma unroll
          for (uint32_t u = 0; u < KU; ++u) a[u][k] = load_partial2(base + min(k0 + k, n - 1) * row_stride + at[u]);
      };
      load_values(0);
#pragma unroll
      for (uint32_t h = 0; h < HEADS; ++h) {
        const float m = fmaxf(M[h], max32((uint32_t)lane < n ? ml[h].x : -INFINITY));
        // A part without a maximum has a sum of 0 (no key with a page) or of NaN (every score
        // is), which any weight above zero keeps.
        const float f = (uint32_t)lane >= n ? 0.0f : fmaxf(exp2_raw((ml[h].x - m) * scale_log2), kSmallest);
        const float r = fmaxf(exp2_raw((M[h] - m) * scale_log2), kSmallest);
        M[h] = m;
        L[h] = fmaf(L[h], r, sum32(f != 0.0f ? ml[h].y * f : 0.0f));
        if ((uint32_t)lane < MOST) s_f[h * FROW + lane] = f;
        if (lane == 0) s_f[h * FROW + MOST] = r, s_f[h * FROW + MOST + 1] = L[h];
      }
#pragma unroll
      for (uint32_t u = 0; u < KU; ++u) {
        const float r = s_f[hd[u] * FROW + MOST];
        A[u].x *= r, A[u].y *= r;
      }
      for (uint32_t k0 = 0;;) {
#pragma unroll
        for (uint32_t k = 0; k < PU; ++k)
#pragma unroll
          for (uint32_t u = 0; u < KU; ++u) {
            const float f = k0 + k < n ? s_f[hd[u] * FROW + k0 + k] : 0.0f;
            A[u].x = f != 0.0f ? fmaf(a[u][k].x, f, A[u].x) : A[u].x;
            A[u].y = f != 0.0f ? fmaf(a[u][k].y, f, A[u].y) : A[u].y;
          }
        k0 += PU;
        if (k0 >= n) break;
        load_values(k0);
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < KU; ++u) {
      const uint32_t i = i0 + 64 * u + lane;
      const float sum = s_f[hd[u] * FROW + MOST + 1];
      if (i >= pairs) continue;
      if (out != nullptr)
        *reinterpret_cast<uint32_t *>(out + i / (D / 2) * o_head + i % (D / 2) * 2) = over_sum(A[u].x, A[u].y, sum);
      else
        store_partial2(partial + at[u], A[u].x, A[u].y);
    }
    if (out == nullptr && lane == 0)
#pragma unroll
      for (uint32_t h = 0; h < HEADS; ++h)
        if (g0 + h < heads) store_partial2(partial + (g0 + h) * ROW, M[h], L[h]);
  }
}

// Whether this part, whose partial has been written, is the last of `parts` to finish.
__device__ __forceinline__ bool finished_last(uint32_t *counter, uint32_t parts) {
  if (arrive(counter) != parts - 1) return false;
  acquire_partials();
  __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

// A unit that the wave (or the workgroup) was the last to finish a piece of.
struct Unit {
  uint32_t b, j, slot, pieces;
};

template <int D>
__global__ __launch_bounds__(kWaves * 64, kPerCu) void attn_decode_paged_kernel(const PagedDecodeParams p) {
  constexpr int WAVES = kWaves, KT = kDecodeTile, DC = D / 32, DB = D / 16;
  constexpr int CPR = D / 8, VL = KT * CPR / 64;  // 16-byte chunks per V row, 1 KB V loads per tile
  constexpr int THREADS = WAVES * 64, STAGE = KT * D, GM = kDecodeRows;
  constexpr uint32_t HELD = 32, ROW = D + 2;  // tiles whose page ids a wave holds; floats of a partial's head
  // Added to every weight's exponent, so that the low terms stay above f16's smallest
  // values; it cancels between the weighted sum and the row sum. The high terms round
  // towards zero, so that the low ones are not negative either, and a term of 0 becomes
  // f16's smallest value (2^-37 of the largest weight): 0 times an infinity that the row
  // sees would be NaN.
  constexpr float kBias = 13.0f, kGrow = 2.0f;
  // A stage of V per wave; the waves' rows once a piece's tiles are done.
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[WAVES * STAGE];
  __shared__ float s_m[WAVES][GM], s_l[WAVES][GM];
  __shared__ uint32_t s_tiles[kPagedMaxBatch], s_pre[kPagedMaxBatch + 1], s_last;
  __shared__ Unit s_unit[WAVES][2];
  static_assert(WAVES * GM * D * 4 <= WAVES * STAGE * 2, "the rows must fit the stages");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const float c2 = p.scale_log2;
  const uint32_t upb = p.kv_heads * p.head_chunks;  // units per sequence
  const uint32_t shift = p.kv.page_shift, in_page = (1u << shift) - 1;
  const Share sh = share_work(p, upb, s_tiles, s_pre, lane);
  // Sequences without a key: 0 / 0.
  for (uint32_t b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (s_tiles[b] == 0)
      for (uint32_t i = tid; i < p.q_heads * D; i += THREADS)
        p.out[(int64_t)b * p.o_seq + (int64_t)(i / D) * p.o_head + i % D] = 0x7e00;
  const bool together = sh.piece != 0;  // the workgroup's waves merge their rows
  const uint32_t w = together ? blockIdx.x : blockIdx.x * WAVES + wave;
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
  uint32_t b = sequence_at(pos), done = 0, split = 0;  // entries of s_unit; whether the piece is of a split unit

  // Offsets of a lane within a half tile (bytes), and its keys there. V: direct-load
  // instruction i writes 1 KB of LDS rows, lane L row (64 i + L) / CPR and 16-byte chunk
  // L % CPR.
  const uint32_t k_row = (uint32_t)p.kv.k_pos * 2, v_row = (uint32_t)p.kv.v_pos * 2;
  const uint32_t k_off = col * k_row + 16 * grp;
  uint32_t v_off[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int r = (64 * i + lane) / CPR, pc = lane % CPR;
    const int chunk = 2 * ((pc >> 1) ^ decode_v_swizzle<D>(r)) + (pc & 1);
    v_off[i] = (uint32_t)(decode_slot_key(r) & 15) * v_row + chunk * 16;
  }
  const int mu = lane & 15, tr_row = 8 * grp + (mu >> 2);
  const int tr_base = tr_row * D + 4 * (mu & 1), tr_hi = (mu & 3) >> 1, tr_f = decode_v_swizzle<D>(tr_row);
  uint16_t *stage = v_lds + wave * STAGE;
  const char *zero = reinterpret_cast<const char *>(zero_row);

  // Of a CU's two workgroups the older one's waves are served first and would end a fifth
  // earlier, leaving the other half of the loads to the tail. The younger's waves go first for
  // the first half of their tiles (32 sequences of 1024 to 8192 keys: 112 -> 108.5 us).
  uint32_t ahead = blockIdx.x >= gridDim.x / 2 ? (together ? (sh.piece + WAVES - 1) / WAVES : sh.seg) / 2 : 0;
  if (ahead != 0) __builtin_amdgcn_s_setprio(1);
  while (pos < end) {
    b = __builtin_amdgcn_readfirstlane(b);
    // This piece: tiles [t0, t1) of unit j of sequence b, and the unit's pieces.
    const uint32_t tiles = s_tiles[b], rel = pos - s_pre[b];
    uint32_t j, t0, t1, piece, pieces, slot;  // slot: consecutive for a unit's pieces
    if (together) {
      pieces = (tiles + sh.piece - 1) / sh.piece;
      j = rel / pieces;
      piece = rel - j * pieces;
      t0 = piece * sh.piece;
      t1 = min(tiles, t0 + sh.piece);
      slot = pos;
    } else if (sh.whole) {
      j = rel, t0 = 0, t1 = tiles, piece = 0, pieces = 1, slot = 0;
    } else {
      j = rel / tiles;
      t0 = rel - j * tiles;
      t1 = min(tiles, t0 + (end - pos));
      const uint32_t start = pos - t0, first = start / sh.seg;  // the unit's first position and wave
      pieces = (start + tiles - 1) / sh.seg - first + 1;
      piece = w - first;
      slot = w + b * upb + j;
    }
    const uint32_t kvh = j / p.head_chunks, hc = j % p.head_chunks;
    const uint32_t GC = min(p.chunk, p.group - hc * p.chunk);  // heads of this chunk
    const uint32_t h0 = kvh * p.group + hc * p.chunk;
    const uint32_t len = paged_length(p.kv, b);
    const uint32_t *table = p.kv.table + (int64_t)b * p.kv.table_seq;
    // The wave's tiles are t0 + from, t0 + from + by, ...
    const uint32_t from = together ? wave : 0, by = together ? WAVES : 1;
    const uint32_t mine = t1 - t0 > from ? (t1 - t0 - from + by - 1) / by : 0;

    // Page ids of the wave's tiles, two per tile: lane l holds the half l & 1 of the
    // wave's tile l / 2 of the HELD since `ids_from`.
    uint32_t ids = 0, ids_from = 0;
    auto load_ids = [&](uint32_t n) {
      const uint32_t key = (t0 + from + by * (n + (lane >> 1))) * KT + 16 * (lane & 1);
      ids = key < len ? table[key >> shift] : ~0u;
      ids_from = n;
    };
    load_ids(0);
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

    const char *k_head = reinterpret_cast<const char *>(p.kv.k + (int64_t)kvh * p.kv.k_head);
    const char *v_head = reinterpret_cast<const char *>(p.kv.v + (int64_t)kvh * p.kv.v_head);
    // The loads of the wave's n-th tile, which start at key `base`: `left` is its keys
    // (none past the last tile: every pass issues as many loads, so that a wait leaves the
    // later ones in flight), in0 / in1 whether its halves have pages. Keys past the last
    // one, and those of a page that is not there, are rows of zeros.
    uint32_t page0 = 0, page1 = 0, left = 0;
    bool in0 = false, in1 = false;
    uint4 kr[2 * DC];
    auto base_of = [&](uint32_t n) { return (t0 + from + by * n) * KT; };
    auto load_k = [&](uint32_t n) __attribute__((always_inline)) {
      if (n - ids_from >= HELD) load_ids(n);
      const uint32_t base = base_of(n);
      left = n < mine ? min(len - base, (uint32_t)KT) : 0;
      page0 = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (n - ids_from)));
      page1 = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (n - ids_from) + 1));
      in0 = page0 < p.kv.pages, in1 = page1 < p.kv.pages;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const char *at = k_head + (int64_t)(hf ? page1 : page0) * (p.kv.k_page * 2) + ((base + 16 * hf) & in_page) * k_row;
        const char *row = 16 * hf + (uint32_t)col < left && (hf ? in1 : in0) ? at + k_off : zero + 16 * grp;
#pragma unroll
        for (int c = 0; c < DC; ++c) kr[hf * DC + c] = load16_nt(reinterpret_cast<const uint16_t *>(row + 64 * c));
      }
    };
    auto load_v = [&](uint32_t n) __attribute__((always_inline)) {
      // The stage's readers are done: a direct load that hits in the cache could land
      // before an LDS read that was issued ahead of it.
      wait_lds();
      const uint32_t base = base_of(n);
      const char *v0 = v_head + (int64_t)page0 * (p.kv.v_page * 2) + (base & in_page) * v_row;
      const char *v1 = v_head + (int64_t)page1 * (p.kv.v_page * 2) + ((base + 16) & in_page) * v_row;
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int r = (64 * i + lane) / CPR, hf = (r >> 2) & 1;
        const bool ok = (uint32_t)decode_slot_key(r) < left && (hf ? in1 : in0);
        const char *row = ok ? (hf ? v1 : v0) + v_off[i] : zero + 16 * (lane % CPR);
        load_lds16_nt(reinterpret_cast<const uint16_t *>(row), stage + i * 512);
      }
    };

    if (mine > 0) {
      load_k(0);
      load_v(0);
    }
    for (uint32_t n = 0; n < mine; ++n) {
      if (ahead != 0 && --ahead == 0) __builtin_amdgcn_s_setprio(0);
      f4_t s[2];  // s[hf][e]: head col, key 16 hf + 4 grp + e
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        s[hf] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < DC; ++c)
          s[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(kr[hf * DC + c]), qop[c], s[hf], 0, 0, 0);
      }
      if (left < KT || !in0 || !in1) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(hf ? in1 : in0) || (uint32_t)(16 * hf + 4 * grp + e) >= left) s[hf][e] = -INFINITY;
      }
      load_k(n + 1);
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      // The reference max moves only when some head outgrows it by 2^kGrow (always on
      // the first tile), which keeps P at 2^15 or less.
      if (__any((mx - m_run) * c2 > kGrow)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -INFINITY ? 1.0f : fmaxf(exp2_raw((m_run - m_new) * c2), kSmallest);
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DB; ++dt) o[dt] *= alpha;
        m_run = m_new;
      }
      const float mc = m_run == -INFINITY ? 0.0f : m_run * c2 - kBias;
      uint32_t pw[4], pl[4];  // P as f16 pairs in the PV operand's key order, and its low terms
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float w0 = exp2_raw(fmaf(s[hf][e], c2, -mc)), w1 = exp2_raw(fmaf(s[hf][e + 1], c2, -mc));
          const uint32_t wv = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(w0, w1));
          pw[2 * hf + e / 2] = above_zero(wv);
          pl[2 * hf + e / 2] = above_zero(pack_f16x2(w0 - lo_f16(wv), w1 - hi_f16(wv)));
          l_run += w0 + w1;
        }
      const h8_t hi_p = as_h8(make_uint4(pw[0], pw[1], pw[2], pw[3]));
      const h8_t lo_p = as_h8(make_uint4(pl[0], pl[1], pl[2], pl[3]));
      // This tile's V has landed; of the loads since, only the next K's are in flight.
      wait_vmcnt<2 * DC>();
#pragma unroll
      for (int dt = 0; dt < DB; ++dt) {
        const uint16_t *a0 = stage + tr_base + (2 * (dt ^ tr_f) + tr_hi) * 8;
        const uint2 lo = read_tr16(a0), hi = read_tr16(a0 + 4 * D);
        const h8_t va = as_h8(make_uint4(lo.x, lo.y, hi.x, hi.y));
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, lo_p, o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, hi_p, o[dt], 0, 0, 0);
      }
      load_v(n + 1);
    }
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    wait_vmcnt<0>();  // the zeros behind the last tile have landed too

    const auto e = params_again<PagedDecodeParams>();
    const int64_t o_head = e->o_head;
    uint16_t *out = e->out + (int64_t)b * e->o_seq + (int64_t)h0 * o_head;
    float *partial = e->partial + (size_t)slot * (e->chunk * ROW);
    const Unit unit{b, j, slot - piece, pieces};
    // The wave's rows through its stage, so that a store's lanes are neighbours.
    float *rows = reinterpret_cast<float *>(stage);  // [GM][D]
    if ((uint32_t)col < GC) {
      if (grp == 0) {
        s_m[wave][col] = m_run;
        s_l[wave][col] = l_run;
      }
#pragma unroll
      for (int dt = 0; dt < DB; ++dt) *reinterpret_cast<f4_t *>(rows + col * D + 16 * dt + 4 * grp) = o[dt];
    }
    if (!together) {
      wait_lds();  // the reads are of other lanes' stores
      for (uint32_t i = lane; i < GC * (D / 2); i += 64) {
        const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
        const float2 v = *reinterpret_cast<const float2 *>(rows + 2 * i);
        const float l = s_l[wave][g];
        if (pieces == 1) {
          *reinterpret_cast<uint32_t *>(out + g * o_head + d) = over_sum(v.x, v.y, l);
        } else {
          store_partial2(partial + g * ROW + 2 + d, v.x, v.y);
          if (d == 0) store_partial2(partial + g * ROW, s_m[wave][g], l);
        }
      }
      if (pieces > 1) {
        wait_vmcnt<0>();
        uint32_t last = 0;
        if (lane == 0) last = finished_last(e->counters + (size_t)(b * upb + j) * e->counter_stride, pieces);
        if (__builtin_amdgcn_readfirstlane(last) != 0) s_unit[wave][done++] = unit;
      }
    } else {
      // The waves' rows: the unit's output, or this piece's partial.
      __syncthreads();
      const float *s_o = reinterpret_cast<const float *>(v_lds);  // [WAVES][GM][D]
      for (uint32_t i = tid; i < GC * (D / 2); i += THREADS) {
        const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) M = fmaxf(M, s_m[v][g]);
        float L = 0.0f, A0 = 0.0f, A1 = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
          const float f = fmaxf(exp2_raw((s_m[v][g] - M) * c2), kSmallest);  // as in a join
          const float2 x = *reinterpret_cast<const float2 *>(s_o + (v * GM + g) * D + d);
          L += s_l[v][g] * f;
          A0 += x.x * f;
          A1 += x.y * f;
        }
        if (pieces == 1) {
          *reinterpret_cast<uint32_t *>(out + g * o_head + d) = over_sum(A0, A1, L);
        } else {
          store_partial2(partial + g * ROW + 2 + d, A0, A1);
          if (d == 0) store_partial2(partial + g * ROW, M, L);
        }
      }
      if (pieces > 1) {
        s_unit[0][0] = unit;
        split = 1;
      }
    }
    pos += together || sh.whole ? 1 : t1 - t0;
    if (pos < end && pos >= s_pre[b + 1]) b = sequence_at(pos);
  }
  // The joins come after the loop, so that they take none of its registers: what they
  // need spilled there cost a tenth of a long call.
  const auto e = params_again<PagedDecodeParams>();
  auto rows_of = [&](const Unit &u, uint32_t *heads) -> uint16_t * {
    const uint32_t kvh = u.j / e->head_chunks, hc = u.j % e->head_chunks;
    *heads = min(e->chunk, e->group - hc * e->chunk);
    return e->out + (int64_t)u.b * e->o_seq + (int64_t)(kvh * e->group + hc * e->chunk) * e->o_head;
  };
  const size_t row_stride = (size_t)e->chunk * ROW;
  float *spare = reinterpret_cast<float *>(stage);
  // Its units' joins are the wave's own; in a workgroup's piece of a split unit, the last
  // of the unit's pieces joins them all, or kJoin of them, and the last of those steps the
  // steps (256 pieces by one workgroup took 70 us).
  uint32_t n = together ? split : done, step = 0;
  for (uint32_t i = 0; i < n; ++i) {
    const Unit u = s_unit[together ? 0 : wave][together ? 0 : i];
    uint32_t heads, parts = u.pieces, first = 0;
    size_t apart = row_stride;
    uint16_t *out = rows_of(u, &heads);
    if (together) {
      const uint32_t groups = u.pieces > 2 * kJoin ? (u.pieces + kJoin - 1) / kJoin : 1;
      uint32_t *counter = e->counters + (size_t)(u.b * upb + u.j) * e->counter_stride;
      if (groups > 1 && step == 0) {
        first = (w - u.slot) / kJoin * kJoin;
        parts = min(kJoin, u.pieces - first);
        counter = e->step_counters + u.slot + first;
        out = nullptr;
        n = 2;  // the steps are next
      } else if (groups > 1) {
        parts = groups;
        apart = kJoin * row_stride;
      }
      step = 1;
      wait_vmcnt<0>();
      __syncthreads();
      if (tid == 0) s_last = finished_last(counter, parts);
      __syncthreads();
      if (s_last == 0) return;
    }
    join_parts<D>(e->partial + (u.slot + first) * row_stride, apart, parts, heads, c2, out, e->o_head, together ? wave : 0,
                  together ? WAVES : 1, spare, lane);
  }
}

template <int D>
hipError_t launch_d(const PagedDecodeParams &p, const Launch &l) {
  return dispatch(attn_decode_paged_kernel<D>, dim3(p.workgroups), dim3(kWaves * 64), 0, l, p);
}

}  // namespace

uint32_t paged_decode_workgroups(uint32_t compute_units) {
  return kPerCu * (compute_units > 1 ? compute_units : 1);
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
