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
//  - at head_dim 256 a wave's accumulators and Q leave room for one wave per SIMD, so the
//    next tile's scores are computed beside this one's softmax, each operand read four
//    products ahead, in the source's order (three prompts of 1000 to 3000 rows, 16 heads on
//    4: 158 us, and 180 us where the products wait for the softmax and for LDS).
//  - Order: the work per row tile is known on the device only. Every workgroup works out
//    the same plan from the sequences' rows and lengths and takes the piece of its rank:
//    tiles with more keys than a workgroup's even share are cut into pieces, which come
//    first, then the whole tiles with most keys first. The pieces of a cut tile leave
//    their max, sum and weighted values (f32), and the last of them to finish joins them
//    in order.
//  - A weight of 0 (a masked key, or one below f16's range) times a value that is not finite
//    is NaN: masked tiles' such values are taken out, and where they, or a NaN in a row with a
//    finite sum, are found, the workgroup looks through its keys' values once more after the
//    last tile and lets each column's infinities and NaN decide it.
// Bound by the matrix instructions with the exponentials beside them for long prompts (two
// of 4000 to 6000 rows, 32 heads on 8 of 128: 414 to 434 us on several cards, 0.96 to 1.0
// PFLOP/s, a large f16 product's rate being 1.34), by the bytes of K and V for a few rows on a
// long cache, and for short prompts by what every row tile needs once: its place in the plan
// (2.5 us), Q and the first tile (3 us) and the output (1.5 us), beside two such workgroups
// per CU.
#include <algorithm>
#include <type_traits>

#include "paged_tile.hpp"
#include "prefill_tile.hpp"

namespace mi {
namespace kernels {
namespace {

using namespace mi::dev;

// Keys per tile: at head_dim 256 half as many, as the accumulators and Q take half of a
// wave's registers (64 keys there spill: 233 us instead of 152 for three prompts of 1000 to
// 3000 rows).
constexpr int tile_keys(int head_dim) { return head_dim == 256 ? 32 : kPrefillBlockN; }
constexpr int BM = kPrefillBlockM;  // rows per workgroup
// Added to every weight's exponent, so that f16 holds weights down to 2^-32 of the
// reference's (a long tail of them counts); it cancels against the row sum.
constexpr float kBias = 8.0f;
// Fewest key tiles of a piece of a cut row tile, and most pieces: a join costs as much as
// some tiles (64 rows of 64 heads on 4000 keys: 32 us with at least 8, 42 us with 4), and the
// time of many pieces' joins grows with them (32 rows of 32 heads on 16384 keys: 41, 38 and
// 49 us with up to 16, 32 and 64; 272 us uncut). Both, and kOneJoin and join_size below, were
// measured at head_dim 128; at 256 the same numbers stand, of tiles half as long and partials
// twice as large.
constexpr uint32_t kLeastPiece = 8, kMostPieces = 32;
// More pieces than kOneJoin are joined a few at a time by several workgroups, and then those
// joins: about the square root of their number. (64 rows of 64 heads on 4000 keys, 16 pieces
// a tile: 48 us by one workgroup each, 42 us four at a time.)
constexpr uint32_t kOneJoin = 8;
__device__ __forceinline__ uint32_t join_size(uint32_t pieces) { return pieces > 16 ? 6 : 4; }
// The least weight of a piece in a join: nothing beside finite sums, but not 0.
constexpr float kSmallest = 0x1p-126f;
constexpr int kReadAhead = 4;       // LDS operand reads in flight ahead of the MFMAs
constexpr int kSchedMfma = 0x008, kSchedDsRead = 0x100;

// A sequence as the plan sees it: its row tiles, the key tiles of the first and of the
// last of them, and the position of its first row (negative: more rows than keys; the
// most that the table can name where it is further).
struct Rows {
  uint32_t tiles, least, most;
  int32_t first;
};

// Key tiles of the row tiles of one sequence. Under the causal mask they grow from tile
// to tile, else all are the same.
template <int BN, bool PAGED>
struct Tiles {
  Divisor group;
  uint32_t causal;
  uint32_t cap;  // keys that the table can name (PAGED)
  // Key tiles of a row tile whose last row is of token `last`.
  __device__ __forceinline__ uint32_t keys(int32_t first, uint32_t last) const {
    const int32_t seen = first + (int32_t)(PAGED ? min(last + 1, cap - (uint32_t)first) : last + 1);
    return ((uint32_t)max(0, seen) + BN - 1) / BN;
  }
  // Key tiles of tile i, of `tokens` tokens.
  __device__ __forceinline__ uint32_t of(int32_t first, uint32_t tokens, uint32_t i) const {
    return keys(first, causal != 0 ? min(tokens - 1, divide((i + 1) * BM - 1, group)) : tokens - 1);
  }
  __device__ __forceinline__ Rows sequence(int32_t first, uint32_t tokens) const {
    const uint32_t n = (tokens * group.value + BM - 1) / BM;
    return n == 0 ? Rows{0, 0, 0, 0} : Rows{n, of(first, tokens, 0), of(first, tokens, n - 1), first};
  }
  // The first row tile with at least x key tiles (the count of them if none has): that of
  // the first token that sees key (x - 1) BN.
  __device__ __forceinline__ uint32_t first_with(Rows r, uint32_t x) const {
    const uint32_t i = (uint32_t)((int32_t)((x - 1) * BN) - r.first) * group.value / BM;
    return x <= r.least ? 0 : x > r.most ? r.tiles : i;
  }
  // Key tiles of tile i.
  __device__ __forceinline__ uint32_t at(Rows r, uint32_t i) const {
    return causal == 0 || i + 1 >= r.tiles ? r.most : keys(r.first, divide((i + 1) * BM - 1, group));
  }
};

// What the workgroup of a rank does: key tiles [begin, end) of a row tile, as piece
// `piece` of `pieces`; `cut` numbers the tiles that are cut.
struct Piece {
  uint32_t b, tile, begin, end, piece, pieces, cut;
};

// The piece of `rank` (of one KV head), the same in every wave that asks. `share`: the
// workgroups that the chip runs at once for one KV head.
template <int BN, bool PAGED>
__device__ __forceinline__ bool plan_piece(const PackedParams &p, const Tiles<BN, PAGED> &t, uint32_t rank, const Rows *s_rows,
                                           uint32_t *s_before, int lane, Piece *out) {
  // The first 64 sequences stay in registers.
  const uint32_t own = min((uint32_t)lane, p.batch - 1);
  const bool is_own = (uint32_t)lane < p.batch;
  const uint32_t tiles = is_own ? s_rows[own].tiles : 0, least = s_rows[own].least, longest = is_own ? s_rows[own].most : 0;
  const int32_t start = s_rows[own].first;
  auto rows_of = [&](uint32_t c0) __attribute__((always_inline)) -> Rows {
    if (c0 == 0) return Rows{tiles, least, longest, start};
    const bool is = c0 + lane < p.batch;
    const uint32_t at = is ? c0 + lane : 0;
    return Rows{is ? s_rows[at].tiles : 0, s_rows[at].least, is ? s_rows[at].most : 0, s_rows[at].first};
  };
  uint32_t all = 0, most = 0, work = 0;  // row tiles; key tiles of the longest; of all (about)
  for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
    const Rows r = rows_of(c0);
    all += r.tiles;
    most = max(most, r.most);
    work += r.tiles * (r.least + r.most + 1) / 2;
  }
  all = wave_sum(all), most = wave_max(most), work = wave_sum(work);
  if (rank >= all + p.max_pieces) return false;
  // Most key tiles of a piece: an even share (room for the pieces that do not fill up,
  // half a piece per tile, where all of them fit the chip at once), at least kLeastPiece,
  // and at most kMostPieces pieces a tile.
  uint32_t cap = most;
  if (most >= 2 * kLeastPiece && p.max_pieces != 0) {
    const uint32_t slots = all < p.share ? p.share - all / 2 : p.share;
    cap = max(max(kLeastPiece, (work + slots - 1) / slots), (most + kMostPieces - 1) / kMostPieces);
  }
  // The cut tiles: those of at least cap + 1 key tiles, sequence after sequence. Should they
  // come to more than max_pieces, again with longer ones, once every wave is past its reads
  // of s_before.
  uint32_t cuts = 0, pieces = 0;
  bool found = false, again = false;
  for (;; cap *= 2) {
    if (again) __syncthreads();
    again = true;
    cuts = pieces = 0;
    found = false;
    if (cap >= most) break;
    for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
      const Rows r = rows_of(c0);
      const uint32_t x = scan64(r.tiles - t.first_with(r, cap + 1));
      if (c0 + lane < p.batch) s_before[c0 + lane + 1] = cuts + x;
      cuts += last_lane(x);
    }
    if (lane == 0) s_before[0] = 0;
    if (cuts > p.max_pieces) continue;
    for (uint32_t k0 = 0; k0 < cuts; k0 += 64) {
      const uint32_t k = k0 + lane;
      uint32_t lo = 0;  // the last sequence with s_before[lo] <= k
      for (uint32_t step = 512; step != 0; step >>= 1)
        if (lo + step < p.batch && s_before[lo + step] <= k) lo += step;
      const Rows r = s_rows[lo];
      const uint32_t i = k < cuts ? t.first_with(r, cap + 1) + k - s_before[lo] : 0;
      const uint32_t n = k < cuts ? t.at(r, i) : 0, s = (n + cap - 1) / cap;
      const uint32_t x = scan64(s);
      const uint64_t le = __ballot(pieces + x <= rank);
      if (!found && le != ~0ull) {
        const int at = __popcll(le);
        const uint32_t s_at = (uint32_t)__builtin_amdgcn_readlane((int)s, at);
        const uint32_t n_at = (uint32_t)__builtin_amdgcn_readlane((int)n, at);
        const uint32_t z = rank - (pieces + (uint32_t)__builtin_amdgcn_readlane((int)x, at) - s_at);
        *out = {(uint32_t)__builtin_amdgcn_readlane((int)lo, at), (uint32_t)__builtin_amdgcn_readlane((int)i, at),
                z * n_at / s_at, (z + 1) * n_at / s_at, z, s_at, k0 + at};
        found = true;
      }
      pieces += last_lane(x);
    }
    if (pieces <= p.max_pieces) break;
  }
  if (found) return true;
  // The whole tiles, most key tiles first: the largest x of which more than rank tiles
  // have at least x. (Seven prompts of 150 to 1500 rows, 40 heads on 8: 95 us, 103 us in the
  // order of the rows; forty of 100 to 500 at head_dim 64 53 and 50 us.)
  rank -= pieces;
  if (rank >= all - cuts) return false;
  auto at_least = [&](uint32_t x) -> uint32_t {
    uint32_t n = 0;
    for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
      const Rows r = rows_of(c0);
      n += r.tiles - t.first_with(r, x);
    }
    return wave_sum(n) - cuts;
  };
  uint32_t x = 0, above = min(cap, most) + 1;  // at_least(x) > rank >= at_least(above)
  // Where all tiles fit the chip at once their order does not matter.
  const bool any_order = all + pieces <= p.share;
  while (!any_order && above - x > 1) {
    const uint32_t mid = (x + above) / 2;
    (at_least(mid) > rank ? x : above) = mid;
  }
  rank -= any_order ? 0 : at_least(above);
  for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
    const Rows r = rows_of(c0);
    const uint32_t first = t.first_with(r, x);
    const uint32_t n = scan64(t.first_with(r, above) - first);
    const uint64_t le = __ballot(n <= rank);
    if (le != ~0ull) {
      const int at = __popcll(le);
      const uint32_t before = at == 0 ? 0 : (uint32_t)__builtin_amdgcn_readlane((int)n, at - 1);
      const uint32_t b = c0 + at, tile = (uint32_t)__builtin_amdgcn_readlane((int)first, at) + rank - before;
      if (b >= p.batch) return false;
      *out = {b, tile, 0, t.at(s_rows[b], tile), 0, 1, 0};
      return true;
    }
    rank -= last_lane(n);
  }
  return false;
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
  constexpr int BN = tile_keys(D), MT = BN / 32;
  constexpr int RPB = 512 / D;         // tile rows per 1 KB direct load
  constexpr int RPW = BN / 4;          // tile rows that a wave loads
  constexpr int BPW = RPW / RPB;       // its direct loads of K (and V) per tile
  constexpr uint32_t GROUPS = BN / 16, HELD = 64 / GROUPS;  // 16-key groups per tile; tiles whose page ids a wave holds
  constexpr int DC = D / 16, DT = D / 32;
  constexpr bool PIPE = D == 256;      // one wave per SIMD
  constexpr int TILE = BN * D, OUT = 64 * D;  // halves of a tile, and of two waves' output rows
  // One array per stage, and the stage a compile-time choice, so that the compiler can
  // tell the loads into one from the reads of the other.
  __shared__ __attribute__((aligned(16))) uint16_t k_lds_a[OUT], k_lds_b[OUT];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds_a[TILE], v_lds_b[TILE];
  __shared__ uint32_t s_bad;  // whether some of the piece's V decide columns whatever their weights are
  __shared__ Rows s_rows[kPackedMaxBatch];
  __shared__ uint32_t s_before[kPackedMaxBatch + 1], s_last;
  auto k_stage = [&](int st) __attribute__((always_inline)) -> uint16_t * { return st ? k_lds_b : k_lds_a; };
  auto v_stage = [&](int st) __attribute__((always_inline)) -> uint16_t * { return st ? v_lds_b : v_lds_a; };

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const uint32_t G = p.group.value;

  // Workgroups go round-robin over the 8 XCDs: where the KV heads divide evenly, each
  // XCD takes whole heads, whose K and V stay in its L2.
  uint32_t kvh, rest;
  {
    const bool whole = p.kv_heads % 8 == 0;
    const uint32_t per = p.heads_apart.value, k = whole ? blockIdx.x / 8 : blockIdx.x;
    rest = divide(k, p.heads_apart);
    kvh = k - rest * per + (whole ? blockIdx.x % 8 * per : 0);
  }
  // The sequences' rows and first positions (every wave writes all of them, and reads back
  // what it wrote itself), and the piece of this rank. Positions past the table have no keys.
  const uint32_t cap = PAGED ? p.kv.table_width << p.kv.page_shift : 0;
  const Tiles<BN, PAGED> row_tiles{p.group, p.causal, cap};
  for (uint32_t c0 = 0; c0 < p.batch; c0 += 64) {
    const uint32_t bb = c0 + lane;
    if (bb >= p.batch) continue;
    const RowRange r = sequence_rows(p.row_starts, bb, p.rows);
    const uint32_t tokens = r.end - r.begin;
    s_rows[bb] = row_tiles.sequence(PAGED ? (int32_t)min((int64_t)p.kv.lengths[bb] - tokens, (int64_t)cap) : 0, tokens);
  }
  Piece pc;
  if (!plan_piece(p, row_tiles, rest, s_rows, s_before, lane, &pc)) return;
  const uint32_t b = __builtin_amdgcn_readfirstlane(pc.b), tile = __builtin_amdgcn_readfirstlane(pc.tile);
  const uint32_t t_begin = __builtin_amdgcn_readfirstlane(pc.begin), t_end = __builtin_amdgcn_readfirstlane(pc.end);
  const RowRange range = sequence_rows(p.row_starts, b, p.rows);
  const uint32_t tokens = range.end - range.begin;
  const uint32_t L = PAGED ? paged_length(p.kv, b) : tokens;
  // Position of the first row (negative: more rows than keys).
  const int64_t off = PAGED ? (int64_t)p.kv.lengths[b] - tokens : 0;

  const uint32_t row0 = tile * BM, my_row = row0 + wave * 32 + n;
  const uint32_t my_t = divide(my_row, p.group), my_g = my_row - my_t * G;
  const bool row_ok = my_t < tokens;
  const uint32_t t_first = divide(row0, p.group), t_last = min(tokens - 1, divide(row0 + BM - 1, p.group));
  const uint32_t kmax = p.causal != 0 ? (uint32_t)max((int64_t)0, min(off + t_last + 1, (int64_t)L)) : L;
  const bool active = row0 + wave * 32 < tokens * G;  // whether this wave has rows
  // Last key that this lane's row sees, and that the tile's first row does.
  const int64_t lim = p.causal != 0 ? min(off + min(my_t, tokens - 1), (int64_t)L - 1) : (int64_t)L - 1;
  const int64_t full_lim = p.causal != 0 ? min(off + t_first, (int64_t)L - 1) : (int64_t)L - 1;

  // Q^T as the B operand: lane (h, n) holds Q[row n][16 c + 8 h .. + 8].
  h8_t qop[DC];
  {
    const uint16_t *qrow = p.q + (int64_t)(range.begin + min(my_t, tokens - 1)) * p.q_tok +
                           (int64_t)(kvh * G + my_g) * p.q_head + 8 * h;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      qop[c] = row_ok ? as_h8(*reinterpret_cast<const uint4 *>(qrow + 16 * c)) : as_h8(make_uint4(0, 0, 0, 0));
  }

  // Page ids of the tiles' 16-key groups: lane l holds group l of the 64 (HELD tiles)
  // since tile HELD k. `absent` has a bit for each group without a page, gone_a / gone_b
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

  // Direct loads of tile ti's K or V into a stage: each wave fills RPW rows, lane L writing
  // bytes 16 L .. 16 L + 15 of a 1 KB block, so it fetches the 16 bytes that belong at that
  // swizzled position. A scalar base and loop-invariant offsets; rows past the last key
  // that any row sees, or without a page, take an offset past the buffer's end, which
  // loads zeros. (Buffer loads without branches: the compiler then counts exactly which
  // loads into LDS are in flight, and waits for no others.)
  uint32_t k_off[BPW], v_off[BPW];
#pragma unroll
  for (int i = 0; i < BPW; ++i) {
    const int r = i * RPB + lane / CPR, row = wave * RPW + r, pc = lane % CPR;
    k_off[i] = ((uint32_t)r * (uint32_t)p.kv.k_pos + ((pc ^ k_swizzle<D>(row)) * 8)) * 2u;
    v_off[i] = ((uint32_t)r * (uint32_t)p.kv.v_pos + ((pc ^ v_swizzle<D>(row)) * 8)) * 2u;
  }
  uint32_t page_of = 0, gone_new = 0;  // of the tile found last: its page, and its groups without one
  auto find = [&](uint32_t ti) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      if (ti % HELD == 0 || ti == t_begin) load_ids(ti / HELD * HELD);
      page_of = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(GROUPS * (ti % HELD) + wave * RPW / 16));
      gone_new = (uint32_t)(absent >> (GROUPS * (ti % HELD))) & ((1u << GROUPS) - 1);
    }
  };
  auto issue = [&](uint32_t ti, const uint16_t *pool, int64_t page_st, int64_t pos_st, int64_t head_st,
                   const uint32_t (&at)[BPW], uint16_t *dst) __attribute__((always_inline)) {
    const uint32_t key = ti * BN + wave * RPW;
    uint32_t rows = key < kmax ? kmax - key : 0;
    const uint16_t *first = pool + (int64_t)kvh * head_st;
    if constexpr (PAGED) {
      rows = page_of < p.kv.pages ? rows : 0;
      first += (int64_t)page_of * page_st + (int64_t)(key & in_page) * pos_st;
    } else {
      first += (int64_t)(range.begin + key) * pos_st;
    }
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const bool ok = i * RPB + lane / CPR < rows;
      load_lds16_buffer(first, ok ? at[i] : kBufferEnd, dst + wave * RPW * D + i * 512);
    }
  };
  auto issue_k = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    issue(ti, p.kv.k, p.kv.k_page, p.kv.k_pos, p.kv.k_head, k_off, k_stage(stage));
  };
  auto issue_v = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    issue(ti, p.kv.v, p.kv.v_page, p.kv.v_pos, p.kv.v_head, v_off, v_stage(stage));
  };
  auto issue_tile = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    find(ti);
    (stage ? gone_b : gone_a) = gone_new;
    issue_k(ti, stage);
    issue_v(ti, stage);
  };
  // Tiles wholly inside the first row's window need no mask.
  const uint32_t n_full = full_lim < 0 ? 0 : (uint32_t)min((int64_t)t_end, (full_lim + 1) / BN);
  // A masked tile's V may hold values that some of its rows must not see and that are
  // not finite, and 0 times those is NaN. Each wave looks at the rows it has loaded: such
  // values become zeros, and the rows that see them get them after the last tile.
  auto look = [&](uint32_t ti, int stage) __attribute__((always_inline)) {
    if (ti < n_full) return;
    uint16_t *mine = v_stage(stage) + wave * RPW * D;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      uint4 *at = reinterpret_cast<uint4 *>(mine + i * 512 + lane * 8);
      const uint4 v = *at;
      if ((not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w)) != 0) {
        *at = make_uint4(finite_part(v.x), finite_part(v.y), finite_part(v.z), finite_part(v.w));
        bad = true;
      }
    }
    if (__any(bad)) s_bad = 1;
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

  float16_t s_cur[MT];  // with PIPE: the scores of the tile that the next step takes
  // S^T[key][row] = K Q^T of a tile.
  auto scores = [&](const uint16_t *k_lds, float16_t (&s)[MT]) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mt][r] = 0.0f;
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const uint16_t *kp = k_lds + (32 * mt + n) * D + (((2 * c + h) ^ k_swizzle<D>(n)) * 8);
        s[mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(*reinterpret_cast<const uint4 *>(kp)), qop[c], s[mt], 0, 0, 0);
      }
    }
  };
  auto step = [&](uint32_t it, auto mask_tag, auto stage_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    constexpr int ST = decltype(stage_tag)::value;
    const uint32_t j0 = it * BN;
    const uint16_t *k_lds = ST ? k_lds_b : k_lds_a;
    const uint16_t *v_lds = ST ? v_lds_b : v_lds_a;
    const uint32_t gone = !PIPE && ST ? gone_b : gone_a;
    // Issued here and not at the end of the step before, where the loads would be in flight
    // over the loop's back edge: the compiler then takes one stage's for the other's, and
    // waits for them before it reads the stage that is complete.
    if (!PIPE && it + 1 < t_end) issue_tile(it + 1, ST ^ 1);
    if (active) {
      float16_t s[MT], nx[MT];
      if constexpr (PIPE) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt] = s_cur[mt];
        // The accumulators stay in one half of the register file: left to itself the compiler
        // moves all of them to the other one and back in every second step.
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) asm volatile("" : "+a"(o[dt]));
      } else {
        // Two 32-key halves, at raised wave priority.
        __builtin_amdgcn_s_setprio(1);
        scores(k_lds, s);
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, kReadAhead, 0);
#pragma unroll
        for (int k = 0; k < MT * DC - kReadAhead; ++k) {
          __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, kReadAhead, 0);
        __builtin_amdgcn_s_setprio(0);
      }
      // Key 32 mt + 8 (r >> 2) + 4 h + (r & 3) of the tile is seen when it is at most
      // lim_rel; the lane's 4 h moves to the limit, so each compare is with a constant.
      int lim_lane = BN;
      if constexpr (MASK) {
        lim_lane = (int)max(min(lim - (int64_t)j0, (int64_t)BN), (int64_t)-1) - 4 * h;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[mt][r] = 32 * mt + 8 * (r >> 2) + (r & 3) > lim_lane ? -INFINITY : s[mt][r];
      }
      if (PAGED && gone != 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (gone >> (2 * mt + (r >> 3)) & 1) s[mt][r] = -INFINITY;
      }
      // P = 2^(s c2 - m c2 + kBias) against the row's reference max m_run, as f16 pairs
      // in accumulator order.
      uint32_t pw[MT][8];
      float psum;
      auto weights = [&](float mc) __attribute__((always_inline)) {
        float ps0 = 0.0f, ps1 = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
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
      uint4 kf[kReadAhead], vf[kReadAhead];
      auto read_k = [&](int c) __attribute__((always_inline)) {
        const uint16_t *kp = (ST ? k_lds_a : k_lds_b) + (32 * (c / DC) + n) * D + (((2 * (c % DC) + h) ^ k_swizzle<D>(n)) * 8);
        kf[c % kReadAhead] = *reinterpret_cast<const uint4 *>(kp);
      };
      auto read_v = [&](int i) __attribute__((always_inline)) {
        const uint16_t *v0 = v_lds + 16 * (i / DT) * D + tr_off + ((4 * (i % DT) + tr_chunk) ^ v_swizzle<D>(tr_key)) * 8;
        const uint2 lo = read_tr16(v0), hi = read_tr16(v0 + 8 * D);
        vf[i % kReadAhead] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      };
      if constexpr (PIPE) {
        // The next tile's scores beside this one's softmax (of the last tile: of whatever the
        // stage holds, and not used), each operand read kReadAhead products early; the order is
        // the source's.
        const float mc = m_run * c2 - kBias;
        float ps0 = 0.0f, ps1 = 0.0f, even = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r) nx[mt][r] = 0.0f;
#pragma unroll
        for (int c = 0; c < kReadAhead; ++c) read_k(c);
#pragma unroll
        for (int c = 0; c < MT * DC; ++c) {
          // One product, the read of a later one's operand, and one of the tile's 16 MT weights.
          static_assert(DC == 16 || !PIPE, "a weight per product");
          const int mt = c / DC, r = c % 16;
          __builtin_amdgcn_sched_barrier(0);
          nx[mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(kf[c % kReadAhead]), qop[c % DC], nx[mt], 0, 0, 0);
          if (c + kReadAhead < MT * DC) read_k(c + kReadAhead);
          else read_v(c + kReadAhead - MT * DC);
          const float e = exp2_raw(fmaf(s[mt][r], c2, -mc));
          if (r & 1) {
            pw[mt][r >> 1] = pack_f16x2(even, e);
            if (r & 2) ps1 = dot2(pw[mt][r >> 1], 0x3c003c00u, ps1);
            else ps0 = dot2(pw[mt][r >> 1], 0x3c003c00u, ps0);
          }
          even = e;
        }
        __builtin_amdgcn_sched_barrier(0);
        psum = ps0 + ps1;
      } else {
        weights(m_run * c2 - kBias);
      }
      // The reference moves only when a weight leaves f16's range: the sum is then +inf
      // or NaN, as it is for a row without a reference yet (m_run = -inf).
      if (__any(!(psum <= __FLT_MAX__))) {
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
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
      // O^T[d][row] += V^T[d][keys] P^T[keys][row], 16-key chunks.
      if constexpr (PIPE) {
#pragma unroll
        for (int i = 0; i < BN / 16 * DT; ++i) {
          const int mt = i / DT >> 1, base = (i / DT & 1) * 4;
          const h8_t pb = as_h8(make_uint4(pw[mt][base], pw[mt][base + 1], pw[mt][base + 2], pw[mt][base + 3]));
          __builtin_amdgcn_sched_barrier(0);
          o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(vf[i % kReadAhead]), pb, o[i % DT], 0, 0, 0);
          if (i + kReadAhead < BN / 16 * DT) read_v(i + kReadAhead);
        }
        __builtin_amdgcn_sched_barrier(0);
      } else {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) {
          const int mt = c >> 1, base = (c & 1) * 4;
          const h8_t pb = as_h8(make_uint4(pw[mt][base], pw[mt][base + 1], pw[mt][base + 2], pw[mt][base + 3]));
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const uint16_t *v0 = v_lds + 16 * c * D + tr_off + ((4 * dt + tr_chunk) ^ v_swizzle<D>(tr_key)) * 8;
            const uint2 lo = read_tr16(v0), hi = read_tr16(v0 + 8 * D);
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, o[dt], 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2 * kReadAhead, 1);
#pragma unroll
        for (int k = 0; k < BN / 16 * DT - kReadAhead; ++k) {
          __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 1);
          __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, kReadAhead, 1);
        __builtin_amdgcn_s_setprio(0);
      }
      if constexpr (PIPE) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s_cur[mt] = nx[mt];
      }
    }
    // Tile it + 1 has landed in this wave's part of the other stage; after the barrier
    // nobody reads this stage, which then receives tile it + 2 (with PIPE its V, and the K
    // of tile it + 3 goes into the other stage).
    wait_vmcnt<0>();
    if (it + 1 < t_end) look(it + 1, ST ^ 1);
    __syncthreads();
    if constexpr (PIPE) {
      gone_a = gone_b, gone_b = gone_new;
      if (it + 2 < t_end) issue_v(it + 2, ST);
      if (it + 3 < t_end) {
        find(it + 3);
        issue_k(it + 3, ST ^ 1);
      }
    }
  };

  if (t_begin < t_end) {
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if constexpr (PIPE) {
      find(t_begin);
      gone_a = gone_new;
      issue_k(t_begin, 0);
      issue_v(t_begin, 0);
      if (t_begin + 1 < t_end) {
        find(t_begin + 1);
        gone_b = gone_new;
        issue_k(t_begin + 1, 1);
      }
      wait_vmcnt<0>();
      look(t_begin, 0);
      __syncthreads();
      if (active) scores(k_lds_a, s_cur);
      __syncthreads();
      if (t_begin + 1 < t_end) issue_v(t_begin + 1, 1);
      if (t_begin + 2 < t_end) {
        find(t_begin + 2);
        issue_k(t_begin + 2, 0);
      }
    } else {
      issue_tile(t_begin, 0);
      wait_vmcnt<0>();
      look(t_begin, 0);
      __syncthreads();
    }
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    uint32_t it = t_begin;
    for (; it + 1 < n_full; it += 2) {
      step(it, std::false_type{}, S0{});
      step(it + 1, std::false_type{}, S1{});
    }
    if (it < n_full) {
      step(it, std::false_type{}, S0{});
      ++it;
    }
    if (((it - t_begin) & 1) != 0 && it < t_end) {
      step(it, std::true_type{}, S1{});
      ++it;
    }
    for (; it + 1 < t_end; it += 2) {
      step(it, std::true_type{}, S0{});
      step(it + 1, std::true_type{}, S1{});
    }
    if (it < t_end) step(it, std::true_type{}, S0{});
  }

  const float l_total = l_run + __shfl_xor(l_run, 32, 64);
  if (t_begin < t_end) {
    // A weight below f16's smallest value is 0, and 0 times an infinity that the row sees is
    // NaN, where the weight itself leaves the infinity. Where a row with a finite sum has a
    // value that is not finite, or a masked tile's were taken out, the workgroup looks at
    // the values of its keys again: a column's infinities and NaN decide it.
    float most = 0.0f;  // NaN if a value is
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(o[dt][r]), fabsf(o[dt][r + 1])), most);
    if (__any(!(most <= __FLT_MAX__) && l_total > 0.0f)) s_bad = 1;
    __syncthreads();  // also: every wave is past its last LDS operand read
    if (__builtin_expect(s_bad != 0, 0)) {
      // The first keys of each column that hold an infinity or NaN, and a negative one or NaN.
      uint32_t *first = reinterpret_cast<uint32_t *>(k_lds_a);
      for (uint32_t i = tid; i < 2 * D; i += 256) first[i] = ~0u;
      __syncthreads();
      const uint32_t last = min(t_end * BN, kmax), chunk = lane % CPR;
#pragma unroll 1
      for (uint32_t key = t_begin * BN + 16 * wave; key < last; key += 64) {
        const uint16_t *row = p.kv.v + (int64_t)kvh * p.kv.v_head + 8 * chunk;
        bool there = true;
        if constexpr (PAGED) {
          const uint32_t page = p.kv.table[(int64_t)b * p.kv.table_seq + (key >> shift)];
          there = page < p.kv.pages;
          row += (int64_t)page * p.kv.v_page + (int64_t)(key & in_page) * p.kv.v_pos;
        } else {
          row += (int64_t)(range.begin + key) * p.kv.v_pos;
        }
#pragma unroll
        for (int i = 0; i < CPR / 4; ++i) {
          const uint32_t r = (64 * i + lane) / CPR;
          if (!there || key + r >= last) continue;
          uint32_t bits = not_finite_columns(*reinterpret_cast<const uint4 *>(row + (int64_t)r * p.kv.v_pos));
          for (uint32_t e = 0; bits != 0; ++e, bits >>= 2) {
            if ((bits & 1) != 0) atomicMin(&first[8 * chunk + e], key + r);
            if ((bits & 2) != 0) atomicMin(&first[D + 8 * chunk + e], key + r);
          }
        }
      }
      __syncthreads();
      if (l_total > 0.0f) {
        // d = 32 dt + 8 q + 4 h + e of this lane's row, which sees the keys up to lim.
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint32_t d = 32 * dt + 8 * (r >> 2) + 4 * h + (r & 3);
            const bool positive = (int64_t)first[d] <= lim, negative = (int64_t)first[D + d] <= lim;
            if (positive) o[dt][r] = negative ? __builtin_nanf("") : INFINITY;
            else if (negative) o[dt][r] = -INFINITY;
          }
      }
      __syncthreads();
    }
  }
  const uint32_t pieces = __builtin_amdgcn_readfirstlane(pc.pieces), piece = __builtin_amdgcn_readfirstlane(pc.piece);
  // 32 rows of each wave as f16, in a region of the idle stages.
  auto rows_lds = [&](int v) __attribute__((always_inline)) { return (v < 2 ? k_lds_a : k_lds_b) + (v & 1) * 32 * D; };
  static_assert(2 * 32 * D <= OUT, "output staging");
  // d = 32 dt + 8 q + 4 h + 0 .. 3 of row n.
  auto stage_row = [&](uint16_t *rows, int dt, int q, float a, float b2, float c, float d) __attribute__((always_inline)) {
    const int chunk = (4 * dt + q) ^ out_swizzle<D>(n);
    *reinterpret_cast<uint2 *>(rows + n * D + chunk * 8 + 4 * h) = make_uint2(pack_f16x2(a, b2), pack_f16x2(c, d));
  };
  bool join = false;
  if (pieces > 1) {
    // This piece's rows, in the accumulators' own order so that a store's lanes are
    // neighbours: per wave 8-byte slots of 64 lanes, (m, l), room for those of a
    // join, and O two by two. A row that saw no key here has m = -inf.
    constexpr uint32_t WAVE = packed_partial_slots(D) * 64 * 2, PIECE = 4 * WAVE;
    float *tile_partial = p.partial + ((size_t)kvh * p.max_pieces + (rest - piece)) * PIECE + lane * 2;
    if (active) {
      float *mine = tile_partial + (size_t)piece * PIECE + wave * WAVE;
      store_partial2(mine, m_run, l_total);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 2) store_partial2(mine + (2 + 8 * dt + r / 2) * 128, o[dt][r], o[dt][r + 1]);
    }
    // The last of a tile's pieces to finish joins all of them, in order; of more than
    // kOneJoin, the last of each few in a row joins those, into the first of them, and the
    // last of these joins does the rest. A wave takes 32 values of d of 32 rows at a time
    // (two such blocks, two pieces a round trip), of whichever wave's rows.
    join = true;
    const bool steps = pieces > kOneJoin;
    const uint32_t few = join_size(pieces);
    uint32_t first = steps ? piece / few * few : 0, parts = steps ? min(pieces - first, few) : pieces, gap = 1;
    uint32_t counter_at = steps ? p.max_pieces * (p.kv_heads + kvh) + (rest - piece) + first : kvh * p.max_pieces + pc.cut;
    counter_at = __builtin_amdgcn_readfirstlane(counter_at);
    const uint32_t blocks = DT * min(4u, (tokens * G - row0 + 31) / 32);
#pragma unroll 1
    for (;;) {
      wait_vmcnt<0>();
      __syncthreads();
      if (tid == 0) {
        uint32_t *counter = p.counters + (size_t)counter_at * p.counter_stride;
        const bool last = arrive(counter) == parts - 1;
        if (last) {
          acquire_partials();
          __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        s_last = last;
      }
      __syncthreads();
      if (s_last == 0) return;
      const bool final = !steps || gap != 1;
      constexpr uint32_t FEW = 2;
      for (uint32_t u0 = 2 * wave; u0 < blocks; u0 += 8) {
        float acc[2][16], M[2], sum[2];
        float *from[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t block = min(u0 + u, blocks - 1);
          from[u] = tile_partial + (size_t)first * PIECE + block / DT * WAVE + (2 + 8 * (block % DT)) * 128;
          M[u] = -INFINITY, sum[u] = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[u][r] = 0.0f;
        }
        // A piece's (m, l) are in its first slot, those of a join in the second.
        auto ml_at = [&](int u) __attribute__((always_inline)) {
          return (gap == 1 ? 2 : 1) * 128 + 8 * (min(u0 + u, blocks - 1) % DT) * 128;
        };
#pragma unroll 1
        for (uint32_t s0 = 0; s0 < parts; s0 += FEW) {
          float2 ml[2][FEW], v[2][FEW][8];
#pragma unroll
          for (uint32_t k = 0; k < FEW; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float *part = from[u] + (size_t)(min(s0 + k, parts - 1) * gap) * PIECE;
              ml[u][k] = load_partial2(part - ml_at(u));
#pragma unroll
              for (int i = 0; i < 8; ++i) v[u][k][i] = load_partial2(part + i * 128);
            }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float m = M[u];
#pragma unroll
            for (uint32_t k = 0; k < FEW; ++k) m = s0 + k < parts ? fmaxf(m, ml[u][k].x) : m;
            // Never 0, so that an infinity of a piece far below the others stays one. A piece
            // without a maximum has a sum of 0 (the row saw no key) or of NaN (every score is).
            const float r = fmaxf(exp2_raw((M[u] - m) * c2), kSmallest);
            M[u] = m;
            sum[u] *= r;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[u][i] *= r;
#pragma unroll
            for (uint32_t k = 0; k < FEW; ++k) {
              const bool use = s0 + k < parts;
              const float f = fmaxf(exp2_raw((ml[u][k].x - m) * c2), kSmallest);
              sum[u] = use ? fmaf(ml[u][k].y, f, sum[u]) : sum[u];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                acc[u][2 * i] = use ? fmaf(v[u][k][i].x, f, acc[u][2 * i]) : acc[u][2 * i];
                acc[u][2 * i + 1] = use ? fmaf(v[u][k][i].y, f, acc[u][2 * i + 1]) : acc[u][2 * i + 1];
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t block = u0 + u;
          if (block >= blocks) continue;
          if (final) {
            const float inv = 1.0f / sum[u];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              stage_row(rows_lds(block / DT), block % DT, q, acc[u][4 * q] * inv, acc[u][4 * q + 1] * inv,
                        acc[u][4 * q + 2] * inv, acc[u][4 * q + 3] * inv);
          } else {
            if (block % DT == 0) store_partial2(from[u] - 128, M[u], sum[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) store_partial2(from[u] + i * 128, acc[u][2 * i], acc[u][2 * i + 1]);
          }
        }
      }
      if (final) break;
      first = 0, parts = (pieces + few - 1) / few, gap = few;
      counter_at = __builtin_amdgcn_readfirstlane(kvh * p.max_pieces + pc.cut);
    }
  }
  // Normalise (a row that saw no key: 0 / 0) and store through LDS as whole 16-byte
  // chunks, D / 8 consecutive lanes per row.
  constexpr int RPI = 64 / CPR;  // rows per store instruction
  if (!join) {
    const float inv = 1.0f / l_total;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        stage_row(rows_lds(wave), dt, q, o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv, o[dt][4 * q + 2] * inv,
                  o[dt][4 * q + 3] * inv);
  }
  __syncthreads();
  const uint16_t *own_rows = rows_lds(wave);
  const int lane_o = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const int c_out = lane_o % CPR;
#pragma unroll
  for (int i = 0; i < 32 / RPI; ++i) {
    const int r = i * RPI + lane_o / CPR;
    const uint4 v = *reinterpret_cast<const uint4 *>(own_rows + r * D + (c_out ^ out_swizzle<D>(r)) * 8);
    const uint32_t prow = row0 + wave * 32 + r, t = divide(prow, p.group), g = prow - t * G;
    if (t < tokens)
      *reinterpret_cast<uint4 *>(p.out + (int64_t)(range.begin + t) * p.o_tok + (int64_t)(kvh * G + g) * p.o_head +
                                 c_out * 8) = v;
  }
}

template <int D>
hipError_t launch_d(const PackedParams &p, const Launch &l) {
  const dim3 grid((p.row_tiles + p.max_pieces) * p.kv_heads);
  return p.kv.table != nullptr ? dispatch(attn_packed_kernel<D, true>, grid, dim3(256), 0, l, p)
                               : dispatch(attn_packed_kernel<D, false>, grid, dim3(256), 0, l, p);
}

}  // namespace

uint32_t packed_workgroups(uint32_t compute_units, uint32_t head_dim) {
  return (head_dim == 256 ? 1 : 2) * (compute_units > 1 ? compute_units : 1);
}

uint64_t packed_pieces(uint64_t keys, uint64_t row_tiles, uint32_t head_dim) {
  const uint64_t tiles = (keys + tile_keys(head_dim) - 1) / tile_keys(head_dim);
  if (tiles < 2 * kLeastPiece) return 0;
  return row_tiles * std::min<uint64_t>(kMostPieces, (tiles + kLeastPiece - 1) / kLeastPiece);
}

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
