// The C ABI's operators over packed rows and the paged KV cache: their checks of
// arguments and launches. Everything that the host can see is checked here; tables,
// lengths and row offsets are device data, which the kernels keep in bounds.
#include <algorithm>
#include <cmath>
#include <exception>
#include <string>

#include "kernels.hpp"
#include "runtime.hpp"

namespace mi {
namespace {

constexpr uint64_t kRows31 = 1ull << 31;
constexpr uint64_t kDecodeTileKeys = 32;  // keys of the decode kernel's tile

mi_status check_batch(const mi_batch *batch) {
  if (batch == nullptr) return fail(MI_ERR_INVALID_ARGUMENT, "null batch");
  if (batch->committed) return fail(MI_ERR_RESOURCE, "batch was already committed");
  return MI_OK;
}

// f16 rows for 16-byte accesses: rank `rank`, unit innermost stride, base and outer
// strides multiples of 8 elements.
mi_status check_rows(const mi_tensor *t, int32_t rank, const char *what) {
  mi_status st = require_f16(t);
  if (st != MI_OK) return st;
  if (t->rank != rank) return fail(MI_ERR_SHAPE, std::string(what) + " must have rank " + std::to_string(rank));
  for (int32_t i = 0; i < rank; ++i)
    if (t->shape[i] < 0 || (uint64_t)t->shape[i] >= kRows31)
      return fail(MI_ERR_SHAPE, std::string(what) + " shape does not fit in u32");
  if (element_count(*t) == 0) return MI_OK;
  if (t->data == nullptr) return fail(MI_ERR_INVALID_ARGUMENT, std::string(what) + " has no data");
  bool ok = t->stride[rank - 1] == 1 && reinterpret_cast<uintptr_t>(t->data) % 16 == 0;
  for (int32_t i = 0; i < rank - 1; ++i) ok = ok && (t->shape[i] == 1 || t->stride[i] % 8 == 0);
  if (!ok) return fail(MI_ERR_SHAPE, std::string(what) + " needs unit-stride, 16-byte aligned rows");
  return MI_OK;
}

// A u32 vector of `count` words at unit stride.
mi_status check_words(const mi_tensor *t, int64_t count, const char *what) {
  if (t->dtype != MI_U32)
    return fail(MI_ERR_DTYPE, std::string("unsupported dtype: expected u32, got ") + dtype_name(t->dtype));
  if (t->rank != 1) return fail(MI_ERR_SHAPE, std::string(what) + " must have rank 1");
  if (t->shape[0] != count)
    return fail(MI_ERR_SHAPE, std::string(what) + " must have " + std::to_string(count) + " entries");
  if (count > 1 && t->stride[0] != 1) return fail(MI_ERR_SHAPE, std::string(what) + " needs a unit stride");
  if (count > 0 && t->data == nullptr) return fail(MI_ERR_INVALID_ARGUMENT, std::string(what) + " has no data");
  return MI_OK;
}

mi_status check_heads(uint64_t query_heads, uint64_t kv_heads, uint64_t head_dim) {
  if (kv_heads == 0 || query_heads == 0 || query_heads % kv_heads != 0)
    return fail(MI_ERR_SHAPE, "query_heads must be divisible by kv_heads");
  if (!kernels::paged_head_dim(head_dim)) return fail(MI_ERR_SHAPE, "head_dim must be 32, 64, 128, or 256");
  return MI_OK;
}

// Whether `rows` rows at `stride` elements can be addressed by unsigned 32-bit byte
// offsets (with room for the row itself).
bool rows_fit(int64_t stride, uint64_t rows) {
  return stride >= 0 && (uint64_t)stride < kRows31 && (uint64_t)stride * rows * 2 + 1024 < kRows31;
}

// The paged cache's tensors: key_pages / value_pages [P, S, Hkv, D], block_table [B, M],
// lengths [B].
mi_status check_paged(const mi_tensor *key_pages, const mi_tensor *value_pages, const mi_tensor *block_table,
                      const mi_tensor *lengths, int64_t batch, int64_t kv_heads, int64_t head_dim,
                      kernels::PagedKv *out) {
  mi_status st;
  if ((st = check_rows(key_pages, 4, "key pages")) != MI_OK || (st = check_rows(value_pages, 4, "value pages")) != MI_OK)
    return st;
  for (int i = 0; i < 4; ++i)
    if (key_pages->shape[i] != value_pages->shape[i])
      return fail(MI_ERR_SHAPE, "key and value pages must have the same shape");
  if (key_pages->shape[2] != kv_heads || key_pages->shape[3] != head_dim)
    return fail(MI_ERR_SHAPE, "attention tensor shapes do not match config");
  const int64_t pages = key_pages->shape[0], size = key_pages->shape[1];
  uint32_t shift = kernels::kPagedMinShift;
  while (shift < 20 && (1ll << shift) < size) ++shift;
  if (pages == 0 || size != (1ll << shift))
    return fail(MI_ERR_SHAPE, "pages must hold a power of two of at least 16 positions");
  if (element_count(*key_pages) != 0 &&
      (!rows_fit(key_pages->stride[1], (uint64_t)size) || !rows_fit(value_pages->stride[1], (uint64_t)size)))
    return fail(MI_ERR_SHAPE, "pages need a position stride that is not negative and less than 2 GiB");
  if (block_table->dtype != MI_U32)
    return fail(MI_ERR_DTYPE, std::string("unsupported dtype: expected u32, got ") + dtype_name(block_table->dtype));
  if (block_table->rank != 2 || block_table->shape[0] != batch || block_table->shape[1] <= 0)
    return fail(MI_ERR_SHAPE, "block table must be [sequences, pages of a sequence]");
  if (block_table->shape[1] > 1 && block_table->stride[1] != 1)
    return fail(MI_ERR_SHAPE, "block table needs a unit innermost stride");
  if ((uint64_t)block_table->shape[1] >= kRows31 >> shift)
    return fail(MI_ERR_SHAPE, "block table positions do not fit in 31 bits");
  if (batch > 0 && block_table->data == nullptr) return fail(MI_ERR_INVALID_ARGUMENT, "block table has no data");
  if ((st = check_words(lengths, batch, "lengths")) != MI_OK) return st;
  kernels::PagedKv kv{};
  kv.k = static_cast<const uint16_t *>(key_pages->data);
  kv.k_page = key_pages->stride[0], kv.k_pos = key_pages->stride[1], kv.k_head = key_pages->stride[2];
  kv.v = static_cast<const uint16_t *>(value_pages->data);
  kv.v_page = value_pages->stride[0], kv.v_pos = value_pages->stride[1], kv.v_head = value_pages->stride[2];
  kv.table = static_cast<const uint32_t *>(block_table->data), kv.table_seq = block_table->stride[0];
  kv.lengths = static_cast<const uint32_t *>(lengths->data);
  kv.pages = (uint32_t)pages, kv.page_shift = shift, kv.table_width = (uint32_t)block_table->shape[1];
  *out = kv;
  return MI_OK;
}

mi_status check_out(const mi_tensor *q, const mi_tensor *out, const char *what) {
  mi_status st = check_rows(out, 3, what);
  if (st != MI_OK) return st;
  for (int i = 0; i < 3; ++i)
    if (out->shape[i] != q->shape[i]) return fail(MI_ERR_SHAPE, std::string(what) + " must have the query's shape");
  return MI_OK;
}

mi_status check_query(const mi_tensor *q, const mi_attention_config *config, const mi_tensor *out) {
  mi_status st;
  if ((st = check_rows(q, 3, "query")) != MI_OK) return st;
  if (q->shape[1] != (int64_t)config->query_heads || q->shape[2] != (int64_t)config->head_dim)
    return fail(MI_ERR_SHAPE, "attention tensor shapes do not match config");
  if ((st = check_heads(config->query_heads, config->kv_heads, config->head_dim)) != MI_OK) return st;
  return check_out(q, out, "attention output");
}

float scale_log2(uint32_t head_dim) { return (1.0f / std::sqrt((float)head_dim)) * 1.4426950408889634f; }

mi_status decode_paged(mi_batch *batch, const mi_tensor *q, const mi_tensor *key_pages, const mi_tensor *value_pages,
                       const mi_tensor *block_table, const mi_tensor *lengths, const mi_attention_config *config,
                       const mi_tensor *out) {
  if (q == nullptr || key_pages == nullptr || value_pages == nullptr || block_table == nullptr || lengths == nullptr ||
      config == nullptr || out == nullptr)
    return fail(MI_ERR_INVALID_ARGUMENT, "null tensor or config");
  mi_status st;
  if ((st = check_query(q, config, out)) != MI_OK) return st;
  kernels::PagedDecodeParams p{};
  if ((st = check_paged(key_pages, value_pages, block_table, lengths, q->shape[0], config->kv_heads,
                        config->head_dim, &p.kv)) != MI_OK)
    return st;
  p.q = static_cast<const uint16_t *>(q->data), p.q_seq = q->stride[0], p.q_head = q->stride[1];
  p.out = static_cast<uint16_t *>(out->data), p.o_seq = out->stride[0], p.o_head = out->stride[1];
  p.batch = (uint32_t)q->shape[0], p.q_heads = config->query_heads, p.kv_heads = config->kv_heads;
  p.group = p.q_heads / p.kv_heads;
  p.head_chunks = (p.group + kernels::kDecodeRows - 1) / kernels::kDecodeRows;
  p.chunk = (p.group + p.head_chunks - 1) / p.head_chunks;
  p.scale_log2 = scale_log2(config->head_dim);
  // As many sequences a launch as its limits take (512 of 8 KV heads), which fill the
  // chip by themselves.
  const uint64_t upb = (uint64_t)p.kv_heads * p.head_chunks;
  const uint64_t most_tiles = ((uint64_t)p.kv.table_width << p.kv.page_shift) / kDecodeTileKeys + 1;
  if (upb > kernels::kPagedMaxUnits || upb * most_tiles >= kRows31)
    return fail(MI_ERR_SHAPE, "attention grid exceeds the launch limits");
  if ((st = check_batch(batch)) != MI_OK || q->shape[0] == 0) return st;
  Context *ctx = batch->ctx;
  const uint32_t step = (uint32_t)std::min<uint64_t>(
      {kernels::kPagedMaxBatch, kernels::kPagedMaxUnits / upb, (kRows31 - 1) / (upb * most_tiles), p.batch});
  p.workgroups = kernels::paged_decode_workgroups(ctx->compute_units);
  if (p.workgroups + kernels::kPagedMaxUnits > ctx->split_counter_count)
    return fail(MI_ERR_RESOURCE, "too few split counters");
  p.step_counters = ctx->split_counters;
  p.counters = ctx->split_counters + p.workgroups;
  p.counter_stride = kernels::counter_stride(step * upb, ctx->split_counter_count - p.workgroups);
  void *scratch = nullptr;
  const uint64_t floats =
      kernels::paged_decode_partial_floats(step * upb, p.workgroups, p.chunk, config->head_dim);
  if ((st = scratch_alloc(batch, floats * sizeof(float), &scratch)) != MI_OK) return st;
  p.partial = static_cast<float *>(scratch);
  for (uint32_t first = 0; first < (uint32_t)q->shape[0] && st == MI_OK; first += step) {
    kernels::PagedDecodeParams part = p;
    part.batch = std::min(step, p.batch - first);
    part.q += first * p.q_seq, part.out += first * p.o_seq;
    part.kv.table += first * p.kv.table_seq, part.kv.lengths += first;
    st = launch(batch, "attn_decode_paged", [&](const kernels::Launch &s) {
      return kernels::launch_paged_decode(part, config->head_dim, s);
    });
  }
  // In-order execution makes the range reusable by later work of the batch.
  scratch_free(ctx, scratch);
  return st;
}

// Packed rows over their own K and V rows (block_table null) or over pages.
mi_status packed(mi_batch *batch, const mi_tensor *q, const mi_tensor *key, const mi_tensor *value,
                 const mi_tensor *block_table, const mi_tensor *lengths, const mi_tensor *row_starts,
                 const mi_attention_config *config, const mi_tensor *out, bool paged) {
  if (q == nullptr || key == nullptr || value == nullptr || row_starts == nullptr || config == nullptr ||
      out == nullptr || (paged && (block_table == nullptr || lengths == nullptr)))
    return fail(MI_ERR_INVALID_ARGUMENT, "null tensor or config");
  mi_status st;
  if ((st = check_query(q, config, out)) != MI_OK) return st;
  if (row_starts->rank == 1 && row_starts->shape[0] < 1)
    return fail(MI_ERR_SHAPE, "row starts must have one entry more than sequences");
  const int64_t sequences = row_starts->rank == 1 ? row_starts->shape[0] - 1 : 0;
  if ((st = check_words(row_starts, sequences + 1, "row starts")) != MI_OK) return st;
  if ((uint64_t)sequences >= kRows31) return fail(MI_ERR_SHAPE, "sequences do not fit in u32");
  kernels::PackedParams p{};
  if (paged) {
    if ((st = check_paged(key, value, block_table, lengths, sequences, config->kv_heads, config->head_dim, &p.kv)) !=
        MI_OK)
      return st;
  } else {
    if ((st = check_rows(key, 3, "key")) != MI_OK || (st = check_rows(value, 3, "value")) != MI_OK) return st;
    for (const mi_tensor *t : {key, value}) {
      if (t->shape[0] != q->shape[0] || t->shape[1] != (int64_t)config->kv_heads || t->shape[2] != q->shape[2])
        return fail(MI_ERR_SHAPE, "attention tensor shapes do not match config");
      if (t->shape[0] > 1 && !rows_fit(t->stride[0], kernels::kPrefillBlockN))
        return fail(MI_ERR_SHAPE, "packed keys and values need a row stride that is not negative and 64 rows within 2 GiB");
    }
    p.kv.k = static_cast<const uint16_t *>(key->data), p.kv.k_pos = key->stride[0], p.kv.k_head = key->stride[1];
    p.kv.v = static_cast<const uint16_t *>(value->data), p.kv.v_pos = value->stride[0], p.kv.v_head = value->stride[1];
  }
  p.q = static_cast<const uint16_t *>(q->data), p.q_tok = q->stride[0], p.q_head = q->stride[1];
  p.out = static_cast<uint16_t *>(out->data), p.o_tok = out->stride[0], p.o_head = out->stride[1];
  p.row_starts = static_cast<const uint32_t *>(row_starts->data);
  p.rows = (uint32_t)q->shape[0], p.batch = (uint32_t)sequences;
  p.q_heads = config->query_heads, p.kv_heads = config->kv_heads;
  p.group = kernels::divisor(p.q_heads / p.kv_heads);
  p.heads_apart = kernels::divisor(p.kv_heads % 8 == 0 ? p.kv_heads / 8 : p.kv_heads);
  p.causal = config->causal != 0 ? 1 : 0;
  p.scale_log2 = scale_log2(config->head_dim);
  // Sequences beyond one launch's go in launches of their own, each with room for all rows.
  const uint32_t step = std::min(p.batch, kernels::kPackedMaxBatch);
  const uint64_t tiles = kernels::packed_row_tiles(p.rows, step, p.group.value);
  if ((uint64_t)p.rows * p.group.value + kernels::kPrefillBlockM >= kRows31 || tiles * p.kv_heads + kernels::kSplitCounters >= kRows31)
    return fail(MI_ERR_SHAPE, "attention grid exceeds the launch limits");
  if ((st = check_batch(batch)) != MI_OK || q->shape[0] == 0 || sequences == 0) return st;
  p.row_tiles = (uint32_t)tiles;
  // Twice the workgroups that run at once: an even share each, and a last piece per tile;
  // no more than the call's rows and keys can be cut into, and none where the KV heads alone
  // fill the chip.
  Context *ctx = batch->ctx;
  const uint32_t workgroups = kernels::packed_workgroups(ctx->compute_units, config->head_dim);
  p.share = std::max(1u, workgroups / p.kv_heads);
  const uint64_t keys = paged ? (uint64_t)p.kv.table_width << p.kv.page_shift : p.rows;
  p.max_pieces = (uint32_t)std::min<uint64_t>(2 * p.share, kernels::packed_pieces(keys, tiles, config->head_dim));
  if (p.kv_heads > workgroups || (uint64_t)2 * p.max_pieces * p.kv_heads > ctx->split_counter_count) p.max_pieces = 0;
  p.counters = ctx->split_counters;
  p.counter_stride = kernels::counter_stride((uint64_t)2 * p.max_pieces * p.kv_heads, ctx->split_counter_count);
  void *scratch = nullptr;
  if (p.max_pieces != 0) {
    const uint64_t floats = kernels::packed_partial_floats(p.max_pieces, p.kv_heads, config->head_dim);
    if ((st = scratch_alloc(batch, floats * sizeof(float), &scratch)) != MI_OK) return st;
  }
  p.partial = static_cast<float *>(scratch);
  for (uint32_t first = 0; first < (uint32_t)sequences && st == MI_OK; first += step) {
    kernels::PackedParams part = p;
    part.batch = std::min(step, p.batch - first);
    part.row_starts += first;
    if (paged) part.kv.table += first * p.kv.table_seq, part.kv.lengths += first;
    st = launch(batch, paged ? "attn_paged" : "attn_packed",
                [&](const kernels::Launch &s) { return kernels::launch_packed(part, config->head_dim, s); });
  }
  // In-order execution makes the range reusable by later work of the batch.
  if (scratch != nullptr) scratch_free(ctx, scratch);
  return st;
}

mi_status append_paged(mi_batch *batch, const mi_tensor *q, const mi_tensor *k, const mi_tensor *value,
                       const mi_tensor *q_weight, const mi_tensor *k_weight, const mi_tensor *key_pages,
                       const mi_tensor *value_pages, const mi_tensor *block_table, const mi_tensor *lengths,
                       const mi_tensor *row_starts, const mi_qk_norm_rope_cache_config *config,
                       const mi_tensor *q_out) {
  if (q == nullptr || k == nullptr || value == nullptr || key_pages == nullptr || value_pages == nullptr ||
      block_table == nullptr || lengths == nullptr || config == nullptr || q_out == nullptr)
    return fail(MI_ERR_INVALID_ARGUMENT, "null tensor or config");
  if ((q_weight == nullptr) != (k_weight == nullptr))
    return fail(MI_ERR_INVALID_ARGUMENT, "the norm needs both weights, or none");
  mi_status st;
  if ((st = check_rows(q, 3, "query")) != MI_OK || (st = check_rows(k, 3, "key")) != MI_OK ||
      (st = check_rows(value, 3, "value")) != MI_OK || (st = check_out(q, q_out, "Q/K transform output")) != MI_OK)
    return st;
  if (k->shape[0] != q->shape[0] || k->shape[2] != q->shape[2])
    return fail(MI_ERR_SHAPE, "Q/K transform tensor shapes are incompatible");
  for (int i = 0; i < 3; ++i)
    if (value->shape[i] != k->shape[i]) return fail(MI_ERR_SHAPE, "value rows must have the key's shape");
  if ((st = check_heads((uint64_t)q->shape[1], (uint64_t)k->shape[1], (uint64_t)q->shape[2])) != MI_OK) return st;
  for (const mi_tensor *w : {q_weight, k_weight}) {
    if (w == nullptr) continue;
    if ((st = check_rows(w, 1, "norm weight")) != MI_OK) return st;
    if (w->shape[0] != q->shape[2]) return fail(MI_ERR_SHAPE, "Q/K transform tensor shapes are incompatible");
  }
  if (!(config->theta > 0.0f) || std::isinf(config->theta))
    return fail(MI_ERR_SHAPE, "Q/K transform needs a positive theta");
  int64_t sequences = q->shape[0];
  if (row_starts != nullptr) {
    if (row_starts->rank == 1 && row_starts->shape[0] < 1)
      return fail(MI_ERR_SHAPE, "row starts must have one entry more than sequences");
    sequences = row_starts->rank == 1 ? row_starts->shape[0] - 1 : 0;
    if ((st = check_words(row_starts, sequences + 1, "row starts")) != MI_OK) return st;
    if ((uint64_t)sequences >= kRows31) return fail(MI_ERR_SHAPE, "sequences do not fit in u32");
  }
  kernels::PagedAppendParams p{};
  if ((st = check_paged(key_pages, value_pages, block_table, lengths, sequences, k->shape[1], k->shape[2], &p.kv)) !=
      MI_OK)
    return st;
  p.q = static_cast<const uint16_t *>(q->data), p.q_tok = q->stride[0], p.q_head = q->stride[1];
  p.k = static_cast<const uint16_t *>(k->data), p.k_tok = k->stride[0], p.k_head = k->stride[1];
  p.v = static_cast<const uint16_t *>(value->data), p.v_tok = value->stride[0], p.v_head = value->stride[1];
  if (q_weight != nullptr) {
    p.q_weight = static_cast<const uint16_t *>(q_weight->data);
    p.k_weight = static_cast<const uint16_t *>(k_weight->data);
  }
  p.q_out = static_cast<uint16_t *>(q_out->data), p.qo_tok = q_out->stride[0], p.qo_head = q_out->stride[1];
  p.key_pages = static_cast<uint16_t *>(key_pages->data);
  p.value_pages = static_cast<uint16_t *>(value_pages->data);
  p.row_starts = row_starts != nullptr ? static_cast<const uint32_t *>(row_starts->data) : nullptr;
  p.rows = (uint32_t)q->shape[0], p.batch = (uint32_t)sequences;
  p.q_heads = (uint32_t)q->shape[1], p.kv_heads = (uint32_t)k->shape[1];
  p.epsilon = config->epsilon;
  p.log2_theta = std::log2((double)config->theta);
  if ((uint64_t)p.rows * (p.q_heads + 2ull * p.kv_heads) >= kRows31)
    return fail(MI_ERR_SHAPE, "Q/K transform grid exceeds the launch limits");
  if ((st = check_batch(batch)) != MI_OK || q->shape[0] == 0 || sequences == 0) return st;
  return launch(batch, "qk_norm_rope_paged", [&](const kernels::Launch &s) {
    return kernels::launch_paged_append(p, (uint32_t)q->shape[2], s);
  });
}

// No C++ exception leaves the C ABI, and the call runs on its batch's device whatever
// device the caller has made current since the batch began.
template <typename Fn>
mi_status entry(mi_batch *batch, Fn &&fn) {
  try {
    if (batch != nullptr) hipSetDevice(batch->ctx->device);
    return fn();
  } catch (const std::exception &) {
    return MI_ERR_RESOURCE;
  }
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

mi_status mi_qk_norm_rope_paged(mi_batch *batch, const mi_tensor *q, const mi_tensor *k, const mi_tensor *value,
                                const mi_tensor *q_weight, const mi_tensor *k_weight, const mi_tensor *key_pages,
                                const mi_tensor *value_pages, const mi_tensor *block_table, const mi_tensor *lengths,
                                const mi_tensor *row_starts, const mi_qk_norm_rope_cache_config *config,
                                const mi_tensor *q_out) {
  return entry(batch, [&] {
    return append_paged(batch, q, k, value, q_weight, k_weight, key_pages, value_pages, block_table, lengths,
                        row_starts, config, q_out);
  });
}

mi_status mi_attention_decode_paged(mi_batch *batch, const mi_tensor *q, const mi_tensor *key_pages,
                                    const mi_tensor *value_pages, const mi_tensor *block_table,
                                    const mi_tensor *lengths, const mi_attention_config *config,
                                    const mi_tensor *out) {
  return entry(batch, [&] { return decode_paged(batch, q, key_pages, value_pages, block_table, lengths, config, out); });
}

mi_status mi_attention_packed(mi_batch *batch, const mi_tensor *q, const mi_tensor *k, const mi_tensor *v,
                              const mi_tensor *row_starts, const mi_attention_config *config, const mi_tensor *out) {
  return entry(batch,
               [&] { return packed(batch, q, k, v, nullptr, nullptr, row_starts, config, out, false); });
}

mi_status mi_attention_paged(mi_batch *batch, const mi_tensor *q, const mi_tensor *key_pages,
                             const mi_tensor *value_pages, const mi_tensor *block_table, const mi_tensor *lengths,
                             const mi_tensor *row_starts, const mi_attention_config *config, const mi_tensor *out) {
  return entry(batch, [&] {
    return packed(batch, q, key_pages, value_pages, block_table, lengths, row_starts, config, out, true);
  });
}

}  // extern "C"
