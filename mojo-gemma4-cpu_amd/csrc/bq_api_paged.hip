// bq_api_paged.hip -- the extern "C" boundary of the paged 16-bit cache and of
// beam selection (include/bq_api.h): argument checks, then launches on the
// caller's stream.
#include <stdarg.h>

#include <atomic>
#include <chrono>

#include "../../include/bq_api.h"
#include "bq_kernels.hpp"
#include "bq_pages.hpp"

namespace {

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  bq::api_failv(code, fmt, ap);
  va_end(ap);
  return code;
}

int check_hip(hipError_t e, const char* what) {
  return e == hipSuccess ? BQ_OK : fail(BQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline bool half_type(int d) { return d == BQ_DT_BF16 || d == BQ_DT_F16; }
inline bool hd_ok(int hd) { return hd == 64 || hd == 128 || hd == 256 || hd == 512; }

// the shapes that every user of a page table has in common
int table_args(const char* who, int num_seqs, int max_pages, int page_shift) {
  if (num_seqs <= 0 || max_pages <= 0)
    return fail(BQ_ERR_SHAPE, "%s: need num_seqs and max_pages > 0", who);
  if (page_shift < 0 || page_shift > bq::kMaxPageShift)
    return fail(BQ_ERR_UNSUPPORTED, "%s: page_shift %d not in [0, %d]", who, page_shift,
                bq::kMaxPageShift);
  return BQ_OK;
}

int pool_args(const char* who, const bq_cache_array* arrays, int num_arrays,
              const int32_t* base_rows, const int32_t* refs, const int32_t* info, int num_seqs,
              int max_pages, int page_shift, int num_pages, const void* workspace,
              size_t workspace_bytes, size_t need, bq::CacheArrays& out) {
  if (!base_rows || !refs || !info || !workspace || (num_arrays > 0 && !arrays))
    return fail(BQ_ERR_INVALID, "%s: null pointer", who);
  const int r = table_args(who, num_seqs, max_pages, page_shift);
  if (r != BQ_OK) return r;
  if (num_arrays < 0 || num_pages <= 0)
    return fail(BQ_ERR_SHAPE, "%s: need num_pages > 0 and num_arrays >= 0", who);
  if (num_seqs > bq::kMaxCacheSeqs || num_arrays > bq::kMaxCacheArrays)
    return fail(BQ_ERR_UNSUPPORTED, "%s: num_seqs %d > %d or num_arrays %d > %d", who, num_seqs,
                bq::kMaxCacheSeqs, num_arrays, bq::kMaxCacheArrays);
  if (((int64_t)num_pages << page_shift) > INT32_MAX ||
      (int64_t)num_seqs * max_pages > INT32_MAX)
    return fail(BQ_ERR_UNSUPPORTED, "%s: %d pages of 2^%d rows or %d x %d entries pass 2^31 - 1",
                who, num_pages, page_shift, num_seqs, max_pages);
  if (!aligned(workspace, 16))
    return fail(BQ_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  if (workspace_bytes < need)
    return fail(BQ_ERR_SHAPE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
  out = bq::CacheArrays{};
  out.n = num_arrays;
  for (int i = 0; i < num_arrays; ++i) {
    if (!arrays[i].data) return fail(BQ_ERR_INVALID, "%s: array %d is null", who, i);
    if (arrays[i].row_bytes <= 0 || arrays[i].row_bytes > (1 << 24))
      return fail(BQ_ERR_SHAPE, "%s: array %d has rows of %lld bytes (1 to 2^24)", who, i,
                  (long long)arrays[i].row_bytes);
    out.data[i] = arrays[i].data;
    out.row_bytes[i] = arrays[i].row_bytes;
  }
  return BQ_OK;
}

}  // namespace

namespace bq {

// A number that no other launch of this process has, and that memory does not hold by
// chance: a mixed count from a start of the clock's and the address space's choosing.
uint64_t launch_tag() {
  static std::atomic<uint64_t> count{
      (uint64_t)std::chrono::system_clock::now().time_since_epoch().count() * 0xD1342543DE82EF95ull ^
      reinterpret_cast<uintptr_t>(&launch_tag) << 16};
  uint64_t x;
  do {
    x = count.fetch_add(1, std::memory_order_relaxed) + 0x9E3779B97F4A7C15ull;
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    x ^= x >> 31;
  } while (x == 0);
  return x;
}

}  // namespace bq

extern "C" {

int bq_rope_append(const void* q, const void* k, const void* v, int64_t q_stride,
                   int64_t k_stride, int64_t v_stride, const void* q_norm, const void* k_norm,
                   int norm_v, float sqrt_n, float n_eps, const float* inv_freq, int rope_half,
                   int pair_stride, float mscale, const int32_t* positions,
                   const int32_t* seq_ids, const int32_t* base_rows, int num_seqs, int max_pages,
                   int page_shift, int64_t num_slots, void* q_out, int64_t q_out_stride,
                   void* k_cache, void* v_cache, int num_q, int num_kv, int head_dim, int dtype,
                   int num_tokens, void* stream) {
  if (num_tokens <= 0) return BQ_OK;
  if (!q || !k || !v || !positions || !base_rows || !q_out || !k_cache || !v_cache ||
      (rope_half > 0 && !inv_freq))
    return fail(BQ_ERR_INVALID, "bq_rope_append: null pointer");
  if (!half_type(dtype)) return fail(BQ_ERR_INVALID, "bq_rope_append: dtype must be bf16 or f16");
  const int r = table_args("bq_rope_append", num_seqs, max_pages, page_shift);
  if (r != BQ_OK) return r;
  if (!hd_ok(head_dim) || num_q <= 0 || num_kv <= 0 || num_slots < 0)
    return fail(BQ_ERR_SHAPE, "bq_rope_append: need head_dim in {64,128,256,512}, num_q, num_kv > "
                              "0, num_slots >= 0");
  if (!seq_ids && num_tokens > num_seqs)
    return fail(BQ_ERR_SHAPE, "bq_rope_append: %d tokens of %d sequences need seq_ids", num_tokens,
                num_seqs);
  if (num_q > (1 << 16) || num_kv > (1 << 16))
    return fail(BQ_ERR_UNSUPPORTED, "bq_rope_append: more than 2^16 heads");
  if (pair_stride < 0 || rope_half < 0 ||
      (pair_stride == 0 ? rope_half % 4 != 0 || 2 * (int64_t)rope_half > head_dim
                        : rope_half % 8 != 0 || pair_stride % 8 != 0 || rope_half > pair_stride ||
                              (int64_t)pair_stride + rope_half > head_dim))
    return fail(BQ_ERR_SHAPE, "bq_rope_append: rope_half %d and pair_stride %d do not fit head_dim "
                              "%d (halves: multiples of 8; neighbours: rope_half %% 4 == 0)",
                rope_half, pair_stride, head_dim);
  const int64_t qw = (int64_t)num_q * head_dim, kw = (int64_t)num_kv * head_dim;
  if (q_stride < qw || q_out_stride < qw || k_stride < kw || v_stride < kw || q_stride % 8 ||
      q_out_stride % 8 || k_stride % 8 || v_stride % 8)
    return fail(BQ_ERR_SHAPE, "bq_rope_append: row strides must cover the heads and be multiples "
                              "of 8");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) ||
      !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(q_norm, 16) ||
      !aligned(k_norm, 16))
    return fail(BQ_ERR_INVALID, "bq_rope_append: 16-bit tensors must be 16-byte aligned");
  bq::RopeArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.q_norm = static_cast<const uint16_t*>(q_norm);
  a.k_norm = static_cast<const uint16_t*>(k_norm);
  a.norm_v = norm_v;
  a.sqrt_n = sqrt_n, a.n_eps = n_eps, a.mscale = mscale;
  a.inv_freq = inv_freq;
  a.rope_half = rope_half, a.pair_stride = pair_stride;
  a.positions = positions, a.seq_ids = seq_ids, a.base_rows = base_rows;
  a.num_seqs = num_seqs, a.max_pages = max_pages, a.page_shift = page_shift;
  a.num_slots = num_slots;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.q_out_stride = q_out_stride;
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.num_q = num_q, a.num_kv = num_kv, a.num_tokens = num_tokens;
  return check_hip(bq::launch_rope_append(a, head_dim, dtype == BQ_DT_F16, S(stream)),
                   "rope_append");
}

int bq_paged_attention_splits(int num_seqs, int num_q, int num_kv, int head_dim, int max_kv_len,
                              int window) {
  if (num_seqs <= 0 || num_q <= 0 || num_kv <= 0 || max_kv_len <= 0) return 1;
  return bq::paged_attn_splits(num_seqs, num_q, num_kv, head_dim, max_kv_len, window);
}

size_t bq_paged_attention_workspace_size(int num_seqs, int num_q, int head_dim, int s_max) {
  if (num_seqs <= 0 || num_q <= 0 || head_dim <= 0 || s_max <= 1) return 0;
  return (size_t)num_seqs * num_q * s_max * ((size_t)head_dim + 4) * sizeof(float);
}

int bq_paged_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                       int64_t num_slots, const int32_t* base_rows, int max_pages, int page_shift,
                       const int32_t* kv_lens, void* out, float* lse, int num_seqs, int num_q,
                       int num_kv, int head_dim, int window, float scale, float softcap, int dtype,
                       int s_max, void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs <= 0) return BQ_OK;
  if (!q || !k_cache || !v_cache || !base_rows || !kv_lens || !out || (s_max > 1 && !workspace))
    return fail(BQ_ERR_INVALID, "bq_paged_attention: null pointer");
  if (!half_type(dtype))
    return fail(BQ_ERR_INVALID, "bq_paged_attention: dtype must be bf16 or f16");
  const int r = table_args("bq_paged_attention", num_seqs, max_pages, page_shift);
  if (r != BQ_OK) return r;
  if (!hd_ok(head_dim) || num_q <= 0 || num_kv <= 0 || num_q % num_kv || num_slots <= 0)
    return fail(BQ_ERR_SHAPE, "bq_paged_attention: need head_dim in {64,128,256,512}, num_q %% "
                              "num_kv == 0, num_slots > 0");
  if (window < 0 || s_max < 1)
    return fail(BQ_ERR_SHAPE, "bq_paged_attention: need window >= 0, s_max >= 1");
  if (s_max > 256 || num_q > (1 << 16))
    return fail(BQ_ERR_UNSUPPORTED, "bq_paged_attention: s_max %d > 256 or more than 2^16 heads", s_max);
  if (!(softcap >= 0.0f) || !(scale == scale))
    return fail(BQ_ERR_SHAPE, "bq_paged_attention: softcap must be >= 0 and scale a number");
  if (q_stride < (int64_t)num_q * head_dim || q_stride % 8)
    return fail(BQ_ERR_SHAPE, "bq_paged_attention: q_stride must cover the heads and be a multiple "
                              "of 8");
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) ||
      !aligned(workspace, 16))
    return fail(BQ_ERR_INVALID, "bq_paged_attention: q, caches, out and workspace must be 16-byte "
                                "aligned");
  const size_t need = bq_paged_attention_workspace_size(num_seqs, num_q, head_dim, s_max);
  if (workspace_bytes < need)
    return fail(BQ_ERR_SHAPE, "bq_paged_attention: workspace %zu < %zu bytes", workspace_bytes, need);
  constexpr float kLog2e = 1.4426950408889634f;
  bq::PagedAttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride, a.num_slots = num_slots;
  a.k_cache = static_cast<const uint16_t*>(k_cache);
  a.v_cache = static_cast<const uint16_t*>(v_cache);
  a.base_rows = base_rows, a.kv_lens = kv_lens;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.ws_acc = static_cast<float*>(workspace);
  a.ws_ml = a.ws_acc ? a.ws_acc + (size_t)num_seqs * num_q * s_max * head_dim : nullptr;
  a.num_seqs = num_seqs, a.num_q = num_q, a.num_kv = num_kv, a.gqa = num_q / num_kv;
  a.head_groups = (a.gqa + 15) / 16;
  a.max_pages = max_pages, a.page_shift = page_shift, a.window = window, a.s_max = s_max;
  a.scale2 = softcap > 0.0f ? scale : scale * kLog2e;
  a.softcap2 = softcap * kLog2e;
  a.inv_cap = softcap > 0.0f ? 2.0f * kLog2e / softcap : 0.0f;
  return check_hip(bq::launch_paged_attn(a, head_dim, dtype == BQ_DT_F16, S(stream)),
                   "paged_attention");
}

size_t bq_cache_reorder_workspace_size(int num_seqs) {
  return num_seqs > 0 ? bq::reorder_workspace(num_seqs) : 0;
}

int bq_cache_reorder(const bq_cache_array* arrays, int num_arrays, int32_t* base_rows,
                     int32_t* lens, int32_t* refs, const int32_t* parents, const int32_t* grow,
                     int num_seqs, int max_pages, int page_shift, int num_pages, int32_t* info,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs <= 0) return BQ_OK;
  if (!lens || !parents) return fail(BQ_ERR_INVALID, "bq_cache_reorder: null pointer");
  bq::CacheArrays c;
  const int r = pool_args("bq_cache_reorder", arrays, num_arrays, base_rows, refs, info, num_seqs,
                          max_pages, page_shift, num_pages, workspace, workspace_bytes,
                          bq_cache_reorder_workspace_size(num_seqs), c);
  if (r != BQ_OK) return r;
  bq::ReorderArgs a{};
  a.base_rows = base_rows, a.lens = lens, a.refs = refs, a.parents = parents, a.grow = grow;
  a.info = info, a.workspace = workspace;
  a.num_seqs = num_seqs, a.max_pages = max_pages, a.page_shift = page_shift;
  a.num_pages = num_pages;
  return check_hip(bq::launch_cache_reorder(a, c, S(stream)), "cache_reorder");
}

size_t bq_cache_compact_workspace_size(int num_pages) {
  return num_pages > 0 ? bq::compact_workspace(num_pages) : 0;
}

int bq_cache_compact(const bq_cache_array* arrays, int num_arrays, int32_t* base_rows,
                     int32_t* refs, int num_seqs, int max_pages, int page_shift, int num_pages,
                     int32_t* info, void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs <= 0) return BQ_OK;
  bq::CacheArrays c;
  const int r = pool_args("bq_cache_compact", arrays, num_arrays, base_rows, refs, info, num_seqs,
                          max_pages, page_shift, num_pages, workspace, workspace_bytes,
                          bq_cache_compact_workspace_size(num_pages), c);
  if (r != BQ_OK) return r;
  bq::CompactArgs a{};
  a.base_rows = base_rows, a.refs = refs, a.info = info, a.workspace = workspace;
  a.num_seqs = num_seqs, a.max_pages = max_pages, a.page_shift = page_shift;
  a.num_pages = num_pages;
  return check_hip(bq::launch_cache_compact(a, c, S(stream)), "cache_compact");
}

size_t bq_beam_select_workspace_size(int rows, int vocab) {
  return rows > 0 && vocab > 0 ? bq::beam_workspace(rows, vocab) : 0;
}

int bq_beam_select(const void* logits, int64_t row_stride, int dtype, const float* scores,
                   const uint8_t* finished, int batch, int beams, int vocab, int n, int eos_id,
                   float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                   uint8_t* out_finished, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch <= 0) return BQ_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace)
    return fail(BQ_ERR_INVALID, "bq_beam_select: null pointer");
  if (!half_type(dtype) && dtype != BQ_DT_F32)
    return fail(BQ_ERR_INVALID, "bq_beam_select: dtype must be bf16, f16 or f32");
  if (beams <= 0 || vocab <= 0 || n <= 0 || row_stride < vocab)
    return fail(BQ_ERR_SHAPE, "bq_beam_select: need beams, vocab, n > 0 and row_stride >= vocab");
  if (beams > bq::kMaxBeams || n > bq::kMaxPicks || vocab > (1 << 20) ||
      (int64_t)batch * beams > (1 << 20))
    return fail(BQ_ERR_UNSUPPORTED, "bq_beam_select: beams %d or n %d > 64, vocab %d or batch * "
                                    "beams > 2^20", beams, n, vocab);
  if (eos_id < -1 || eos_id >= vocab || (finished && eos_id < 0))
    return fail(BQ_ERR_SHAPE, "bq_beam_select: eos_id %d outside [-1, vocab), or -1 with finished "
                              "beams", eos_id);
  if (out_scores == scores || (finished && out_finished == finished))
    return fail(BQ_ERR_INVALID, "bq_beam_select: outputs may not be the inputs");
  const int size = dtype == BQ_DT_F32 ? 4 : 2;
  if (!aligned(logits, size) || !aligned(workspace, 16))
    return fail(BQ_ERR_INVALID, "bq_beam_select: logits must be aligned to their type, workspace "
                                "to 16 bytes");
  const size_t need = bq_beam_select_workspace_size(batch * beams, vocab);
  if (workspace_bytes < need)
    return fail(BQ_ERR_SHAPE, "bq_beam_select: workspace %zu < %zu bytes", workspace_bytes, need);
  bq::BeamArgs a{};
  a.logits = logits, a.row_stride = row_stride, a.scores = scores, a.finished = finished;
  a.out_scores = out_scores, a.out_parents = out_parents, a.out_tokens = out_tokens;
  a.out_finished = out_finished, a.workspace = workspace;
  a.batch = batch, a.beams = beams, a.vocab = vocab, a.n = n, a.eos_id = eos_id;
  return check_hip(bq::launch_beam_select(a, size, dtype == BQ_DT_F16, S(stream)), "beam_select");
}

}  // extern "C"
