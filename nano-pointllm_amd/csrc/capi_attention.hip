// extern "C" entry points of the attention core (declared in
// include/w8a8_gfx950.h): argument checks and dispatch.  The kernels live in
// rotary.hip, attention_decode.hip, attention_prefill.h and cache_accept.hip.
#include <algorithm>
#include <utility>

#include "w8a8_gfx950.h"
#include "w8a8_internal.h"

using namespace w8a8;

namespace {

using i128 = __int128;

inline bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline bool half_dtype(int d) { return d == kF16 || d == kBF16; }

constexpr int64_t kMaxTokens = INT32_MAX - 4096;
constexpr int64_t kMaxHeads = 4096;
// Workgroups of 256 threads; a launch's threads are counted in 32 bits.
constexpr int64_t kMaxBlocks = UINT32_MAX / 256;
constexpr int64_t kMaxGridYZ = 65535;
constexpr int64_t kMaxStride = int64_t{1} << 60;
constexpr i128 kMaxBytes = i128(1) << 62;  // of any tensor's address range

// 16-bit rows [tokens, heads, dim], strides in elements.
struct Rows {
  const void* p;
  int64_t st, sh, tokens, heads, dim;
};

inline bool strides_ok(int64_t a, int64_t b) {
  return a >= 0 && b >= 0 && a <= kMaxStride && b <= kMaxStride;
}

// Whether no two rows share an element (what an output needs).
inline bool distinct(const Rows& r) {
  const bool many_t = r.tokens > 1, many_h = r.heads > 1;
  if (many_t && many_h) {
    const i128 head_span = i128(r.heads - 1) * r.sh + r.dim;
    const i128 token_span = i128(r.tokens - 1) * r.st + r.dim;
    return (r.sh >= r.dim && r.st >= head_span) || (r.st >= r.dim && r.sh >= token_span);
  }
  return (!many_t || r.st >= r.dim) && (!many_h || r.sh >= r.dim);
}

inline i128 begin_of(const Rows& r) { return i128(reinterpret_cast<uintptr_t>(r.p)); }
inline i128 bytes_of(const Rows& r) {
  return 2 * (i128(r.tokens - 1) * r.st + i128(r.heads - 1) * r.sh + r.dim);
}

// Whether the rows share no byte: their address ranges are apart, or they are
// column ranges of one matrix (equal token strides, and the heads of each
// inside one row of it).
inline bool apart(const Rows& a, const Rows& b) {
  if (a.p == nullptr || b.p == nullptr) return true;
  const i128 a0 = begin_of(a), b0 = begin_of(b);
  if (a0 + bytes_of(a) <= b0 || b0 + bytes_of(b) <= a0) return true;
  if (a.st != b.st || a.st == 0) return false;
  const i128 st = 2 * i128(a.st);
  const i128 wa = 2 * (i128(a.heads - 1) * a.sh + a.dim);
  const i128 wb = 2 * (i128(b.heads - 1) * b.sh + b.dim);
  const i128 off = (((b0 - a0) % st) + st) % st;  // where b's row starts inside a's
  return wa <= off && off + wb <= st;
}

// The pages [pages, heads, page, dim] of one cache tensor.
struct Cache {
  int64_t c_page, c_head, c_tok, pages, page_size, heads, dim;
};

inline i128 cache_bytes(const Cache& c) {
  return 2 * (i128(c.pages - 1) * c.c_page + i128(c.heads - 1) * c.c_head +
              i128(c.page_size - 1) * c.c_tok + c.dim);
}

// The axes of a cache, or of `layers` of them at a stride, that have more than one
// row, largest stride first.
struct Axis {
  int64_t stride, count;
  i128 inner;   // elements that the axes of smaller strides and a row span
};
struct Axes {
  Axis axis[4];
  int n;
};
inline Axes axes_of(const Cache& c, int64_t c_layer, int64_t layers) {
  Axes x{{{c_layer, layers, 0}, {c.c_page, c.pages, 0}, {c.c_head, c.heads, 0},
          {c.c_tok, c.page_size, 0}}, 4};
  x.n = static_cast<int>(std::remove_if(x.axis, x.axis + 4,
                                        [](const Axis& a) { return a.count <= 1; }) - x.axis);
  std::sort(x.axis, x.axis + x.n, [](const Axis& a, const Axis& b) { return a.stride > b.stride; });
  i128 extent = c.dim;
  for (int i = x.n - 1; i >= 0; --i) {
    x.axis[i].inner = extent;
    extent += i128(x.axis[i].count - 1) * x.axis[i].stride;
  }
  return x;
}

// Whether no two rows share an element: each stride covers the extent of the axes
// with smaller strides.
inline bool cache_distinct(const Cache& c, int64_t c_layer = 0, int64_t layers = 1) {
  const Axes x = axes_of(c, c_layer, layers);
  for (int i = 0; i < x.n; ++i)
    if (x.axis[i].stride < x.axis[i].inner) return false;
  return true;
}

inline bool clear_of(const Rows& r, const void* cache, const Cache& c) {
  if (r.p == nullptr || cache == nullptr) return true;
  const i128 a0 = begin_of(r), b0 = i128(reinterpret_cast<uintptr_t>(cache));
  return a0 + bytes_of(r) <= b0 || b0 + cache_bytes(c) <= a0;
}

// Whether a row of one cache and one of another of the same axes, `bytes` behind it,
// share an element: whether differences d of their indexes bring bytes - sum of
// 2 d stride to less than a row's length.  The strides cover what is inside them
// (cache_distinct), so on every axis only the two d around the quotient can.
inline bool rows_meet(const Axes& x, int i, i128 bytes, int64_t dim) {
  if (i == x.n) return bytes > -2 * i128(dim) && bytes < 2 * i128(dim);
  const Axis& a = x.axis[i];
  const i128 step = 2 * i128(a.stride), d0 = bytes / step - (bytes % step < 0 ? 1 : 0);
  for (i128 d = d0; d <= d0 + 1; ++d) {
    const i128 rest = bytes - d * step;
    if (d > -a.count && d < a.count && rest > -2 * a.inner && rest < 2 * a.inner &&
        rows_meet(x, i + 1, rest, dim))
      return true;
  }
  return false;
}

// Whether k and v, whose rows do not share elements among themselves, share none:
// apart, or side by side within layers, pages, heads or tokens.
inline bool caches_apart(const void* k, const void* v, const Cache& c, int64_t c_layer,
                         int64_t layers) {
  const i128 a = i128(reinterpret_cast<uintptr_t>(k)), b = i128(reinterpret_cast<uintptr_t>(v));
  return !rows_meet(axes_of(c, c_layer, layers), 0, b - a, c.dim);
}

// log2 of a power of two up to 2^20, or -1.
inline int page_shift_of(int64_t page_size) {
  for (int s = 0; s <= 20; ++s)
    if (page_size == int64_t{1} << s) return s;
  return -1;
}

int check_cache(const Cache& c, int64_t align_elems) {
  if (c.pages < 0 || c.pages > INT32_MAX) return W8A8_ERR_SHAPE;
  if (page_shift_of(c.page_size) < 0) return W8A8_ERR_SHAPE;
  if (!strides_ok(c.c_page, c.c_head) || !strides_ok(c.c_tok, 0)) return W8A8_ERR_SHAPE;
  // An offset in the cache stays below 2^62 bytes.
  if (c.pages > 0 && cache_bytes(c) > kMaxBytes) return W8A8_ERR_SHAPE;
  // The stride of an axis of one is multiplied by zero only.
  if ((c.pages > 1 && c.c_page % align_elems) || (c.heads > 1 && c.c_head % align_elems) ||
      (c.page_size > 1 && c.c_tok % align_elems))
    return W8A8_ERR_ALIGN;
  return W8A8_OK;
}

}  // namespace

extern "C" {

int w8a8_rotary(const void* x, int64_t x_stride_t, int64_t x_stride_h, int dtype,
                const int64_t* positions, const double* inv_freq, int64_t rotary_dim, int layout,
                float factor, void* y, int64_t y_stride_t, int64_t y_stride_h, int64_t tokens,
                int64_t heads, int64_t head_dim, hipStream_t stream) {
  return w8a8_rotary_store(x, x_stride_t, x_stride_h, nullptr, 0, 0, nullptr, 0, 0, dtype,
                           positions, nullptr, inv_freq, rotary_dim, layout, factor, y, y_stride_t,
                           y_stride_h, nullptr, nullptr, 0, 0, 0, 0, 1, tokens, heads, 0, head_dim,
                           stream);
}

int w8a8_rotary_store(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                      int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                      int64_t v_stride_h, int dtype, const int64_t* positions,
                      const int64_t* slots, const double* inv_freq, int64_t rotary_dim, int layout,
                      float factor, void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h,
                      void* k_cache, void* v_cache, int64_t cache_stride_page,
                      int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                      int64_t page_size, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                      int64_t head_dim, hipStream_t stream) {
  if (!half_dtype(dtype)) return W8A8_ERR_DTYPE;
  if (layout != W8A8_ROTARY_HALF && layout != W8A8_ROTARY_INTERLEAVED) return W8A8_ERR_DTYPE;
  if (tokens < 0 || tokens > kMaxBlocks || q_heads < 0 || q_heads > kMaxHeads || kv_heads < 0 ||
      kv_heads > kMaxHeads)
    return W8A8_ERR_SHAPE;
  if (head_dim <= 0 || head_dim % 8 || head_dim > kRotaryMaxDim) return W8A8_ERR_SHAPE;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2) return W8A8_ERR_SHAPE;
  if (!__builtin_isfinite(factor)) return W8A8_ERR_SHAPE;
  if (!strides_ok(q_stride_t, q_stride_h) || !strides_ok(k_stride_t, k_stride_h) ||
      !strides_ok(v_stride_t, v_stride_h) || !strides_ok(q_out_stride_t, q_out_stride_h))
    return W8A8_ERR_SHAPE;
  const Cache c{cache_stride_page, cache_stride_head, cache_stride_token, pages,
                page_size,         kv_heads,          head_dim};
  if (kv_heads > 0) {
    const int rc = check_cache(c, 1);
    if (rc != W8A8_OK) return rc;
  }
  if (tokens == 0 || q_heads + kv_heads == 0) return W8A8_OK;
  if (positions == nullptr || (rotary_dim > 0 && inv_freq == nullptr)) return W8A8_ERR_NULL;
  if (q_heads > 0 && (q == nullptr || q_out == nullptr)) return W8A8_ERR_NULL;
  for (const Rows& r : {Rows{q, q_stride_t, q_stride_h, tokens, q_heads, head_dim},
                        Rows{q_out, q_out_stride_t, q_out_stride_h, tokens, q_heads, head_dim},
                        Rows{k, k_stride_t, k_stride_h, tokens, kv_heads, head_dim},
                        Rows{v, v_stride_t, v_stride_h, tokens, kv_heads, head_dim}})
    if (bytes_of(r) > kMaxBytes) return W8A8_ERR_SHAPE;
  if (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(positions, 8) || !aligned(inv_freq, 8))
    return W8A8_ERR_ALIGN;
  const Rows qr{q_heads > 0 ? q : nullptr, q_stride_t, q_stride_h, tokens, q_heads, head_dim};
  const Rows qo{q_heads > 0 ? q_out : nullptr, q_out_stride_t, q_out_stride_h, tokens, q_heads,
                head_dim};
  if (q_heads > 0) {
    if (!distinct(qo)) return W8A8_ERR_OVERLAP;
    // In place: every element is read and written by one thread.
    const bool in_place = q == q_out && (tokens == 1 || q_stride_t == q_out_stride_t) &&
                          (q_heads == 1 || q_stride_h == q_out_stride_h);
    if (!in_place && !apart(qo, qr)) return W8A8_ERR_OVERLAP;
  }
  if (kv_heads > 0) {
    if (k == nullptr || v == nullptr || slots == nullptr) return W8A8_ERR_NULL;
    if (pages > 0 && (k_cache == nullptr || v_cache == nullptr)) return W8A8_ERR_NULL;
    if (!aligned(k, 2) || !aligned(v, 2) || !aligned(k_cache, 2) || !aligned(v_cache, 2) ||
        !aligned(slots, 8))
      return W8A8_ERR_ALIGN;
    const Rows kr{k, k_stride_t, k_stride_h, tokens, kv_heads, head_dim};
    const Rows vr{v, v_stride_t, v_stride_h, tokens, kv_heads, head_dim};
    if (!apart(qo, kr) || !apart(qo, vr)) return W8A8_ERR_OVERLAP;
    if (pages > 0) {
      if (k_cache == v_cache || !cache_distinct(c)) return W8A8_ERR_OVERLAP;
      for (const void* cache : {k_cache, v_cache})
        if (!clear_of(qr, cache, c) || !clear_of(qo, cache, c) || !clear_of(kr, cache, c) ||
            !clear_of(vr, cache, c))
          return W8A8_ERR_OVERLAP;
    }
  }
  RotaryRows r;
  r.q = q;
  r.q_st = q_stride_t;
  r.q_sh = q_stride_h;
  r.k = kv_heads > 0 ? k : nullptr;
  r.k_st = k_stride_t;
  r.k_sh = k_stride_h;
  r.v = v;
  r.v_st = v_stride_t;
  r.v_sh = v_stride_h;
  r.positions = positions;
  r.slots = slots;
  r.inv_freq = inv_freq;
  r.q_out = q_out;
  r.qo_st = q_out_stride_t;
  r.qo_sh = q_out_stride_h;
  r.k_cache = k_cache;
  r.v_cache = v_cache;
  r.c_page = cache_stride_page;
  r.c_head = cache_stride_head;
  r.c_tok = cache_stride_token;
  r.pages = pages;
  r.tokens = tokens;
  r.page_shift = kv_heads > 0 ? page_shift_of(page_size) : 0;
  r.q_heads = static_cast<int>(q_heads);
  r.kv_heads = static_cast<int>(kv_heads);
  r.head_dim = static_cast<int>(head_dim);
  r.rotary_dim = static_cast<int>(rotary_dim);
  r.half = layout == W8A8_ROTARY_HALF;
  r.factor = factor;
  return status_of(launch_rotary(r, dtype, stream));
}

}  // extern "C"

namespace {

// Whether rows and workgroups stay inside what a launch counts: of each key
// head's rows, counted in 32 bits, a workgroup takes `rows`, of one sequence; a
// cut over the keys adds at most 1024 workgroups.
bool counts_ok(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int rows) {
  if (tokens < 0 || tokens > kMaxTokens || batch < 0 || batch > kMaxTokens || q_heads <= 0 ||
      q_heads > kMaxHeads || kv_heads <= 0 || q_heads % kv_heads)
    return false;
  const int64_t group_rows = tokens * (q_heads / kv_heads);
  return group_rows <= kMaxTokens &&
         kv_heads * (group_rows / rows + batch + 1) <= kMaxBlocks - 1024;
}
constexpr int kDecodeRows = 16, kPrefillRows = 128;

// The checks that both attention entry points share; fills p but for
// q_starts and the workspace.
int check_attention(PagedAttention& p, const void* q, int64_t q_st, int64_t q_sh,
                    const void* k_cache, const void* v_cache, const Cache& c,
                    const int32_t* table, int64_t ld_table, int64_t table_pages,
                    const int32_t* lengths, int dtype, float scale, void* out, int64_t o_st,
                    int64_t o_sh, int64_t tokens, int64_t batch, int64_t q_heads, int rows) {
  if (!half_dtype(dtype)) return W8A8_ERR_DTYPE;
  if (!counts_ok(tokens, batch, q_heads, c.heads, rows)) return W8A8_ERR_SHAPE;
  if (c.dim <= 0 || c.dim % 8 || c.dim > kAttentionMaxDim) return W8A8_ERR_SHAPE;
  if (!__builtin_isfinite(scale)) return W8A8_ERR_SHAPE;
  if (!strides_ok(q_st, q_sh) || !strides_ok(o_st, o_sh)) return W8A8_ERR_SHAPE;
  const int rc = check_cache(c, 8);
  if (rc != W8A8_OK) return rc;
  if (table_pages < 0 || ld_table < table_pages || ld_table > kMaxStride ||
      table_pages > kMaxTokens / c.page_size)
    return W8A8_ERR_SHAPE;
  if (tokens == 0 || batch == 0) return W8A8_OK;
  if (q == nullptr || out == nullptr || lengths == nullptr) return W8A8_ERR_NULL;
  if (table_pages > 0 && c.pages > 0 &&
      (table == nullptr || k_cache == nullptr || v_cache == nullptr))
    return W8A8_ERR_NULL;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      !aligned(table, 4) || !aligned(lengths, 4) || (tokens > 1 && (q_st % 8 || o_st % 8)) ||
      (q_heads > 1 && (q_sh % 8 || o_sh % 8)))
    return W8A8_ERR_ALIGN;
  const Rows qr{q, q_st, q_sh, tokens, q_heads, c.dim};
  const Rows orr{out, o_st, o_sh, tokens, q_heads, c.dim};
  if (bytes_of(qr) > kMaxBytes || bytes_of(orr) > kMaxBytes || i128(batch) * ld_table > kMaxBytes)
    return W8A8_ERR_SHAPE;
  if (!distinct(orr) || !apart(orr, qr)) return W8A8_ERR_OVERLAP;
  if (c.pages > 0 && (!clear_of(orr, k_cache, c) || !clear_of(orr, v_cache, c)))
    return W8A8_ERR_OVERLAP;
  p.q = q;
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.k = k_cache;
  p.v = v_cache;
  p.c_page = c.c_page;
  p.c_head = c.c_head;
  p.c_tok = c.c_tok;
  p.pages = c.pages;
  p.table = table;
  p.ld_table = ld_table;
  p.lengths = lengths;
  p.out = out;
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.page_shift = page_shift_of(c.page_size);
  p.max_keys = c.pages > 0 ? static_cast<int>(table_pages * c.page_size) : 0;
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(tokens);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(c.heads);
  p.head_dim = static_cast<int>(c.dim);
  p.scale = scale;
  return W8A8_OK;
}

bool sizes_ok(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
              int64_t max_keys, int rows) {
  return counts_ok(tokens, batch, q_heads, kv_heads, rows) && head_dim > 0 && head_dim % 8 == 0 &&
         head_dim <= kAttentionMaxDim && max_keys >= 0 && max_keys <= kMaxTokens;
}

// What a row sees: all keys up to its own place, or of those the first `sinks`
// and the last `window`, or by the masks of a tree.
struct Sight {
  int64_t window = 0, sinks = 0;
  bool windowed = false;
  bool tree = false;
  const uint64_t* masks = nullptr;
  int64_t ld_masks = 0, words = 0;
};

// A window that no table's keys pass hides nothing, whatever the lengths.
bool window_ok(int64_t window, int64_t sinks) { return window >= 1 && sinks >= 0; }
Sight window_of(int64_t window, int64_t sinks, int64_t max_keys) {
  Sight s;
  s.windowed = window < max_keys;
  s.window = std::min(window, max_keys);
  s.sinks = std::min(sinks, max_keys);
  return s;
}

int64_t prefill_workspace(const Sight& s, int64_t tokens, int64_t batch, int64_t q_heads,
                          int64_t kv_heads, int64_t head_dim, int64_t max_keys) {
  if (s.windowed)
    return paged_prefill_window_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys,
                                          s.window, s.sinks);
  if (s.tree) return paged_tree_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
  return paged_prefill_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
}

// All prefill entry points; clear: rows of no sequence become zeros.
int paged_prefill(Sight sight, bool clear, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                  const void* k_cache, const void* v_cache, int64_t cache_stride_page,
                  int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                  int64_t page_size, const int32_t* page_table, int64_t ld_table,
                  int64_t table_pages, const int32_t* lengths, const int32_t* q_starts, int dtype,
                  float scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                  int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                  int64_t head_dim, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const Cache c{cache_stride_page, cache_stride_head, cache_stride_token, pages,
                page_size,         kv_heads,          head_dim};
  PagedAttention p;
  const int rc = check_attention(p, q, q_stride_t, q_stride_h, k_cache, v_cache, c, page_table,
                                 ld_table, table_pages, lengths, dtype, scale, out, out_stride_t,
                                 out_stride_h, tokens, batch, q_heads, kPrefillRows);
  if (rc != W8A8_OK || tokens == 0) return rc;
  // Nothing says then which rows the batch's workgroups would clear.
  if (batch == 0) return clear ? W8A8_ERR_SHAPE : W8A8_OK;
  if (q_starts == nullptr) return W8A8_ERR_NULL;
  if (!aligned(q_starts, 4)) return W8A8_ERR_ALIGN;
  if (sight.windowed) sight = window_of(sight.window, sight.sinks, p.max_keys);
  if (sight.tree) {
    if (sight.words > 0 && sight.masks == nullptr) return W8A8_ERR_NULL;
    if (!aligned(sight.masks, 8)) return W8A8_ERR_ALIGN;
    const Rows orr{out, out_stride_t, out_stride_h, tokens, q_heads, head_dim};
    const i128 m0 = i128(reinterpret_cast<uintptr_t>(sight.masks));
    const i128 m1 = m0 + 8 * (i128(tokens - 1) * sight.ld_masks + sight.words);
    if (m1 - m0 > kMaxBytes) return W8A8_ERR_SHAPE;
    if (sight.words > 0 && m0 < begin_of(orr) + bytes_of(orr) && begin_of(orr) < m1)
      return W8A8_ERR_OVERLAP;
  }
  const int64_t need =
      prefill_workspace(sight, tokens, batch, q_heads, kv_heads, head_dim, p.max_keys);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return W8A8_ERR_WORKSPACE;
  if (need > 0 && !aligned(workspace, 16)) return W8A8_ERR_ALIGN;
  p.workspace = workspace;
  p.q_starts = q_starts;
  if (sight.tree)
    return status_of(launch_paged_tree(p, sight.masks, sight.ld_masks,
                                       static_cast<int>(sight.words), clear, dtype, stream));
  if (sight.windowed)
    return status_of(launch_paged_prefill_window(p, static_cast<int>(sight.window),
                                                 static_cast<int>(sight.sinks), clear, dtype,
                                                 stream));
  return status_of(launch_paged_prefill(p, clear, dtype, stream));
}

// Both decode entry points.
int paged_decode(Sight sight, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                 const void* k_cache, const void* v_cache, int64_t cache_stride_page,
                 int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                 int64_t page_size, const int32_t* page_table, int64_t ld_table,
                 int64_t table_pages, const int32_t* lengths, int dtype, float scale, void* out,
                 int64_t out_stride_t, int64_t out_stride_h, int64_t batch, int64_t q_heads,
                 int64_t kv_heads, int64_t head_dim, void* workspace, int64_t workspace_bytes,
                 hipStream_t stream) {
  const Cache c{cache_stride_page, cache_stride_head, cache_stride_token, pages,
                page_size,         kv_heads,          head_dim};
  PagedAttention p;
  const int rc = check_attention(p, q, q_stride_t, q_stride_h, k_cache, v_cache, c, page_table,
                                 ld_table, table_pages, lengths, dtype, scale, out, out_stride_t,
                                 out_stride_h, batch, batch, q_heads, kDecodeRows);
  if (rc != W8A8_OK || batch == 0) return rc;
  if (sight.windowed) sight = window_of(sight.window, sight.sinks, p.max_keys);
  const int64_t need =
      sight.windowed ? paged_decode_window_workspace(batch, q_heads, kv_heads, head_dim,
                                                     p.max_keys, sight.window, sight.sinks)
                     : paged_decode_workspace(batch, q_heads, kv_heads, head_dim, p.max_keys);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return W8A8_ERR_WORKSPACE;
  if (need > 0 && !aligned(workspace, 16)) return W8A8_ERR_ALIGN;
  p.workspace = workspace;
  p.q_starts = nullptr;
  if (sight.windowed)
    return status_of(launch_paged_decode_window(p, static_cast<int>(sight.window),
                                                static_cast<int>(sight.sinks), dtype, stream));
  return status_of(launch_paged_decode(p, dtype, stream));
}

}  // namespace

extern "C" {

int64_t w8a8_paged_decode_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                          int64_t head_dim, int64_t max_keys) {
  if (!sizes_ok(batch, batch, q_heads, kv_heads, head_dim, max_keys, kDecodeRows)) return -1;
  return paged_decode_workspace(batch, q_heads, kv_heads, head_dim, max_keys);
}

int w8a8_paged_decode(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                      const void* v_cache, int64_t cache_stride_page, int64_t cache_stride_head,
                      int64_t cache_stride_token, int64_t pages, int64_t page_size,
                      const int32_t* page_table, int64_t ld_table, int64_t table_pages,
                      const int32_t* lengths, int dtype, float scale, void* out,
                      int64_t out_stride_t, int64_t out_stride_h, int64_t batch, int64_t q_heads,
                      int64_t kv_heads, int64_t head_dim, void* workspace,
                      int64_t workspace_bytes, hipStream_t stream) {
  return paged_decode(Sight{}, q, q_stride_t, q_stride_h, k_cache, v_cache, cache_stride_page,
                      cache_stride_head, cache_stride_token, pages, page_size, page_table,
                      ld_table, table_pages, lengths, dtype, scale, out, out_stride_t,
                      out_stride_h, batch, q_heads, kv_heads, head_dim, workspace,
                      workspace_bytes, stream);
}

int64_t w8a8_paged_prefill_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads,
                                           int64_t kv_heads, int64_t head_dim,
                                           int64_t max_keys) {
  if (!sizes_ok(tokens, batch, q_heads, kv_heads, head_dim, max_keys, kPrefillRows)) return -1;
  return paged_prefill_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
}

int w8a8_paged_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                       const void* v_cache, int64_t cache_stride_page, int64_t cache_stride_head,
                       int64_t cache_stride_token, int64_t pages, int64_t page_size,
                       const int32_t* page_table, int64_t ld_table, int64_t table_pages,
                       const int32_t* lengths, const int32_t* q_starts, int dtype, float scale,
                       void* out, int64_t out_stride_t, int64_t out_stride_h, int64_t tokens,
                       int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                       void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return paged_prefill(Sight{}, false, q, q_stride_t, q_stride_h, k_cache, v_cache, cache_stride_page,
                       cache_stride_head, cache_stride_token, pages, page_size, page_table,
                       ld_table, table_pages, lengths, q_starts, dtype, scale, out, out_stride_t,
                       out_stride_h, tokens, batch, q_heads, kv_heads, head_dim, workspace,
                       workspace_bytes, stream);
}

int w8a8_paged_prefill_padded(const void* q, int64_t q_stride_t, int64_t q_stride_h,
                              const void* k_cache, const void* v_cache, int64_t cache_stride_page,
                              int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                              int64_t page_size, const int32_t* page_table, int64_t ld_table,
                              int64_t table_pages, const int32_t* lengths, const int32_t* q_starts,
                              int dtype, float scale, void* out, int64_t out_stride_t,
                              int64_t out_stride_h, int64_t tokens, int64_t batch, int64_t q_heads,
                              int64_t kv_heads, int64_t head_dim, void* workspace,
                              int64_t workspace_bytes, hipStream_t stream) {
  return paged_prefill(Sight{}, true, q, q_stride_t, q_stride_h, k_cache, v_cache, cache_stride_page,
                       cache_stride_head, cache_stride_token, pages, page_size, page_table,
                       ld_table, table_pages, lengths, q_starts, dtype, scale, out, out_stride_t,
                       out_stride_h, tokens, batch, q_heads, kv_heads, head_dim, workspace,
                       workspace_bytes, stream);
}

int64_t w8a8_paged_decode_window_workspace_bytes(int64_t batch, int64_t q_heads,
                                                 int64_t kv_heads, int64_t head_dim,
                                                 int64_t max_keys, int64_t window,
                                                 int64_t sinks) {
  if (!sizes_ok(batch, batch, q_heads, kv_heads, head_dim, max_keys, kDecodeRows) ||
      !window_ok(window, sinks))
    return -1;
  const Sight s = window_of(window, sinks, max_keys);
  return s.windowed ? paged_decode_window_workspace(batch, q_heads, kv_heads, head_dim, max_keys,
                                                    s.window, s.sinks)
                    : paged_decode_workspace(batch, q_heads, kv_heads, head_dim, max_keys);
}

int w8a8_paged_decode_window(const void* q, int64_t q_stride_t, int64_t q_stride_h,
                             const void* k_cache, const void* v_cache, int64_t cache_stride_page,
                             int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                             int64_t page_size, const int32_t* page_table, int64_t ld_table,
                             int64_t table_pages, const int32_t* lengths, int64_t window,
                             int64_t sinks, int dtype, float scale, void* out,
                             int64_t out_stride_t, int64_t out_stride_h, int64_t batch,
                             int64_t q_heads, int64_t kv_heads, int64_t head_dim, void* workspace,
                             int64_t workspace_bytes, hipStream_t stream) {
  if (!window_ok(window, sinks)) return W8A8_ERR_SHAPE;
  Sight s;
  s.windowed = true;
  s.window = window;
  s.sinks = sinks;
  return paged_decode(s, q, q_stride_t, q_stride_h, k_cache, v_cache, cache_stride_page,
                      cache_stride_head, cache_stride_token, pages, page_size, page_table,
                      ld_table, table_pages, lengths, dtype, scale, out, out_stride_t,
                      out_stride_h, batch, q_heads, kv_heads, head_dim, workspace,
                      workspace_bytes, stream);
}

int64_t w8a8_paged_prefill_window_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads,
                                                  int64_t kv_heads, int64_t head_dim,
                                                  int64_t max_keys, int64_t window,
                                                  int64_t sinks) {
  if (!sizes_ok(tokens, batch, q_heads, kv_heads, head_dim, max_keys, kPrefillRows) ||
      !window_ok(window, sinks))
    return -1;
  return prefill_workspace(window_of(window, sinks, max_keys), tokens, batch, q_heads, kv_heads,
                           head_dim, max_keys);
}

int w8a8_paged_prefill_window(const void* q, int64_t q_stride_t, int64_t q_stride_h,
                              const void* k_cache, const void* v_cache, int64_t cache_stride_page,
                              int64_t cache_stride_head, int64_t cache_stride_token, int64_t pages,
                              int64_t page_size, const int32_t* page_table, int64_t ld_table,
                              int64_t table_pages, const int32_t* lengths, const int32_t* q_starts,
                              int64_t window, int64_t sinks, int clear_rows, int dtype,
                              float scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                              int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                              int64_t head_dim, void* workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  if (!window_ok(window, sinks)) return W8A8_ERR_SHAPE;
  Sight s;
  s.windowed = true;
  s.window = window;
  s.sinks = sinks;
  return paged_prefill(s, clear_rows != 0, q, q_stride_t, q_stride_h, k_cache, v_cache,
                       cache_stride_page, cache_stride_head, cache_stride_token, pages, page_size,
                       page_table, ld_table, table_pages, lengths, q_starts, dtype, scale, out,
                       out_stride_t, out_stride_h, tokens, batch, q_heads, kv_heads, head_dim,
                       workspace, workspace_bytes, stream);
}

int64_t w8a8_paged_tree_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int64_t max_keys) {
  if (!sizes_ok(tokens, batch, q_heads, kv_heads, head_dim, max_keys, kPrefillRows)) return -1;
  return paged_tree_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
}

int w8a8_paged_tree(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                    const void* v_cache, int64_t cache_stride_page, int64_t cache_stride_head,
                    int64_t cache_stride_token, int64_t pages, int64_t page_size,
                    const int32_t* page_table, int64_t ld_table, int64_t table_pages,
                    const int32_t* lengths, const int32_t* q_starts, const uint64_t* masks,
                    int64_t ld_masks, int64_t mask_words, int clear_rows, int dtype, float scale,
                    void* out, int64_t out_stride_t, int64_t out_stride_h, int64_t tokens,
                    int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                    void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (mask_words < 0 || mask_words > kMaxTokens / 64 || ld_masks < mask_words ||
      ld_masks > kMaxStride)
    return W8A8_ERR_SHAPE;
  Sight s;
  s.tree = true;
  s.masks = masks;
  s.ld_masks = ld_masks;
  s.words = mask_words;
  return paged_prefill(s, clear_rows != 0, q, q_stride_t, q_stride_h, k_cache, v_cache,
                       cache_stride_page, cache_stride_head, cache_stride_token, pages, page_size,
                       page_table, ld_table, table_pages, lengths, q_starts, dtype, scale, out,
                       out_stride_t, out_stride_h, tokens, batch, q_heads, kv_heads, head_dim,
                       workspace, workspace_bytes, stream);
}

int w8a8_cache_accept(void* k_cache, void* v_cache, int64_t cache_stride_layer,
                      int64_t cache_stride_page, int64_t cache_stride_head,
                      int64_t cache_stride_token, int64_t layers, int64_t pages,
                      int64_t page_size, const int32_t* page_table, int64_t ld_table,
                      int64_t table_pages, const int32_t* lengths, const int32_t* path,
                      int64_t ld_path, int64_t path_length, int dtype, int64_t batch,
                      int64_t kv_heads, int64_t head_dim, hipStream_t stream) {
  if (!half_dtype(dtype)) return W8A8_ERR_DTYPE;
  const Cache c{cache_stride_page, cache_stride_head, cache_stride_token, pages,
                page_size,         kv_heads,          head_dim};
  if (head_dim <= 0 || head_dim % 8 || head_dim > kAttentionMaxDim || kv_heads <= 0 ||
      kv_heads > kMaxHeads || batch < 0 || batch > kMaxGridYZ || layers < 0 ||
      layers > kMaxGridYZ / 2 ||
      cache_accept_workgroups(layers, batch, kv_heads, head_dim) > kMaxBlocks)
    return W8A8_ERR_SHAPE;
  const int rc = check_cache(c, 8);
  if (rc != W8A8_OK) return rc;
  if (table_pages < 0 || ld_table < table_pages || ld_table > kMaxStride ||
      table_pages > kMaxTokens / page_size || path_length < 0 || path_length > kMaxTokens ||
      ld_path < path_length || ld_path > kMaxStride || !strides_ok(cache_stride_layer, 0))
    return W8A8_ERR_SHAPE;
  if (layers > 1 && cache_stride_layer % 8) return W8A8_ERR_ALIGN;
  if (batch == 0 || layers == 0 || pages == 0 || table_pages == 0 || path_length == 0)
    return W8A8_OK;
  if (k_cache == nullptr || v_cache == nullptr || page_table == nullptr || lengths == nullptr ||
      path == nullptr)
    return W8A8_ERR_NULL;
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(page_table, 4) ||
      !aligned(lengths, 4) || !aligned(path, 4))
    return W8A8_ERR_ALIGN;
  const i128 bytes = cache_bytes(c) + 2 * i128(layers - 1) * cache_stride_layer;
  if (bytes > kMaxBytes || i128(batch) * ld_table > kMaxBytes || i128(batch) * ld_path > kMaxBytes)
    return W8A8_ERR_SHAPE;
  if (!cache_distinct(c, cache_stride_layer, layers) ||
      !caches_apart(k_cache, v_cache, c, cache_stride_layer, layers))
    return W8A8_ERR_OVERLAP;
  // Up to the last row's last entry: what is behind it may be another tensor's.
  for (const auto& in :
       {std::pair<const void*, i128>{page_table, 4 * (i128(batch - 1) * ld_table + table_pages)},
        {lengths, 4 * i128(batch)},
        {path, 4 * (i128(batch - 1) * ld_path + path_length)}}) {
    const i128 a0 = i128(reinterpret_cast<uintptr_t>(in.first));
    for (const void* cache : {k_cache, v_cache}) {
      const i128 b0 = i128(reinterpret_cast<uintptr_t>(cache));
      if (a0 < b0 + bytes && b0 < a0 + in.second) return W8A8_ERR_OVERLAP;
    }
  }
  CacheAccept p;
  p.k = k_cache;
  p.v = v_cache;
  p.c_layer = cache_stride_layer;
  p.c_page = cache_stride_page;
  p.c_head = cache_stride_head;
  p.c_tok = cache_stride_token;
  p.pages = pages;
  p.table = page_table;
  p.ld_table = ld_table;
  p.lengths = lengths;
  p.path = path;
  p.ld_path = ld_path;
  p.steps = static_cast<int>(path_length);
  p.page_shift = page_shift_of(page_size);
  p.max_keys = static_cast<int>(table_pages * page_size);
  p.layers = static_cast<int>(layers);
  p.batch = static_cast<int>(batch);
  p.kv_heads = static_cast<int>(kv_heads);
  p.head_dim = static_cast<int>(head_dim);
  return status_of(launch_cache_accept(p, stream));
}

}  // extern "C"
