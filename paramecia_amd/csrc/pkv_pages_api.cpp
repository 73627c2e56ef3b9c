// C entry points of a serving step over pages that tables on the device name (include/pkv.h):
// the checks of their arguments, in front of the launchers.
#include <cmath>
#include <initializer_list>

#include "pkv_internal.hpp"

namespace pkv {
namespace {

struct Span {
  const void *p;
  uint64_t bytes;
  bool written;
};
// A written buffer that shares a byte with another one of the call.
bool clash(std::initializer_list<Span> spans) {
  for (const Span *a = spans.begin(); a != spans.end(); ++a)
    for (const Span *b = a + 1; b != spans.end(); ++b) {
      if ((!a->written && !b->written) || !a->p || !b->p || !a->bytes || !b->bytes) continue;
      const uint64_t x = reinterpret_cast<uintptr_t>(a->p), y = reinterpret_cast<uintptr_t>(b->p);
      if (x < y + b->bytes && y < x + a->bytes) return true;
    }
  return false;
}

bool page_size(int page_tokens) {
  return page_tokens >= 32 && page_tokens <= (1 << 20) && (page_tokens & (page_tokens - 1)) == 0;
}
int refuse_page_size() { return set_error(PKV_ERR_ARG, "page_tokens must be a power of two in [32, 2^20]"); }

constexpr int64_t kMost32 = (int64_t)1 << 31;

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

int pkv_pages_map(const int *lens, const int *add, int n, int *tables, int max_pages, int *held,
                  int *free_pages, int *free_count, int capacity, int page_tokens,
                  int64_t *slots, int *positions, int64_t max_tokens, int *starts, int *totals,
                  int *status, pkv_stream stream) {
  if (n <= 0 || max_pages <= 0 || capacity <= 0)
    return set_error(PKV_ERR_ARG, "n, max_pages and capacity must be > 0");
  if (!page_size(page_tokens)) return refuse_page_size();
  if (max_tokens < 0 || max_tokens >= kMost32)
    return set_error(PKV_ERR_ARG, "max_tokens must be in [0, 2^31)");
  if ((int64_t)n * max_pages >= kMost32)
    return set_error(PKV_ERR_UNSUPPORTED, "the tables must hold fewer than 2^31 pages");
  if (!lens || !add || !tables || !held || !free_pages || !free_count || !starts || !totals ||
      !status || (max_tokens && (!slots || !positions)))
    return set_error(PKV_ERR_ARG, "null argument");
  const uint64_t m = 4 * (uint64_t)n;
  if (clash({{lens, m, false}, {add, m, false}, {tables, m * max_pages, true}, {held, m, true},
             {free_pages, 4 * (uint64_t)capacity, true}, {free_count, 4, true},
             {slots, 8 * (uint64_t)max_tokens, true}, {positions, 4 * (uint64_t)max_tokens, true},
             {starts, m + 4, true}, {totals, m, true}, {status, 4, true}}))
    return set_error(PKV_ERR_ARG, "the buffers must not overlap");
  return launch_pages_map(lens, add, n, tables, max_pages, held, free_pages, free_count, capacity,
                          page_tokens, slots, positions, max_tokens, starts, totals, status,
                          static_cast<hipStream_t>(stream));
}

int pkv_pages_append(int quant, const float *k, const float *v, int64_t k_stride, int64_t v_stride,
                     const int64_t *slots, int64_t n, void *k_pages, void *v_pages,
                     int64_t n_slots, int n_kv_heads, int head_dim, pkv_stream stream) {
  if (n < 0 || n_slots <= 0 || n_kv_heads <= 0 || head_dim <= 0)
    return set_error(PKV_ERR_ARG, "n must be >= 0, and n_slots, n_kv_heads and head_dim > 0");
  if (quant == PKV_QUANT_NONE) quant = PKV_QUANT_F16;
  if (quant != PKV_QUANT_F16 && quant != PKV_QUANT_BF16)
    return set_error(PKV_ERR_UNSUPPORTED, "pages of F16 or BF16 rows");
  if (n == 0) return PKV_OK;
  if (!k || !v || !slots || !k_pages || !v_pages) return set_error(PKV_ERR_ARG, "null argument");
  const int64_t width = (int64_t)n_kv_heads * head_dim;
  if (width >= kMost32 || n >= kMost32 || n * width >= kMost32)
    return set_error(PKV_ERR_UNSUPPORTED, "n * n_kv_heads * head_dim must be below 2^31");
  if (n > 1 && (k_stride < width || v_stride < width))
    return set_error(PKV_ERR_ARG, "a token's row holds all its heads, and rows do not overlap");
  if (k_stride < 0 || v_stride < 0) return set_error(PKV_ERR_ARG, "strides must be >= 0");
  const uint64_t plane = 2 * (uint64_t)n_slots * width;
  if (clash({{k, 4 * ((uint64_t)(n - 1) * k_stride + width), false},
             {v, 4 * ((uint64_t)(n - 1) * v_stride + width), false},
             {slots, 8 * (uint64_t)n, false}, {k_pages, plane, true}, {v_pages, plane, true}}))
    return set_error(PKV_ERR_ARG, "the pages must not overlap another buffer");
  return launch_pages_append(quant, k, v, k_stride, v_stride, slots, n, k_pages, v_pages, n_slots,
                             (int)width, static_cast<hipStream_t>(stream));
}

static bool attend_shape(int n, int64_t tokens, int num_heads, int num_kv_heads) {
  return n > 0 && tokens >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 &&
         n < (1 << 24) && tokens < kMost32 && tokens * num_heads < kMost32 && num_kv_heads <= (1 << 14) &&
         (n + tokens) * num_kv_heads < kMost32;
}
static bool attend_dim(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

size_t pkv_pages_attend_workspace(int n, int64_t tokens, int num_heads, int num_kv_heads, int head_dim) {
  if (!attend_shape(n, tokens, num_heads, num_kv_heads) || !attend_dim(head_dim) || tokens == 0) return 0;
  return pages_attend_workspace(n, tokens, num_heads, num_kv_heads, head_dim);
}

int pkv_pages_attend(int quant, const float *q, int64_t q_stride_t, int64_t q_stride_h,
                     const void *k_pages, const void *v_pages, int n_pages, int page_tokens,
                     const int *tables, int max_pages, const int *lens, const int *starts, int n,
                     int64_t tokens, int num_heads, int num_kv_heads, int head_dim, float scale,
                     int window, int sinks, float *out, void *workspace, size_t workspace_bytes,
                     pkv_stream stream) {
  if (n <= 0 || tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return set_error(PKV_ERR_ARG, "n and num_heads > 0, tokens >= 0, and num_heads a multiple of num_kv_heads");
  if (n_pages <= 0 || max_pages <= 0) return set_error(PKV_ERR_ARG, "n_pages and max_pages must be > 0");
  if (!page_size(page_tokens)) return refuse_page_size();
  if ((int64_t)max_pages * page_tokens > kMost32 - 64)
    return set_error(PKV_ERR_ARG, "a table must name fewer than 2^31 - 64 tokens");
  if (window < 0 || sinks < 0) return set_error(PKV_ERR_ARG, "window and sinks must be >= 0");
  // the kernels hold scores times log2(e)
  if (!std::isfinite(scale * 1.4426950408889634f)) return set_error(PKV_ERR_ARG, "scale times log2(e) must be finite");
  if (!starts && tokens != n)
    return set_error(PKV_ERR_ARG, "without starts every request has one row: tokens must be n");
  if (quant == PKV_QUANT_NONE) quant = PKV_QUANT_F16;
  if (quant != PKV_QUANT_F16 && quant != PKV_QUANT_BF16)
    return set_error(PKV_ERR_UNSUPPORTED, "pages of F16 or BF16 rows");
  if (!attend_dim(head_dim)) return set_error(PKV_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
  if (!attend_shape(n, tokens, num_heads, num_kv_heads))
    return set_error(PKV_ERR_UNSUPPORTED, "n must be below 2^24, tokens * num_heads and (n + tokens) * "
                                          "num_kv_heads below 2^31, num_kv_heads at most 2^14");
  if (tokens == 0) return PKV_OK;
  if (!q || !k_pages || !v_pages || !tables || !lens || !out || !workspace)
    return set_error(PKV_ERR_ARG, "null argument");
  if ((num_heads > 1 && q_stride_h < head_dim) || q_stride_h < 0 || q_stride_t < 0 ||
      (tokens > 1 && q_stride_t < (int64_t)(num_heads - 1) * q_stride_h + head_dim))
    return set_error(PKV_ERR_ARG, "q: a token's row holds all its heads, and rows do not overlap");
  if (q_stride_t % 4 != 0 || q_stride_h % 4 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
        reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) != 0)
    return set_error(PKV_ERR_ARG, "q, out and the pages must be 16-byte aligned, q's strides multiples of 4");
  const size_t need = pages_attend_workspace(n, tokens, num_heads, num_kv_heads, head_dim);
  if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return set_error(PKV_ERR_ARG, "the workspace must hold pkv_pages_attend_workspace() bytes, 256-byte aligned");
  const uint64_t plane = (uint64_t)n_pages * page_tokens * num_kv_heads * head_dim * 2;
  if (clash({{q, 4 * ((uint64_t)(tokens - 1) * q_stride_t + (uint64_t)(num_heads - 1) * q_stride_h + head_dim), false},
             {k_pages, plane, false}, {v_pages, plane, false}, {tables, 4 * (uint64_t)n * max_pages, false},
             {lens, 4 * (uint64_t)n, false}, {starts, 4 * ((uint64_t)n + 1), false},
             {out, 4 * (uint64_t)tokens * num_heads * head_dim, true}, {workspace, need, true}}))
    return set_error(PKV_ERR_ARG, "out and the workspace must not overlap another buffer");
  PagesAttend p;
  p.quant = quant;
  p.q = q;
  p.q_t = q_stride_t;
  p.q_h = q_stride_h;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.n_pages = n_pages;
  p.page_tokens = page_tokens;
  p.max_pages = max_pages;
  p.tables = tables;
  p.lens = lens;
  p.starts = starts;
  p.n = n;
  p.tokens = tokens;
  p.heads = num_heads;
  p.kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.window = window;
  p.sinks = sinks;
  p.scale = scale;
  p.out = out;
  return launch_pages_attend(p, workspace, static_cast<hipStream_t>(stream));
}

size_t pkv_verify_drafts_workspace(int n, int vocab) {
  return n > 0 && vocab > 0 ? verify_drafts_workspace(n, vocab) : 0;
}

int pkv_verify_drafts(const float *target, int64_t target_stride, const float *draft,
                      int64_t draft_stride, const int *drafts, const int *n_drafts, const float *u,
                      int n, int k, int vocab, int *tokens, int *accepted, void *workspace,
                      size_t workspace_bytes, pkv_stream stream) {
  if (n < 0 || k < 0 || vocab <= 0) return set_error(PKV_ERR_ARG, "n and k must be >= 0, vocab > 0");
  if (k > 63 || n > 65535) return set_error(PKV_ERR_UNSUPPORTED, "at most 63 drafts of 65535 sequences");
  if (n == 0) return PKV_OK;
  if (!target || (k && !drafts) || !u || !tokens || !accepted || !workspace)
    return set_error(PKV_ERR_ARG, "null argument");
  if (target_stride < vocab || (k && draft && draft_stride < vocab))
    return set_error(PKV_ERR_ARG, "rows of probabilities do not overlap");
  if (workspace_bytes < verify_drafts_workspace(n, vocab) || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0)
    return set_error(PKV_ERR_ARG, "the workspace must hold pkv_verify_drafts_workspace() bytes, 8-byte aligned");
  const uint64_t rows = (uint64_t)n * (k + 1);
  if (clash({{target, 4 * ((rows - 1) * (uint64_t)target_stride + vocab), false},
             {draft, k && draft ? 4 * (((uint64_t)n * k - 1) * (uint64_t)draft_stride + vocab) : 0, false},
             {drafts, 4 * (uint64_t)n * k, false}, {n_drafts, 4 * (uint64_t)n, false}, {u, 4 * rows, false},
             {tokens, 4 * rows, true}, {accepted, 4 * (uint64_t)n, true},
             {workspace, verify_drafts_workspace(n, vocab), true}}))
    return set_error(PKV_ERR_ARG, "tokens, accepted and the workspace must not overlap another buffer");
  return launch_verify_drafts(target, target_stride, draft, draft_stride, drafts, n_drafts, u, n, k,
                              vocab, tokens, accepted, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
