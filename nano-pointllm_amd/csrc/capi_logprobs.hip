// extern "C" entry points of the log probabilities (declared in
// include/w8a8_gfx950.h): argument checks and dispatch.  The kernels live in
// logprobs.hip.
#include "w8a8_gfx950.h"
#include "w8a8_internal.h"

using namespace w8a8;

namespace {

using i128 = __int128;

struct Range {
  const void* p;
  i128 bytes;
};
bool apart(const Range& a, const Range& b) {
  if (a.p == nullptr || b.p == nullptr) return true;
  const i128 a0 = i128(reinterpret_cast<uintptr_t>(a.p));
  const i128 b0 = i128(reinterpret_cast<uintptr_t>(b.p));
  return a0 + a.bytes <= b0 || b0 + b.bytes <= a0;
}
bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// A launch's threads are counted in 32 bits, a workgroup has up to 1024.
constexpr int64_t kMaxRows = (int64_t{1} << 22) - 1;   // and of workgroups
constexpr int64_t kMaxGiven = int64_t{1} << 20;
constexpr int64_t kMaxLd = int64_t{1} << 38;

bool sizes_ok(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  return rows >= 0 && rows <= kMaxRows && vocab >= 1 && vocab <= kLogprobsMaxVocab && top >= 0 &&
         top <= kLogprobsMaxTop && top <= vocab &&
         token_logprobs_workgroups(rows, vocab, dtype) <= kMaxRows;
}

}  // namespace

extern "C" {

int64_t w8a8_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  if ((dtype != kF32 && dtype != kF16 && dtype != kBF16) || !sizes_ok(rows, vocab, top, dtype))
    return -1;
  return token_logprobs_workspace(rows, vocab, top, dtype);
}

int w8a8_token_logprobs(const void* logits, int64_t ld_logits, int dtype, const int64_t* tokens,
                        int64_t ld_tokens, int64_t given, int64_t top, float* logprobs,
                        float* entropy, float* top_logprobs, int64_t* top_tokens, int64_t rows,
                        int64_t vocab, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream) {
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return W8A8_ERR_DTYPE;
  if (!sizes_ok(rows, vocab, top, dtype) || given < 0 || given > kMaxGiven) return W8A8_ERR_SHAPE;
  if (ld_logits < 0 || ld_logits > kMaxLd || ld_tokens < 0 || ld_tokens > kMaxLd)
    return W8A8_ERR_SHAPE;
  if (rows == 0) return W8A8_OK;
  const int size = dtype == kF32 ? 4 : 2;
  if (logits == nullptr || (given > 0 && (tokens == nullptr || logprobs == nullptr)) ||
      (top > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return W8A8_ERR_NULL;
  if (!aligned(logits, size) || !aligned(tokens, 8) || !aligned(logprobs, 4) ||
      !aligned(entropy, 4) || !aligned(top_logprobs, 4) || !aligned(top_tokens, 8))
    return W8A8_ERR_ALIGN;
  const int64_t need = token_logprobs_workspace(rows, vocab, top, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return W8A8_ERR_WORKSPACE;
  if (need > 0 && !aligned(workspace, 16)) return W8A8_ERR_ALIGN;
  const Range in[2] = {{logits, size * (i128(rows - 1) * ld_logits + vocab)},
                       {given > 0 ? tokens : nullptr, 8 * (i128(rows - 1) * ld_tokens + given)}};
  const Range out[5] = {{given > 0 ? logprobs : nullptr, 4 * i128(rows) * given},
                        {entropy, 4 * i128(rows)},
                        {top > 0 ? top_logprobs : nullptr, 4 * i128(rows) * top},
                        {top > 0 ? top_tokens : nullptr, 8 * i128(rows) * top},
                        {need > 0 ? workspace : nullptr, need}};
  for (int i = 0; i < 5; ++i) {
    for (const Range& r : in)
      if (!apart(out[i], r)) return W8A8_ERR_OVERLAP;
    for (int j = 0; j < i; ++j)
      if (!apart(out[i], out[j])) return W8A8_ERR_OVERLAP;
  }
  TokenLogprobs p;
  p.logits = logits;
  p.ld = ld_logits;
  p.tokens = tokens;
  p.ld_tokens = ld_tokens;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.top_logprobs = top_logprobs;
  p.top_tokens = top_tokens;
  p.workspace = workspace;
  p.rows = rows;
  p.vocab = static_cast<int>(vocab);
  p.given = static_cast<int>(given);
  p.top = static_cast<int>(top);
  return status_of(launch_token_logprobs(p, dtype, stream));
}

}  // extern "C"
