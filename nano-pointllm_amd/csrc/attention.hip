// Attention over a paged key-value cache, one wavefront per query row and
// head: the plainest kernel of the two entry points.
#include "w8a8_internal.h"

namespace w8a8 {

namespace {

constexpr int kWaves = 4;

// NCH: lanes of one key (each holds 8 elements of it), a power of two.
template <typename T, int NCH>
__global__ __launch_bounds__(64 * kWaves) void attention_rows_kernel(PagedAttention p) {
  const int lane = threadIdx.x & 63;
  const int head = static_cast<int>(blockIdx.y) * kWaves + (threadIdx.x >> 6);
  if (head >= p.q_heads) return;
  const int t = blockIdx.x;
  int seq = t;
  int last = 0;  // the last key this row sees
  if (p.q_starts != nullptr) {
    seq = -1;
    for (int b = 0; b < p.batch; ++b) {
      const int s0 = max(p.q_starts[b], 0), s1 = min(p.q_starts[b + 1], p.tokens);
      if (t >= s0 && t < s1) {
        seq = b;
        last = min(p.lengths[b], p.max_keys) - (s1 - s0) + (t - s0);
        break;
      }
    }
    if (seq < 0) return;
  } else {
    last = min(p.lengths[seq], p.max_keys) - 1;
  }
  const int chunk = lane % NCH;
  const bool live = chunk * 8 < p.head_dim;
  const int kvh = head / (p.q_heads / p.kv_heads);
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = 0.0f;
  if (live)
    load8<T>(static_cast<const T*>(p.q) + t * p.q_st + head * p.q_sh + chunk * 8, q, true, 8);
  float m = -INFINITY, l = 0.0f, o[8] = {};
  for (int j = lane / NCH; j <= last; j += 64 / NCH) {
    const int page = p.table[seq * p.ld_table + (j >> p.page_shift)];
    if (page < 0 || page >= p.pages) continue;
    const int64_t at = page * p.c_page + kvh * p.c_head +
                       (j & ((1 << p.page_shift) - 1)) * p.c_tok + chunk * 8;
    float k[8] = {}, v[8] = {};
    if (live) {
      load8<T>(static_cast<const T*>(p.k) + at, k, true, 8);
      load8<T>(static_cast<const T*>(p.v) + at, v, true, 8);
    }
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(q[e], k[e], s);
#pragma unroll
    for (int w = 1; w < NCH; w <<= 1) s += __shfl_xor(s, w);
    s *= p.scale;
    const float m1 = fmaxf(m, s);
    // Without a key above -inf so far the weights are taken against 0: those
    // of -inf are 0, and a NaN score stays one.
    const float base = m1 == -INFINITY ? 0.0f : m1;
    const float f = expf(m - base), w = expf(s - base);
    m = m1;
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f + w * v[e];
  }
#pragma unroll
  for (int w = NCH; w < 64; w <<= 1) {
    const float m2 = __shfl_xor(m, w), l2 = __shfl_xor(l, w);
    const float m1 = fmaxf(m, m2);
    // Without one on either side both are kept as they are: 0, or NaN.
    const float base = m1 == -INFINITY ? 0.0f : m1;
    const float f = m1 == -INFINITY ? 1.0f : expf(m - base);
    const float f2 = m1 == -INFINITY ? 1.0f : expf(m2 - base);
    m = m1;
    l = l * f + l2 * f2;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f + __shfl_xor(o[e], w) * f2;
  }
  if (lane < NCH && live) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = pack2_bits<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
    *reinterpret_cast<u32x4*>(static_cast<T*>(p.out) + t * p.o_st + head * p.o_sh + chunk * 8) = y;
  }
}

template <typename T>
hipError_t launch_t(const PagedAttention& p, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(p.tokens),
                  static_cast<uint32_t>(ceil_div(p.q_heads, kWaves)));
  const dim3 block(64 * kWaves);
  if (p.head_dim <= 64)
    hipLaunchKernelGGL((attention_rows_kernel<T, 8>), grid, block, 0, st, p);
  else if (p.head_dim <= 128)
    hipLaunchKernelGGL((attention_rows_kernel<T, 16>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((attention_rows_kernel<T, 32>), grid, block, 0, st, p);
  return hipGetLastError();
}

hipError_t launch_rows(const PagedAttention& p, int dtype, hipStream_t st) {
  return dtype == kF16 ? launch_t<__half>(p, st) : launch_t<__hip_bfloat16>(p, st);
}

}  // namespace

int64_t paged_prefill_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
  return 0;
}

hipError_t launch_paged_prefill(const PagedAttention& p, int dtype, hipStream_t st) {
  return launch_rows(p, dtype, st);
}

}  // namespace w8a8
