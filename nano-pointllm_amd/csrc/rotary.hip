// Rotary positions, and the store of rotated keys and values into a paged
// key-value cache (gfx950).
//
// Mathematics.  Pair i of a head at position p turns by the angle
// p * inv_freq[i]: (x, y) -> (x c - y s, y c + x s), c = a cos, s = a sin with
// one amplitude a for all pairs (the attention factor of scaled contexts).
// Layout half pairs elements (i, i + R/2) of the first R elements of a head,
// layout interleaved (2i, 2i + 1); elements past R pass through.
//
// The angle is formed in binary64 as turns (p * inv_freq / 2 pi), reduced to
// the nearest whole turn there, and only the remainder is rounded to binary32:
// a position of 10^6 loses nothing, where a binary32 angle is off by 0.06 rad.
// Products and sums run in binary32 with one rounding to the 16-bit type.
//
// Bound by memory: 2 bytes in and 2 out per element, 6 operations per pair.
// 4097 tokens of 32 query heads and 8 key heads: 19.7 us, 5.1 TB/s.  Small calls
// are bound by their launch: one token 3.2 us, 560 tokens of 32 and 32 heads 7.3.
// A workgroup takes one token and up to kThreads items of it (an item is one
// 16-byte chunk, or the two chunks of a half pair), so cos and sin are formed
// once per workgroup by R/2 threads, in LDS, while the row loads are in flight.
// Two items per thread, for half the sines, are 9% slower at 4097 tokens.
#include <algorithm>

#include "w8a8_internal.h"

namespace w8a8 {

namespace {

constexpr int kThreads = 256;

struct RotaryParams {
  RotaryRows r;
  int items_qk;       // items of one rotated head
  int items_v;        // items of one value head
  uint32_t magic_qk;  // divide() multiplier of items_qk and items_v
  uint32_t magic_v;
  int total;          // items of one token
};

// n / d for n d < 2^32 by its multiplier floor(2^32 / d) + 1 (0 for d = 1,
// whose own does not fit).
inline uint32_t multiplier(int d) {
  return d == 1 ? 0 : static_cast<uint32_t>((uint64_t{1} << 32) / d + 1);
}
__device__ inline int divide(int n, uint32_t mult) {
  return mult == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), mult));
}

// W consecutive 16-bit elements.
template <int W> struct Chunk { uint16_t e[W]; };
template <int W>
__device__ inline Chunk<W> load_chunk(const uint16_t* p) {
  Chunk<W> c;
  if constexpr (W == 8) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
    __builtin_memcpy(c.e, &v, 16);
  } else if constexpr (W == 4) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    __builtin_memcpy(c.e, &v, 8);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) c.e[j] = p[j];
  }
  return c;
}
template <int W>
__device__ inline void store_chunk(uint16_t* p, const Chunk<W>& c) {
  if constexpr (W == 8) {
    u32x4 v;
    __builtin_memcpy(&v, c.e, 16);
    *reinterpret_cast<u32x4*>(p) = v;
  } else if constexpr (W == 4) {
    u32x2 v;
    __builtin_memcpy(&v, c.e, 8);
    *reinterpret_cast<u32x2*>(p) = v;
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = c.e[j];
  }
}

template <typename T>
__device__ inline void turn(uint16_t& a, uint16_t& b, float2 cs) {
  const float x = bits_to_f32<T>(a), y = bits_to_f32<T>(b);
  const float u = x * cs.x - y * cs.y, v = y * cs.x + x * cs.y;
  a = __builtin_bit_cast(uint16_t, from_f32<T>(u));
  b = __builtin_bit_cast(uint16_t, from_f32<T>(v));
}

// W: elements per chunk (divides R/2 for half, R for interleaved, and every
// address).
template <typename T, bool HALF, int W>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p) {
  __shared__ float2 cs[kRotaryMaxDim / 2];
  const RotaryRows& r = p.r;
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x;
  const int half = r.rotary_dim >> 1;
  const int n = static_cast<int>(blockIdx.y) * kThreads + tid;
  const int rotated = (r.q_heads + r.kv_heads) * p.items_qk;

  // An item's rows and elements: a rotated pair of chunks (half), a rotated
  // chunk (interleaved) or a copied one.
  struct Item {
    const uint16_t* src;
    uint16_t* dst;
    int e0;       // first element
    int e1;       // first element of the second chunk, or -1
    bool turned;
  };
  const int64_t slot = r.k != nullptr ? r.slots[t] : -1;
  const bool kept = slot >= 0 && slot < (r.pages << r.page_shift);
  const int64_t cache_row = kept ? (slot >> r.page_shift) * r.c_page +
                                       (slot & ((int64_t{1} << r.page_shift) - 1)) * r.c_tok
                                 : 0;
  auto locate = [&](Item& it) -> bool {
    if (n >= p.total) return false;
    if (n < rotated) {
      const int head = divide(n, p.magic_qk);
      const int i = n - head * p.items_qk;
      if (head < r.q_heads) {
        it.src = static_cast<const uint16_t*>(r.q) + t * r.q_st + head * r.q_sh;
        it.dst = static_cast<uint16_t*>(r.q_out) + t * r.qo_st + head * r.qo_sh;
      } else {
        if (!kept) return false;
        const int h = head - r.q_heads;
        it.src = static_cast<const uint16_t*>(r.k) + t * r.k_st + h * r.k_sh;
        it.dst = static_cast<uint16_t*>(r.k_cache) + cache_row + h * r.c_head;
      }
      if (HALF) {
        it.turned = i * W < half;
        it.e0 = it.turned ? i * W : i * W + half;
        it.e1 = it.turned ? i * W + half : -1;
      } else {
        it.e0 = i * W;
        it.e1 = -1;
        it.turned = it.e0 < r.rotary_dim;
      }
      return true;
    }
    if (!kept) return false;
    const int m = n - rotated;
    const int h = divide(m, p.magic_v);
    it.src = static_cast<const uint16_t*>(r.v) + t * r.v_st + h * r.v_sh;
    it.dst = static_cast<uint16_t*>(r.v_cache) + cache_row + h * r.c_head;
    it.e0 = (m - h * p.items_v) * W;
    it.e1 = -1;
    it.turned = false;
    return true;
  };

  Chunk<W> a, b;
  Item it;
  const bool mine = locate(it);
  if (mine) {
    a = load_chunk<W>(it.src + it.e0);
    if (HALF && it.e1 >= 0) b = load_chunk<W>(it.src + it.e1);
  }
  for (int i = tid; i < half; i += kThreads) {
    constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
    const double turns = static_cast<double>(r.positions[t]) * r.inv_freq[i] * kTurn;
    const float rest = static_cast<float>(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    cs[i] = float2{r.factor * c, r.factor * s};
  }
  __syncthreads();
  if (!mine) return;
  if (HALF) {
    if (it.turned) {
#pragma unroll
      for (int e = 0; e < W; ++e) turn<T>(a.e[e], b.e[e], cs[it.e0 + e]);
      store_chunk<W>(it.dst + it.e1, b);
    }
  } else if (it.turned) {
#pragma unroll
    for (int e = 0; e < W; e += 2) turn<T>(a.e[e], a.e[e + 1], cs[(it.e0 + e) >> 1]);
  }
  store_chunk<W>(it.dst + it.e0, a);
}

template <typename T, bool HALF, int W>
hipError_t launch_w(RotaryRows const& r, hipStream_t st) {
  RotaryParams p;
  p.r = r;
  p.items_qk = HALF ? (r.head_dim - r.rotary_dim / 2) / W : r.head_dim / W;
  p.items_v = r.head_dim / W;
  p.magic_qk = multiplier(p.items_qk);
  p.magic_v = multiplier(p.items_v);
  p.total = (r.q_heads + r.kv_heads) * p.items_qk + r.kv_heads * p.items_v;
  const dim3 grid(static_cast<uint32_t>(r.tokens),
                  static_cast<uint32_t>(ceil_div(p.total, kThreads)));
  hipLaunchKernelGGL((rotary_kernel<T, HALF, W>), grid, dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

// Elements (at most 8) that `v` elements divide into.
inline int width_of(int64_t v) { return v % 8 == 0 ? 8 : v % 4 == 0 ? 4 : v % 2 == 0 ? 2 : 1; }
inline int width_of(const void* ptr) {
  return width_of(static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr) / 2));
}

template <typename T>
hipError_t launch_t(const RotaryRows& r, hipStream_t st) {
  // The widest chunk that every address and the rotated part divide into.
  int w = r.half ? width_of(r.rotary_dim / 2) : width_of(r.rotary_dim);
  for (const int64_t v : {r.q_st, r.q_sh, r.qo_st, r.qo_sh}) w = std::min(w, width_of(v));
  w = std::min(w, std::min(width_of(r.q), width_of(r.q_out)));
  if (r.k != nullptr) {
    for (const int64_t v : {r.k_st, r.k_sh, r.v_st, r.v_sh, r.c_page, r.c_head, r.c_tok})
      w = std::min(w, width_of(v));
    for (const void* v : {r.k, r.v, static_cast<const void*>(r.k_cache),
                          static_cast<const void*>(r.v_cache)})
      w = std::min(w, width_of(v));
  }
  if (r.half) {
    if (w == 8) return launch_w<T, true, 8>(r, st);
    if (w == 4) return launch_w<T, true, 4>(r, st);
    return launch_w<T, true, 1>(r, st);
  }
  if (w == 8) return launch_w<T, false, 8>(r, st);
  if (w == 4) return launch_w<T, false, 4>(r, st);
  return launch_w<T, false, 2>(r, st);
}

}  // namespace

hipError_t launch_rotary(const RotaryRows& r, int dtype, hipStream_t st) {
  return dtype == kF16 ? launch_t<__half>(r, st) : launch_t<__hip_bfloat16>(r, st);
}

}  // namespace w8a8
