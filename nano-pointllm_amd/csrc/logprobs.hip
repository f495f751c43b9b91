// Log probabilities of given tokens, entropy and top tokens of logit rows (gfx950).
//
// Mathematics.  With m the largest logit of a row, n how many are equal to it and
// R = sum over the smaller ones of exp(x - m) plus n - 1, log sum exp(x) is m +
// log1p(R): a given token's log probability is (x - m) - log1p(R), the entropy
// log1p(R) + sum (m - x) exp(x - m) / (1 + R), all terms of one sign, so that a
// row that is nearly decided keeps its digits.
//
// Bound by memory where there are rows for every CU: 2048 rows of 32003 binary32 logits
// (262 MB) take 46 to 50 us, 5.2 to 5.7 TB/s.  16-bit logits are close to the vector
// units' bound, about ten instructions an element, four cycles each and sixteen for the
// exponential: 1024 rows of 128256 bfloat16 logits 61 us, 4.3 TB/s.  A few rows are bound
// by one workgroup's way through them: 8 of 32003 take 6.5 us, with 5 top tokens 8.4, 20
// 11, 64 16.
//
// Design:
//   * A workgroup holds a row, or a slice of a long one, in registers: the logits
//     are read once.  The sums run while later loads are in flight, against a
//     reference per thread that is the maximum so far or up to kSlack below.
//   * The thread whose logit is the row's maximum leaves its sums: its wavefront
//     adds its logits up again through LDS, with the maximum left out and counted
//     (of many such threads each reads its own again: 2048 rows of 32003 zeros 238
//     instead of 488 us).
//   * Top tokens: the k-th largest of 128 groups' maxima bounds the k-th largest
//     logit from below, and few logits reach it (k and some, rarely 2 k).  They go
//     through LDS, in any order, and each counts those before it: its place (k rounds
//     of the largest that is left, over the whole row, took 1 ms for 256 rows of
//     128256 and k = 20, this 4 us).  Ties
//     are broken by the token's number, so the order of arrival changes nothing.
//     Where more than kMost reach the bound (equal logits, masked ones at the type's
//     lowest value) the maxima of all threads give a better one, and of logits equal
//     to that the first tokens are counted off: 256 rows of 128256 zeros, 20 top
//     tokens, 106 us (one by one, as what is left after that is found, 1060), 8 rows of
//     32003 of which all but 3 are masked, 64 top tokens, 41 us (780).
//   * Rows of more vectors than a workgroup holds are cut into equal slices, whose
//     sums and top tokens a second launch joins.
#include <algorithm>

#include "attention_common.h"

namespace w8a8 {

namespace {

constexpr int kMost = 1024;        // candidates that a workgroup ranks
constexpr int kGroups = 128;       // maxima that the bound is taken from
constexpr int kFewHolders = 4;     // threads of a wavefront whose logits are spread over it
constexpr int kRankers = 8;        // threads that count those before one of many candidates
constexpr int kFew = 24;
constexpr int kMany = 256;         // candidates that are thinned out before they are ranked
constexpr float kSlack = 8.0f;     // in powers of two
constexpr float kLn2 = 0.693147180559945309417f;
constexpr int kJoinThreads = 256;
constexpr int kMaxSlices = 32;

// What a slice leaves for the join.
struct Part {
  float top;     // its largest logit
  float equal;   // how many are equal to it
  float sum;     // sum of exp(x - top) over the others, 0 if top is -inf
  float spread;  // sum of (top - x) exp(x - top)
};

template <typename T> constexpr int per_vector() { return 16 / sizeof(T); }

// Element j of a vector.
template <typename T> __device__ inline float element(const u32x4& v, int j) {
  if constexpr (std::is_same<T, float>::value) {
    return __uint_as_float(v[j]);
  } else {
    const uint32_t w = v[j >> 1];
    return bits_to_f32<T>((j & 1) ? w >> 16 : w & 0xffffu);
  }
}
template <typename T> __device__ inline uint32_t minus_infinity() {
  if constexpr (std::is_same<T, float>::value)
    return 0xff800000u;
  else if constexpr (std::is_same<T, __half>::value)
    return 0xfc00fc00u;
  else
    return 0xff80ff80u;
}

// The order of logits as whole numbers: by value, one zero, NaN above all.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? ~0u : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t order) {
  return __uint_as_float((order >> 31) ? order & 0x7fffffffu : ~order);
}
// ... and of equal ones by the token's number.
__device__ inline uint64_t rank_of(float x, int token) {
  return static_cast<uint64_t>(order_of(x)) << 32 | ~static_cast<uint32_t>(token);
}
__device__ inline int token_of(uint64_t rank) {
  return static_cast<int>(~static_cast<uint32_t>(rank));
}

__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) x += __shfl_xor(x, w);
  return x;
}
__device__ inline float wave_max(float x) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) x = fmaxf(x, __shfl_xor(x, w));
  return x;
}
__device__ inline uint64_t wave_max64(uint64_t x) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const uint64_t y = __shfl_xor(static_cast<unsigned long long>(x), w);
    x = y > x ? y : x;
  }
  return x;
}

// The k-th largest of 64 M orders, to its bits from LOW on, rounded down.
template <int LOW, int M> __device__ inline uint32_t kth_order(const uint32_t (&g)[M], int k) {
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t next = t | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) n += __popcll(__ballot(g[i] >= next));
    if (n >= k) t = next;
  }
  return t;
}

// f(place, rank) of each of n different ranks in LDS: its place among them, by counting
// those before it; of many, by several threads each.
template <typename F>
__device__ inline void rank_all(const uint64_t* ranks, int n, int tid, int threads, F f) {
  if (n <= kFew) {
    if (tid >= n) return;
    const uint64_t mine = ranks[tid];
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) place += ranks[j] > mine;
    f(place, mine);
    return;
  }
  const int part = tid % kRankers;
  for (int i = tid / kRankers; i < n; i += threads / kRankers) {
    const uint64_t mine = ranks[i];
    int place = 0;
#pragma unroll 4
    for (int j = part; j < n; j += kRankers) place += ranks[j] > mine;
#pragma unroll
    for (int w = 1; w < kRankers; w <<= 1) place += __shfl_xor(place, w);
    if (part == 0) f(place, mine);
  }
}

// The results of a row whose logits are known but for the given tokens'.
struct Row {
  float top, norm, entropy;   // norm: log sum exp(x - top)
  __device__ float logprob(float x) const { return (x - top) - norm; }
};
__device__ inline Row finish(float top, float equal, float sum, float spread) {
  const float rest = sum + (equal - 1.0f);
  const float norm = top == -INFINITY ? NAN : log1pf(rest);
  return Row{top, norm, norm + spread / (1.0f + rest)};
}
template <typename T>
__device__ inline void write_given(const TokenLogprobs& p, int64_t row, const Row& r, int i,
                                   int n) {
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  for (; i < p.given; i += n) {
    const int64_t token = p.tokens[row * p.ld_tokens + i];
    float y = token == -1 ? 0.0f : NAN;
    if (token >= 0 && token < p.vocab) y = r.logprob(to_f32(x[token]));
    p.logprobs[row * p.given + i] = y;
  }
}
__device__ inline void write_top(const TokenLogprobs& p, int64_t row, const Row& r, int place,
                                 uint64_t rank) {
  p.top_tokens[row * p.top + place] = token_of(rank);
  const uint32_t order = static_cast<uint32_t>(rank >> 32);
  p.top_logprobs[row * p.top + place] = r.logprob(order == ~0u ? NAN : value_of(order));
}

// W wavefronts, NV vectors of 16 bytes a thread.  slices: workgroups of a row, of
// `step` vectors each; parts and ranks are theirs if there are several.
template <typename T, int W, int NV>
__global__ __launch_bounds__(64 * W, NV > 8 ? 4 : NV > 4 ? 6 : 8) void logprobs_kernel(
    TokenLogprobs p, int slices, int step, Part* parts, uint64_t* ranks) {
  constexpr int E = per_vector<T>();
  constexpr int N = 64 * W;
  __shared__ u32x4 stage[W][NV + 1];
  __shared__ float tops[W];
  __shared__ float sums[3][W];
  __shared__ uint32_t group[kGroups];
  __shared__ uint64_t found[kMost];
  __shared__ uint64_t best[W];
  __shared__ uint32_t bound;
  __shared__ int count;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // Vectors are aligned: of the row's first and last one a part may lie outside.
  // Those two are read element by element, by the first slice's threads 0 and 1.
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int full0 = skew > 0 ? 1 : 0, full1 = (p.vocab + skew) / E;   // whole ones
  const int v0 = full0 + slice * step, v1 = min(v0 + step, full1);
  const int first_token = slice == 0 ? 0 : v0 * E - skew;
  const u32x4* vectors = reinterpret_cast<const u32x4*>(x - skew);
  // The token of element j of the thread's vector n (below 0: none).
  const int lone = slice > 0 ? -1 : tid == 0 && skew > 0 ? 0
                                : tid == 1 && full1 >= full0 && full1 * E < p.vocab + skew ? full1
                                                                                          : -1;
  auto token_at = [&](int thread_lone, int thread, int n, int j) {
    return (n == NV ? thread_lone : v0 + n * N + thread) * E - skew + j;
  };

  u32x4 raw[NV + 1];
  {
    const uint32_t none = minus_infinity<T>();
    raw[NV] = u32x4{none, none, none, none};
  }
  if (lone >= 0) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int token = lone * E - skew + j;
      if (token < 0 || token >= p.vocab) continue;
      if constexpr (std::is_same<T, float>::value) {
        raw[NV][j] = __float_as_uint(x[token]);
      } else {
        const uint32_t b = reinterpret_cast<const uint16_t*>(x)[token];
        const uint32_t w = raw[NV][j >> 1];
        raw[NV][j >> 1] = (j & 1) ? (w & 0xffffu) | b << 16 : (w & 0xffff0000u) | b;
      }
    }
  }
  // Every thread loads every vector, one behind the slice's end its last: without
  // branches the first are used while the others are in flight.
  if (v0 < v1) {
#pragma unroll
    for (int n = 0; n < NV; ++n) raw[n] = vectors[min(v0 + n * N + tid, v1 - 1)];
  }
  if (tid == 0) count = 0;

  // sum = sum of 2^t, spread = sum of t 2^t with t = (x - ref) log2(e).
  float top = -INFINITY, ref = 0.0f, sum = 0.0f, spread = 0.0f;
#pragma unroll
  for (int n = 0; n <= NV; ++n) {
    if (n == NV ? lone < 0 : v0 + n * N + tid >= v1) continue;
    float most = element<T>(raw[n], 0);
#pragma unroll
    for (int j = 1; j < E; ++j) most = fmaxf(most, element<T>(raw[n], j));
    if ((most - ref) * kLog2e > kSlack || (top == -INFINITY && most > -INFINITY)) {
      const float next = fminf(most, 3.40282347e38f);   // of infinities the sums are NaN
      const float t = (ref - next) * kLog2e, f = exp2_hw(t);
      const bool none = sum == 0.0f || f == 0.0f;
      spread = none ? 0.0f : (spread + t * sum) * f;
      sum = sum == 0.0f ? 0.0f : sum * f;
      ref = next;
    }
    top = fmaxf(top, most);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float t = (element<T>(raw[n], j) - ref) * kLog2e;
      const float e = exp2_hw(t);
      sum += e;
      // A logit of -inf adds 0, one of NaN is in e.
      spread = __builtin_fmaf(fmaxf(t, -200.0f), e, spread);
    }
  }

  // The largest of the workgroup and of each group of threads.
  {
    float most = top;
#pragma unroll
    for (int w = 1; w < N / kGroups; w <<= 1) most = fmaxf(most, __shfl_xor(most, w));
    if (p.top > 1 && tid % (N / kGroups) == 0) group[tid / (N / kGroups)] = order_of(most);
    most = wave_max(most);
    if (lane == 0) tops[wave] = most;
  }
  __syncthreads();
  float peak = tops[0];
#pragma unroll
  for (int w = 1; w < W; ++w) peak = fmaxf(peak, tops[w]);
  if (p.top > 1 && wave == 0) {
    uint32_t g[kGroups / 64];
#pragma unroll
    for (int i = 0; i < kGroups / 64; ++i) g[i] = group[lane + 64 * i];
    const uint32_t t = kth_order<16>(g, p.top);
    if (lane == 0) bound = t;
  }

  // One thread's logits, spread over its wavefront: f(logit, token) of each.
  auto spread_out = [&](int from, auto f) __attribute__((always_inline)) {
    __builtin_amdgcn_wave_barrier();
    if (lane == from) {
#pragma unroll
      for (int n = 0; n <= NV; ++n) stage[wave][n] = raw[n];
    }
    const int its = __builtin_amdgcn_readlane(lone, from);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const T* values = reinterpret_cast<const T*>(stage[wave]);
#pragma unroll
    for (int i = 0; i < (NV + 1) * E; i += 64) {
      const int at = i + lane, n = at / E;
      if (at >= (NV + 1) * E || (n == NV ? its < 0 : v0 + n * N + wave * 64 + from >= v1)) continue;
      const int token = token_at(its, wave * 64 + from, n, at % E);
      if (token >= 0 && token < p.vocab) f(to_f32(values[at]), token);
    }
    __builtin_amdgcn_wave_barrier();
  };

  // The thread's logits from memory again, f(logit, token) of each in vectors of which
  // one is wanted (in a loop that keeps no registers for them).
  auto each_again = [&](auto wanted, auto f) __attribute__((always_inline)) {
    auto look = [&](int vector) {
#pragma unroll 1
      for (int j = 0; j < E; ++j) {
        const int token = vector * E - skew + j;
        if (token >= 0 && token < p.vocab) f(to_f32(x[token]), token);
      }
    };
#pragma unroll 1
    for (int i = v0 + tid; i < v1; i += N) {
      const u32x4 v = vectors[i];
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) any = any || wanted(element<T>(v, j));
      if (any) look(i);
    }
    if (lone >= 0) look(lone);
  };

  const float m = peak == -INFINITY ? 0.0f : peak;
  float equal = 0.0f;
  {
    // From the thread's reference to the row's: t grows by (ref - m) log2(e).
    const float t = (ref - m) * kLog2e, f = exp2_hw(t);
    const bool nan = sum != sum;
    spread = sum == 0.0f || f == 0.0f ? 0.0f : -(spread + t * sum) * f * kLn2;
    sum = sum == 0.0f ? 0.0f : sum * f;   // f may be infinite for a thread without logits
    const bool holds = top == peak && top > -INFINITY && !nan;
    uint64_t holders = __ballot(holds);
    if (holds) sum = spread = 0.0f;
    auto add = [&](float y, int) {
      const float d = y - m, e = exp2_hw(d * kLog2e);
      if (d == 0.0f) {
        equal += 1.0f;
      } else {
        sum += e;
        spread -= fmaxf(d, -200.0f) * e;
      }
    };
    if (__popcll(holders) > kFewHolders) {
      // Many equal ones: each reads its own again.
      if (holds) each_again([](float) { return true; }, add);
    } else {
      while (holders != 0) {
        const int from = __ffsll(static_cast<unsigned long long>(holders)) - 1;
        holders &= holders - 1;
        spread_out(from, add);
      }
    }
    const float s = wave_sum(sum), d = wave_sum(spread), n = wave_sum(equal);
    if (lane == 0) {
      sums[0][wave] = s;
      sums[1][wave] = d;
      sums[2][wave] = n;
    }
  }
  const bool odd = sum != sum;   // the thread holds a NaN or an infinity
  __syncthreads();
  float all = 0.0f, wide = 0.0f, same = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    all += sums[0][w];
    wide += sums[1][w];
    same += sums[2][w];
  }
  const Row r = finish(peak, same, all, wide);
  if (slices == 1) {
    if (tid == 0 && p.entropy != nullptr) p.entropy[row] = r.entropy;
    write_given<T>(p, row, r, tid, N);
  } else if (tid == 0) {
    parts[blockIdx.x] = Part{peak, same, all, wide};
  }
  if (p.top == 0) return;

  // The bound's own order may be that of a NaN's bits below -inf.
  float least = p.top == 1 ? peak : bound <= 0x007fffffu ? -INFINITY : value_of(bound);
  // Of the tokens at -inf only the first `top` can be among the top ones.
  bool above = false;   // and those at the bound are none
  auto below = [&](float y) { return y < least || (above && y == least); };
  auto offer = [&](float y, int token) {
    if (below(y) || (y == -INFINITY && token >= first_token + p.top)) return;
    const int at = atomicAdd(&count, 1);
    if (at < kMost) found[at] = rank_of(y, token);
  };
  const bool holds = !(top < least) || odd;
  uint64_t holders = __ballot(holds);
  if (__popcll(holders) <= kFewHolders) {
    while (holders != 0) {
      const int from = __ffsll(static_cast<unsigned long long>(holders)) - 1;
      holders &= holders - 1;
      spread_out(from, offer);
    }
  } else if (holds) {
    // Each looks through its own, a vector at a time.
#pragma unroll
    for (int n = 0; n <= NV; ++n) {
      if (n == NV ? lone < 0 : v0 + n * N + tid >= v1) continue;
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) any = any || !(element<T>(raw[n], j) < least);
      if (!any) continue;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int token = token_at(lone, tid, n, j);
        if (token >= 0 && token < p.vocab) offer(element<T>(raw[n], j), token);
      }
    }
  }
  __syncthreads();
  auto write = [&](int place, uint64_t rank) {
    if (slices == 1)
      write_top(p, row, r, place, rank);
    else
      ranks[static_cast<int64_t>(blockIdx.x) * p.top + place] = rank;
  };
  int n = count;
  const int last_token = slices == 1 ? p.vocab : max(v1 * E - skew, first_token);
  // The first of several slices has the row's last tokens too.
  const int more = slices > 1 && slice == 0 ? p.vocab - (full1 * E - skew) : 0;
  auto nth_token = [&](int i) { return i < last_token ? i : i - last_token + full1 * E - skew; };
  // Rare: too many candidates, where few groups hold a logit or masked logits are the
  // type's lowest value.  Those from the top-th largest maximum of a thread on, then,
  // where too many are equal to that, those above it and its first tokens.  The slice
  // is read again (kept in registers for this, it does not fit them).
  for (int round = 1; n > kMost && round <= 2; ++round) {
    __syncthreads();
    if (round == 1) {
      uint32_t* maxima = reinterpret_cast<uint32_t*>(found);
      maxima[tid] = order_of(top);
      __syncthreads();
      if (wave == 0) {
        uint32_t g[W];
#pragma unroll
        for (int i = 0; i < W; ++i) g[i] = maxima[lane + 64 * i];
        const uint32_t t = kth_order<0>(g, p.top);
        if (lane == 0) bound = t;
      }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    least = value_of(bound);
    above = round == 2;
    // (No more than that they are too many is to be known.)
    if (!below(top) || odd)
      each_again([&](float y) { return !below(y) && *static_cast<volatile int*>(&count) <= kMost; },
                 offer);
    __syncthreads();
    n = count;
  }
  if (above && n < p.top) {
    for (int i0 = first_token; n < p.top && i0 < last_token + more; i0 += N) {
      const int i = i0 + tid, token = nth_token(i);
      const bool equal = i < last_token + more && to_f32(x[token]) == least;
      const uint64_t in = __ballot(equal);
      if (lane == 0) best[wave] = __popcll(in);
      __syncthreads();
      int at = n + __popcll(in & ((uint64_t{1} << lane) - 1)), upto = n;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < wave) at += static_cast<int>(best[w]);
        upto += static_cast<int>(best[w]);
      }
      if (equal && at < p.top) found[at] = rank_of(least, token);
      n = min(upto, p.top);
      __syncthreads();
    }
  }
  if (n > kMany && n <= kMost) {
    // Few groups hold a logit, or many logits are equal: the candidates from the
    // top-th largest rank on, found bit by bit, are `top` exactly.
    if (wave == 0) {
      uint64_t mine[kMost / 64];
#pragma unroll
      for (int i = 0; i < kMost / 64; ++i) mine[i] = lane + 64 * i < n ? found[lane + 64 * i] : 0;
      // Bits that are the same in all of them are known.
      const uint64_t any = found[0];
      uint64_t differ = 0;
#pragma unroll
      for (int i = 0; i < kMost / 64; ++i) differ |= lane + 64 * i < n ? mine[i] ^ any : 0;
#pragma unroll
      for (int w = 1; w < 64; w <<= 1)
        differ |= __shfl_xor(static_cast<unsigned long long>(differ), w);
      uint64_t t = any & ~differ;
#pragma unroll 1
      for (int bit = 63; bit >= 0; --bit) {
        if (!((differ >> bit) & 1)) continue;
        // Above this bit t is the rank's own, below it the least with the known bits.
        const uint64_t next = (t | uint64_t{1} << bit) & (~uint64_t{0} << bit);
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kMost / 64; ++i) reach += __popcll(__ballot(mine[i] >= next));
        if (reach >= p.top) t |= uint64_t{1} << bit;
      }
      uint32_t kept = 0;
#pragma unroll
      for (int i = 0; i < kMost / 64; ++i) {
        const uint64_t in = __ballot(mine[i] >= t);
        if (mine[i] >= t) found[kept + __popcll(in & ((uint64_t{1} << lane) - 1))] = mine[i];
        kept += __popcll(in);
      }
    }
    n = p.top;
    __syncthreads();
  }
  if (n <= kMost) {
    rank_all(found, n, tid, N, [&](int place, uint64_t rank) {
      if (place < p.top) write(place, rank);
    });
    for (int i = n + tid; i < p.top; i += N) write(i, 0);   // a short slice
    return;
  }
  // Rare (thousands of NaN): the slice's logits are read again for each place.  A NaN of
  // token 0 has the largest rank that there is, so the first place takes any.
  uint64_t last = ~uint64_t{0};
  for (int place = 0; place < p.top; ++place) {
    uint64_t mine = 0;
    for (int i = first_token + tid; i < last_token + more; i += N) {
      const int token = nth_token(i);
      const uint64_t rank = rank_of(to_f32(x[token]), token);
      if ((place == 0 || rank < last) && rank > mine) mine = rank;
    }
    mine = wave_max64(mine);
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    mine = best[0];
#pragma unroll
    for (int w = 1; w < W; ++w) mine = best[w] > mine ? best[w] : mine;
    __syncthreads();
    last = mine;
    if (tid == 0) write(place, mine);
  }
}

// One workgroup per row: its slices' sums, given tokens and top tokens.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void logprobs_join_kernel(TokenLogprobs p, int slices,
                                                                     const Part* parts,
                                                                     const uint64_t* ranks) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  parts += row * slices;
  ranks += row * slices * p.top;
  float peak = -INFINITY;
  for (int i = 0; i < slices; ++i) peak = fmaxf(peak, parts[i].top);
  float equal = 0.0f, sum = 0.0f, spread = 0.0f;
  for (int i = 0; i < slices; ++i) {
    const Part s = parts[i];
    if (s.top == peak) {
      equal += s.equal;
      sum += s.sum;
      spread += s.spread;
    } else {
      const float d = peak - s.top, f = exp2_hw(-d * kLog2e);
      const float part = (s.sum + s.equal) * f;
      sum += part;
      spread += s.spread * f + (part == 0.0f ? 0.0f : d * part);
    }
  }
  const Row r = finish(peak, equal, sum, spread);
  if (tid == 0 && p.entropy != nullptr) p.entropy[row] = r.entropy;
  write_given<T>(p, row, r, tid, kJoinThreads);
  if (p.top == 0) return;
  // 0 stands behind the ranks of a short slice.
  __shared__ uint64_t all[kMaxSlices * kLogprobsMaxTop];
  const int n = slices * p.top;
  for (int i = tid; i < n; i += kJoinThreads) all[i] = ranks[i];
  __syncthreads();
  rank_all(all, n, tid, kJoinThreads, [&](int place, uint64_t rank) {
    if (place < p.top && rank != 0) write_top(p, row, r, place, rank);
  });
}

// How a row is cut: slices of `step` vectors.  A workgroup of 16 wavefronts holds
// 16384 vectors but has its CU to itself, so that nothing covers its loads: rows that
// need so many are cut in two, for two workgroups on a CU, once there are two rows
// per CU (1024 rows of 128256 bfloat16 logits: 61 against 70 us, with 20 top tokens
// 79 against 84; 256 rows: 21 against 19, 29 against 24), and so is any row that is
// cut at all (8 rows of 262144: 12 against 16 us).
struct Cut {
  int slices, step;
};
constexpr int kMostVectors = 16 * 64 * 16;
constexpr int kShared = 8 * 64 * 16;   // of a workgroup that shares its CU
constexpr int64_t kManyRows = 512;
static_assert(kLogprobsMaxVocab / 4 / kShared <= kMaxSlices);
Cut cut_of(int64_t rows, int64_t vocab, int dtype) {
  const int64_t vectors = std::max<int64_t>(vocab / (dtype == kF32 ? 4 : 8), 1);   // whole ones
  const bool alone = vectors <= kMostVectors && rows <= kManyRows;
  const int64_t slices = ceil_div(vectors, alone ? kMostVectors : kShared);
  return Cut{static_cast<int>(slices), static_cast<int>(ceil_div(vectors, slices))};
}
int64_t parts_bytes(int64_t items) { return items * static_cast<int64_t>(sizeof(Part)); }

template <typename T>
hipError_t launch_t(const TokenLogprobs& p, const Cut& c, hipStream_t st) {
  Part* parts = static_cast<Part*>(p.workspace);
  uint64_t* ranks = reinterpret_cast<uint64_t*>(static_cast<char*>(p.workspace) +
                                                parts_bytes(p.rows * c.slices));
  const dim3 grid(static_cast<uint32_t>(p.rows * c.slices));
  auto go = [&](auto waves, auto nv) {
    constexpr int W = decltype(waves)::value, NV = decltype(nv)::value;
    hipLaunchKernelGGL((logprobs_kernel<T, W, NV>), grid, dim3(64 * W), 0, st, p, c.slices, c.step,
                       parts, ranks);
  };
  using std::integral_constant;
  const integral_constant<int, 4> w4;
  const integral_constant<int, 8> w8;
  const integral_constant<int, 16> w16;
  if (c.step <= 256)
    go(w4, integral_constant<int, 1>{});
  else if (c.step <= 1024)
    go(w4, integral_constant<int, 4>{});
  else if (c.step <= 4096)
    go(w8, integral_constant<int, 8>{});
  else if (c.step <= 8192)
    go(w8, integral_constant<int, 16>{});
  else
    go(w16, integral_constant<int, 16>{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || c.slices == 1) return e;
  hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3(static_cast<uint32_t>(p.rows)),
                     dim3(kJoinThreads), 0, st, p, c.slices, parts, ranks);
  return hipGetLastError();
}

}  // namespace

int64_t token_logprobs_workgroups(int64_t rows, int64_t vocab, int dtype) {
  return rows * cut_of(rows, vocab, dtype).slices;
}

int64_t token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  const Cut c = cut_of(rows, vocab, dtype);
  if (c.slices == 1) return 0;
  return parts_bytes(rows * c.slices) + rows * c.slices * top * 8;
}

hipError_t launch_token_logprobs(const TokenLogprobs& p, int dtype, hipStream_t st) {
  const Cut c = cut_of(p.rows, p.vocab, dtype);
  if (dtype == kF32) return launch_t<float>(p, c, st);
  if (dtype == kF16) return launch_t<__half>(p, c, st);
  return launch_t<__hip_bfloat16>(p, c, st);
}

}  // namespace w8a8
