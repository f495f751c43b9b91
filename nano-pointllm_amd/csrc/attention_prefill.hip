// Causal attention of prompts and prompt chunks over a paged key-value cache
// (gfx950).
//
// Mathematics.  Rows (token, query head of one key head) are the columns of
// S^T = K Q^T; P = 2^(S^T c - r) with c = scale log2(e) and a running reference
// r per row (Reference in attention_common.h), rounded to the rows' type; O^T =
// V^T P and l = sum P over the rounded values; the result is O / l.  The rounding
// of P is the one that is not forced: half a step each, independent of each other
// and the same in O and l, it leaves 1.3 to 1.4 times the error of the rounded
// result alone, where P in two parts would double the second product.
//
// Bound by the matrix units and the exponentials together: per 32 keys and 32
// rows of 128 elements a wavefront issues 16 matrix instructions of 32 cycles
// and 400 to 450 cycles of vector work, which run side by side only as far as
// the order of the instructions lets them.  8192 tokens of 32 heads: 0.58 to
// 0.60 ms (0.64 on one card of many), 0.92 to 0.95 PFLOP/s, 77 to 79% of what a
// large matrix product reaches; the matrix units are busy 47% of the time and
// the vector units 42%, at a clock that this load holds at 1.9 to 2.0 GHz.  LDS is busy for a quarter of the time, so
// copying ahead by three units instead of one changes nothing, and neither does
// a barrier for every second unit only.
//
// Design:
//   * A workgroup takes 128 rows of one key head, 32 per wavefront, held in
//     registers; the queries that share a key head are packed as rows, so a
//     short chunk fills its tiles and every key is read once per 128 rows.  Two
//     workgroups share a CU: alone one takes 0.77 us per unit, two 1.2 us for
//     one each.
//   * Units of 32 keys and of 32 values pass through double buffers in LDS,
//     filled by LDS-DMA buffer loads straight from the pages, a unit ahead of
//     their use: a wavefront forms one descriptor per operand and unit, whose
//     range ends at the sequence's last key, so what lies behind it arrives as
//     zeros.  16-byte chunks are permuted by key (in the source address), which
//     leaves the reads of both operands without bank conflicts.
//   * While a unit's scores become probabilities on the vector unit, the
//     matrix unit forms the next one's scores; the product of the unit before
//     with its values comes first, with the operands of both read ahead.
//   * The score tile's registers are the second product's operand as they
//     are: its inner index is summed over, so the values are read (transposing
//     ds_read_b64_tr_b16) in the key order that the scores have.
//   * Masks are formed for the units that a row of the wavefront sees in part,
//     the last ones; the others have none.
//   * Few rows far into a long cache are cut over its length: each piece
//     leaves (O, r, l) in the workspace and prefill_join_kernel adds them up.
//     Whether there may be pieces the host decides by the table's width: 560
//     rows over a table of 2048 keys or more take 21.1 us instead of 18.8, for a
//     join that finds nothing to do.
//   * A masked key's probability is 0, but 0 times an infinite or NaN value is
//     NaN.  Such values are not searched for: a row whose sums are not finite
//     is computed again by careful_rows, key by key.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"

namespace w8a8 {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const int32_t __attribute__((address_space(4))) const_i32;   // scalar loads

constexpr int kKeys = 32;            // keys of a unit
constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;   // rows of a workgroup
// Below so many workgroups (two per CU) the keys are cut, into pieces of at
// least 16 units: a join costs 4 to 9 us (512 tokens behind 7680, 32 heads over 8:
// 78 + 8 us in 4 pieces, 179 whole).
constexpr int kSlots = 512;
constexpr int kMinUnits = 16;
// While there is no workgroup for every CU, into pieces of 8 units and more (4
// tokens behind 4000, 32 heads over 8: 13 + 4 us, in pieces of 16 19 + 4; back to
// back in a graph 4 behind 600, 19 units: 15.8 in two pieces, 20.0 whole; 150
// behind 500, 21 units: 19.0 and 21.9; a prompt of 520 rows of 8 heads, 17 units
// at most: 18.9 and 18.3, of 760: 19.4 and 24.3).
constexpr int kCus = 256;
constexpr int kFewUnits = 8;
constexpr int kMaxCut = 32;
// Up to so many workgroups the longest go first: 7 prompts of 146 to 777 tokens,
// 832 workgroups, take 49 us instead of 53; 12 of 432 to 655, 822 workgroups, 36
// instead of 43, 1264 workgroups 54 instead of 58, 1672 workgroups 69 instead of
// 66; 12 of 98 to 655, 1168 workgroups, 46 instead of 49.  More of them even out
// by themselves, and read less when a sequence's run together (12 chunks of 739
// to 1400 tokens of 40 heads, 4200 workgroups: 383 us by sequence, 462 sorted;
// 2072 workgroups: 80 and 84).
constexpr int kSortedItems = 2048;
constexpr int kOutside = 0x7ffffff0;   // a buffer offset past every range
constexpr int kBufferWord3 = 0x00020000;
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 8;          // pieces that a thread of the join has in flight

struct PrefillParams {
  PagedAttention a;
  int group;           // query heads per key head
  int cut;             // most pieces of a row tile
  int few;             // ... of kFewUnits and more
  bool sorted;         // row tiles go by the keys they see, at most 64 sequences
  bool clear;          // rows of no sequence become zeros
  float* part_o;       // [row tiles x kv_heads x cut, kRows, head_dim]
  f32x2* part_rl;      // [row tiles x kv_heads x cut, kRows]
};

// r / group for 0 <= r < 2^31, by a binary32 estimate that is put right.
__device__ inline int divide_rows(int r, int group) {
  if (group == 1) return r;
  int q = static_cast<int>(static_cast<float>(r) / static_cast<float>(group));
  int rest = r - q * group;
  while (rest < 0) {
    --q;
    rest += group;
  }
  while (rest >= group) {
    ++q;
    rest -= group;
  }
  return q;
}

// One row tile: which rows of which sequence, and the keys that they see.
struct Place {
  int seq;      // or -1: the batch has no such tile
  int start;    // the sequence's first row of q
  int count;    // its tokens
  int row0;     // the tile's first row of count x group; without one, the batch's tiles
  int keys;     // the sequence's keys
};

// The batch's row tile number `rank`, every lane gets the same answer.  Sorted:
// those that see the most keys first, of all sequences, so that the short ones
// fill up behind them; else by sequence, the last tile of the last one first.
__device__ inline Place find_tile(const PrefillParams& p, int rank) {
  const int lane = threadIdx.x & 63;
  const PagedAttention& a = p.a;
  struct Seq {
    int start, count, keys, tiles;
  };
  auto read = [&](int b) {
    Seq s{0, 0, 0, 0};
    if (b >= 0 && b < a.batch) {
      s.start = max(a.q_starts[b], 0);
      s.count = max(min(a.q_starts[b + 1], a.tokens) - s.start, 0);
      s.keys = max(0, min(a.lengths[b], a.max_keys));
      s.tiles = static_cast<int>((static_cast<uint32_t>(s.count) * p.group + kRows - 1) / kRows);
    }
    return s;
  };
  // Lane `at` holds sequence `seq`.
  auto place = [&](int seq, const Seq& s, int at, int tile) {
    return Place{seq, lane_value(s.start, at), lane_value(s.count, at), tile * kRows,
                 lane_value(s.keys, at)};
  };
  auto first_lane = [](uint64_t found) {
    return __ffsll(static_cast<unsigned long long>(found)) - 1;
  };
  if (p.sorted) {
    const Seq s = read(lane);
    const int tiles = lane_value(scan64(s.tiles), 63);
    if (tiles <= rank) return Place{-1, 0, 0, tiles, 0};
    if (a.batch == 1) return place(0, s, 0, tiles - 1 - rank);
    // How many of the lane's tiles see fewer than u units: its first ones, up to
    // the first token that sees more than (u - 1) kKeys keys.
    auto fewer = [&](int u) {
      if (u <= 0) return 0;
      const int past = (u - 1) * kKeys - s.keys;
      if (past >= 0) return s.tiles;
      const int token = max(s.count + past, 0);
      return static_cast<int>(static_cast<uint32_t>(token) * p.group / kRows);
    };
    // The most units u that more than `rank` tiles see at least.
    int u = 0, none = (a.max_keys + kKeys - 1) / kKeys + 1, more = 0;
    while (none - u > 1) {
      const int mid = u + (none - u) / 2;
      const int n = lane_value(scan64(s.tiles - fewer(mid)), 63);
      if (n > rank) {
        u = mid;
      } else {
        none = mid;
        more = n;   // tiles that see more than u units, in the end
      }
    }
    const int below = fewer(u);
    const uint32_t equal = fewer(u + 1) - below;
    const uint32_t upto = scan64(equal);
    const int at = first_lane(__ballot(static_cast<int>(upto) > rank - more));
    return place(at, s, at, lane_value(below + rank - more - (upto - equal), at));
  }
  int before = 0;
  for (int b0 = a.batch - 1; b0 >= 0; b0 -= 64) {
    const Seq s = read(b0 - lane);
    const uint32_t upto = scan64(s.tiles);
    const uint64_t found = __ballot(before + static_cast<int>(upto) > rank);
    if (found != 0) {
      const int at = first_lane(found);
      return place(b0 - at, s, at, before + lane_value(upto, at) - 1 - rank);
    }
    before += lane_value(upto, 63);
  }
  return Place{-1, 0, 0, before, 0};
}

// Units of keys that the rows of a tile see, and how many pieces they are cut
// into.
__device__ inline int key_units(const PrefillParams& p, const Place& at) {
  const int last = min(at.row0 + kRows, at.count * p.group) - 1;
  const int seen = at.keys - at.count + divide_rows(last, p.group) + 1;
  return (max(seen, 0) + kKeys - 1) / kKeys;
}
__device__ inline int pieces_of(const PrefillParams& p, int units) {
  return max(1, max(min(p.few, units / kFewUnits), min(p.cut, units / kMinUnits)));
}

template <typename T>
__device__ inline f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, __half>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a),
                                                   __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
}

// Two probabilities rounded to the 16-bit type, packed, and l plus the two
// rounded values.
template <typename T>
__device__ inline uint32_t round2(float p0, float p1, float& l) {
  if constexpr (std::is_same<T, __half>::value) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = __builtin_convertvector(f32x2{p0, p1}, h2);
    l = __builtin_amdgcn_fdot2(v, h2{1, 1}, l, false);
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = __builtin_convertvector(f32x2{p0, p1}, b2);
    l = __builtin_amdgcn_fdot2_f32_bf16(v, b2{1.0f, 1.0f}, l, false);
    return __builtin_bit_cast(uint32_t, v);
  }
}

// 16 bytes per lane from the buffer into LDS at lds + 16 * lane; zeros from
// past its range.
__device__ inline void dma16(__amdgpu_buffer_rsrc_t r, char* lds, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, offset, 0, 0, 0);
}

// The upper 32 lanes of x and the lower 32 of y change places.
__device__ inline void swap_halves(uint32_t& x, uint32_t& y) {
  const auto z = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = z[0];
  y = z[1];
}

// Each 16 lanes read 16 x 8 bytes, four rows of 16 elements (lane i: element
// 4 (i % 4) of row i / 4), and lane i gets element i of the four rows.
__device__ inline u32x2 read_transposed(lds_s16x4* __restrict__ lds) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds));
}

// Chunk permutations of a key's row of DP / 8 chunks of 16 bytes: position =
// chunk ^ swizzle.  Keys: the 32 keys that a matrix operand reads at one chunk
// spread over all banks.  Values: the four keys that a transposing read takes
// at 64 bytes spread over all banks.
template <int DP> __device__ inline int swizzle_k(int key) {
  return DP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int DP> __device__ inline int swizzle_v(int key) {
  return DP == 64 ? ((key >> 1) & 1) << 2 | ((key >> 2) & 3) : (key & 3) << 2 | ((key >> 2) & 3);
}

// Where a row's result goes.
template <typename T>
__device__ inline T* out_row(const PagedAttention& a, int start, int token, int head) {
  return static_cast<T*>(a.out) + (start + token) * a.o_st + head * a.o_sh;
}

// Zeros in the rows of no sequence, those before the first one's and behind the
// last one's: workgroup i of n takes every n-th.
__device__ inline void clear_rows(const PrefillParams& p, int kvh, int i, int n) {
  const PagedAttention& a = p.a;
  const int first = max(0, min(a.q_starts[0], a.tokens));
  const int end = max(first, min(a.q_starts[a.batch], a.tokens));
  const int chunks = a.head_dim / 8;   // of 16 bytes
  for (int64_t r = i; r < first + (a.tokens - end); r += n) {
    uint16_t* row = static_cast<uint16_t*>(a.out) + (r < first ? r : r - first + end) * a.o_st;
    for (int c = threadIdx.x; c < p.group * chunks; c += 64 * kWaves)
      *reinterpret_cast<u32x4*>(row + (kvh * p.group + c / chunks) * a.o_sh + c % chunks * 8) =
          u32x4{0, 0, 0, 0};
  }
}

// The rows of `bad` (bit c: row c of the wavefront's 32), key by key: lane i
// holds elements i, i + 64, ... of the head.  Masked and unknown keys are not
// read.  Rare, so kept simple: 2048 tokens of 32 heads that all see a NaN take 42
// ms (64 keys at a time, 23 ms).
template <typename T, int DP>
__device__ inline void careful_rows(const PrefillParams& p, const Place& at, int kvh,
                                    int wave_row, uint32_t bad, int k0, int k1, int64_t item,
                                    bool whole) {
  constexpr int N = DP / 64;
  const PagedAttention& a = p.a;
  const int lane = threadIdx.x & 63;
  const int D = a.head_dim;
  const float sc = a.scale * kLog2e;
  const int32_t* table = a.table + at.seq * a.ld_table;
  while (bad != 0) {
    const int c = __ffs(bad) - 1;
    bad &= bad - 1;
    const int row = wave_row + c;
    const int token = divide_rows(row, p.group);
    const int head = kvh * p.group + row - token * p.group;
    const T* q = static_cast<const T*>(a.q) + (at.start + token) * a.q_st + head * a.q_sh;
    float qv[N], o[N] = {}, ref = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) qv[i] = lane + 64 * i < D ? to_f32(q[lane + 64 * i]) : 0.0f;
    const int end = min(k1, at.keys - at.count + token + 1);
    for (int j = k0; j < end; ++j) {
      const int page = table[j >> a.page_shift];
      if (page < 0 || page >= a.pages) continue;
      const int64_t off = page * a.c_page + kvh * a.c_head +
                          (j & ((1 << a.page_shift) - 1)) * a.c_tok;
      float s = 0.0f, v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = lane + 64 * i;
        v[i] = d < D ? to_f32(static_cast<const T*>(a.v)[off + d]) : 0.0f;
        if (d < D) s += qv[i] * to_f32(static_cast<const T*>(a.k)[off + d]);
      }
#pragma unroll
      for (int w = 1; w < 64; w <<= 1) s += __shfl_xor(s, w);
      s *= sc;
      const float next = fmaxf(ref, s - Reference<T>::kBelow);
      const float base = next == -INFINITY ? 0.0f : next;
      const float f = exp2_hw(ref - base), w = exp2_hw(s - base);
      ref = next;
      l = l * f + w;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = o[i] * f + w * v[i];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t r = item * kRows + row % kRows;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) continue;
      if (whole)
        out_row<T>(a, at.start, token, head)[d] = from_f32<T>(o[i] * inv);
      else
        p.part_o[r * D + d] = o[i];
    }
    if (!whole && lane == 0) p.part_rl[r] = f32x2{ref, l};
  }
}

// DU: head_dim rounded up to 64, 96, 128 or 256, what the products run over (4096
// tokens of 32 heads of 96 elements: 136 us, over 128 elements 157); DP: the
// power of two that a key's row takes in LDS.  DMA: pages of at least 8
// keys, the part of a unit that a wavefront copies; else each chunk is copied
// through registers.
template <typename T, int DP, int DU, bool DMA>
__global__ __launch_bounds__(64 * kWaves, DP == 256 ? 1 : 2) void prefill_kernel(PrefillParams p) {
  constexpr int KS = DU / 16;               // first product: steps over the head
  constexpr int DT = DU / 32;               // second product: row tiles of O^T
  constexpr int RB = DP * 2;                // bytes of a key's row
  constexpr int RL = 1024 / RB;             // keys of a load
  constexpr int NL = kKeys / RL / kWaves;   // loads per wavefront, unit and operand
  constexpr int UB = kKeys * RB;            // bytes of a unit of one operand
  // Four arrays, so that the compiler sees that one is read while loads into
  // the others are in flight.
  __shared__ __align__(16) char k0[UB], k1[UB], v0[UB], v1[UB];
  __shared__ int odd_pages[kWaves];

  const PagedAttention& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5;
  // Consecutive workgroups, key heads here, go to the eight dies in turn (a die's
  // workgroups on one head at a time instead, for its L2, measures the same).
  const int kvh = blockIdx.x % a.kv_heads;
  const Place at = find_tile(p, blockIdx.x / a.kv_heads);
  if (at.seq < 0) {
    if (p.clear && blockIdx.y == 0)
      clear_rows(p, kvh, blockIdx.x / a.kv_heads - at.row0, gridDim.x / a.kv_heads - at.row0);
    return;
  }
  const int all_units = key_units(p, at);
  const int pieces = pieces_of(p, all_units);
  const int piece = blockIdx.y;
  if (piece >= pieces) return;
  const int u0 = __builtin_amdgcn_readfirstlane(
      static_cast<int>(static_cast<int64_t>(all_units) * piece / pieces));
  const int u1 = __builtin_amdgcn_readfirstlane(
      static_cast<int>(static_cast<int64_t>(all_units) * (piece + 1) / pieces));
  const int D = a.head_dim;
  const int total_rows = at.count * p.group;
  const int wave_row = at.row0 + 32 * wave;
  const int row = min(wave_row + c, total_rows - 1);
  const bool live = wave_row + c < total_rows;
  const int token = divide_rows(row, p.group);
  const int head = kvh * p.group + row - token * p.group;
  const int seen = live ? at.keys - at.count + token : -1;   // the row's last key
  // The first row's and the last row's last key of the wavefront.
  const int seen_first = __builtin_amdgcn_readlane(seen, 0);
  const int seen_last = __builtin_amdgcn_readlane(
      seen, max(0, min(31, total_rows - 1 - wave_row)));
  // The wavefront's units end here; it copies and waits to u1 with the others.
  const int end =
      __builtin_amdgcn_readfirstlane(max(u0, seen_last < 0 ? 0 : min(u1, seen_last / kKeys + 1)));

  // Loading: lane's key within a load and its chunk's position there.
  const int lk = lane / (RB / 16), lp = lane % (RB / 16);
  const_i32* table = (const_i32*)(a.table + at.seq * a.ld_table);
  const int page_mask = (1 << a.page_shift) - 1;
  const int ctok = static_cast<int>(a.c_tok);   // DMA: a page stays below 2^31 elements
  const int pages = static_cast<int>(a.pages);
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + kvh * a.c_head;
  const uint16_t* vb = static_cast<const uint16_t*>(a.v) + kvh * a.c_head;
  int off_k[NL], off_v[NL];
#pragma unroll
  for (int m = 0; m < NL; ++m) {
    const int key = (wave * NL + m) * RL + lk;
    const int ck = (lp ^ swizzle_k<DP>(key)) * 8, cv = (lp ^ swizzle_v<DP>(key)) * 8;
    off_k[m] = ck < D ? ((m * RL + lk) * ctok + ck) * 2 : kOutside;
    off_v[m] = cv < D ? ((m * RL + lk) * ctok + cv) * 2 : kOutside;
  }
  // A wavefront copies eight keys of a unit.  DMA: they lie in one page, whose
  // place (of keys and of values) is formed once, in scalar registers; rows
  // past the sequence's last key and of unknown pages arrive as zeros (unless
  // the cache's rows share elements: masked all the same).
  const int first_key = wave * (kKeys / kWaves);
  struct Source {
    int64_t offset;   // elements
    int range;        // bytes
  };
  auto lookup = [&](int u) __attribute__((always_inline)) {
    return DMA ? table[min(u * kKeys + first_key, at.keys - 1) >> a.page_shift] : 0;
  };
  auto locate = [&](int u, int page) __attribute__((always_inline)) {
    const int key = u * kKeys + first_key;
    const int left = at.keys - key;
    const bool known = left > 0 && static_cast<uint32_t>(page) < static_cast<uint32_t>(pages);
    return Source{known ? page * a.c_page + (key & page_mask) * ctok : int64_t{0},
                  known ? ((left < 8 ? left : 8) - 1) * (2 * ctok) + 2 * D : 0};
  };
  auto copy = [&](int u, const Source& src, const uint16_t* cache, const int (&off)[NL],
                  char* dst, auto is_key) __attribute__((always_inline)) {
    char* to = dst + wave * NL * 1024;
    if constexpr (DMA) {
      // Told to be uniform: values carried around the loop may sit in vector
      // registers, and a descriptor there would cost a loop over the lanes.
      const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(src.offset));
      const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(src.offset >> 32));
      const int64_t offset = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(cache + offset), 0, __builtin_amdgcn_readfirstlane(src.range),
          kBufferWord3);
#pragma unroll
      for (int m = 0; m < NL; ++m) dma16(r, to + m * 1024, off[m]);
    } else {
#pragma unroll
      for (int m = 0; m < NL; ++m) {
        const int in_unit = first_key + m * RL + lk;
        const int key = u * kKeys + in_unit;
        int page = -1;
        if (key < at.keys) page = a.table[at.seq * a.ld_table + (key >> a.page_shift)];
        const int chunk =
            (lp ^ (decltype(is_key)::value ? swizzle_k<DP>(in_unit) : swizzle_v<DP>(in_unit))) * 8;
        u32x4 x{0, 0, 0, 0};
        if (page >= 0 && page < pages && chunk < D)
          x = *reinterpret_cast<const u32x4*>(cache + page * a.c_page +
                                              (key & page_mask) * a.c_tok + chunk);
        *reinterpret_cast<u32x4*>(to + m * 1024 + lane * 16) = x;
      }
    }
  };
  auto copy_k = [&](int u, const Source& src, char* dst) __attribute__((always_inline)) {
    copy(u, src, kb, off_k, dst, std::true_type{});
  };
  auto copy_v = [&](int u, const Source& src, char* dst) __attribute__((always_inline)) {
    copy(u, src, vb, off_v, dst, std::false_type{});
  };
  // At most N of this wavefront's loads are in flight, so are the others', and
  // every wavefront has read what it was reading.  The wait is the builtin,
  // which the compiler's own insertion of waits follows.
  auto arrived = [&](auto n) __attribute__((always_inline)) {
    constexpr int N = decltype(n)::value;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));   // lgkmcnt(0) too
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float ref = -INFINITY, l = 0.0f;

  if (u0 < u1) {
    // The places of the two units whose values come next; the page of the one
    // whose keys do.
    Source source = locate(u0, lookup(u0)), source_1 = locate(u0 + 1, lookup(u0 + 1));
    int page = lookup(u0 + 2);
    copy_k(u0, source, k0);
    copy_k(u0 + 1, source_1, k1);
    auto copies = [&](int i, char* kfree, char* vn) __attribute__((always_inline)) {
      const Source source_2 = locate(i + 2, page);
      copy_k(i + 2, source_2, kfree);
      copy_v(i, source, vn);
      source = source_1;
      source_1 = source_2;
    };

    // Values of the unit before the first.
    for (int i = threadIdx.x * 16; i < UB; i += 64 * kWaves * 16)
      *reinterpret_cast<u32x4*>(v1 + i) = u32x4{0, 0, 0, 0};
    // Whether a page of these keys is unknown: then every unit looks its keys
    // up.
    int odd = 0;
    {
      const int n = ((min(u1 * kKeys, at.keys) - 1) >> a.page_shift) + 1;
      for (int i = (u0 * kKeys >> a.page_shift) + threadIdx.x; i < n; i += 64 * kWaves) {
        const int page = a.table[at.seq * a.ld_table + i];
        odd |= page < 0 || page >= a.pages;
      }
      const bool any = __any(odd);
      if (lane == 0) odd_pages[wave] = any;
    }
    // Queries, negated for a negative scale so that the one below is not, and
    // zeros for a scale of zero.
    u32x4 qf[KS];
    {
      const uint16_t* q =
          static_cast<const uint16_t*>(a.q) + (at.start + token) * a.q_st + head * a.q_sh + 8 * h;
      const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[s] = u32x4{0, 0, 0, 0};
        if (live && a.scale != 0.0f && 16 * s + 8 * h < D)
          qf[s] = *reinterpret_cast<const u32x4*>(q + 16 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[s][i] ^= flip;
      }
    }
    const float sc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;

    // Reading: byte offsets of the operands in a unit.
    int read_k[KS], read_v[DT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) read_k[s] = c * RB + (((2 * s + h) ^ swizzle_k<DP>(c)) * 16);
    {
      const int i = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = 8 * b + 4 * h + (i >> 2);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          read_v[d][b] = key * RB +
                         (((4 * d + 2 * g + ((i & 3) >> 1)) ^ swizzle_v<DP>(key)) * 16) +
                         8 * (i & 1);
      }
    }

    f32x16 even, odd_s;   // scores of this unit and of the next one
    u32x4 pf[2];   // probabilities of the unit before
    pf[0] = pf[1] = u32x4{0, 0, 0, 0};
    auto key_operand = [&](const char* kt, int k) __attribute__((always_inline)) {
      return *reinterpret_cast<const u32x4*>(kt + read_k[k]);
    };
    auto value_operand = [&](char* vt, int u, int d) __attribute__((always_inline)) {
      const u32x2 x = read_transposed((lds_s16x4*)(vt + u * 16 * RB + read_v[d][0]));
      const u32x2 y = read_transposed((lds_s16x4*)(vt + u * 16 * RB + read_v[d][1]));
      return u32x4{x[0], x[1], y[0], y[1]};
    };
    auto weight = [&](f32x16& s, int i, float base) __attribute__((always_inline)) {
      s[i] = exp2_hw(__builtin_fmaf(s[i], sc, base));
    };
    auto weights_of = [&](f32x16& s, int i) __attribute__((always_inline)) {
      pf[i >> 2][i & 3] = round2<T>(s[2 * i], s[2 * i + 1], l);
    };
    arrived(std::integral_constant<int, DMA ? NL : 0>{});
    odd = odd_pages[0] | odd_pages[1] | odd_pages[2] | odd_pages[3];
    odd = __builtin_amdgcn_readfirstlane(odd);
#pragma unroll
    for (int n = 0; n < 16; ++n) even[n] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) even = mfma_32x32x16<T>(key_operand(k0, k), qf[k], even);

    // Unit i: the product of the unit before with its values (zeros for the
    // first), then the scores of the next one while this one's become
    // probabilities.  The order of the instructions is held (sched_barrier):
    // operands are read ahead of their matrix instructions, copies are issued
    // and the vector work is done while those run.
    auto unit = [&](int i, f32x16& s, f32x16& next, char* kn, char* kfree, char* vp, char* vn)
        __attribute__((always_inline)) {
      arrived(std::integral_constant<int, 0>{});
      // Ahead of the SIMD's other wavefront while this one feeds the matrix unit
      // (8192 tokens of 32 heads: 590 against 602 us).
      __builtin_amdgcn_s_setprio(1);
      u32x4 vf[2][DT], kf[KS];
#pragma unroll
      for (int d = 0; d < DT; ++d) vf[0][d] = value_operand(vp, 0, d);
      __builtin_amdgcn_sched_barrier(0);
      copies(i, kfree, vn);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        vf[1][d] = value_operand(vp, 1, d);
        o[d] = mfma_32x32x16<T>(vf[0][d], pf[0], o[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        kf[d] = key_operand(kn, d);
        o[d] = mfma_32x32x16<T>(vf[1][d], pf[1], o[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      const int key0 = i * kKeys;
      if (key0 + kKeys - 1 > seen_first || odd != 0) {
        uint32_t shown = 0xffffu;
        if (odd != 0) {
#pragma unroll 1
          for (int n = 0; n < 16; ++n) {
            const int key = key0 + 8 * (n >> 2) + 4 * h + (n & 3);
            int page = 0;
            if (key < at.keys) page = a.table[at.seq * a.ld_table + (key >> a.page_shift)];
            if (page < 0 || page >= pages) shown &= ~(1u << n);
          }
        }
        const int left = seen - key0 - 4 * h;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const bool there = 8 * (n >> 2) + (n & 3) <= left && ((shown >> n) & 1);
          s[n] = there ? s[n] : -INFINITY;
        }
      }
      float top = s[0];
#pragma unroll
      for (int n = 1; n < 16; ++n) top = fmaxf(top, s[n]);
      top *= sc;
      if (__any(top > ref + Reference<T>::kSlack)) {
        // Raise the reference of the rows that need it; both lanes of a row
        // agree.
        top = fmaxf(top, __shfl_xor(top, 32));
        if (top > ref + Reference<T>::kSlack) {
          const float raised = top - Reference<T>::kBelow;
          const float f = ref == -INFINITY ? 1.0f : exp2_hw(ref - raised);
          ref = raised;
          l *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int n = 0; n < 16; ++n) o[d][n] *= f;
        }
      }
      const float base = ref == -INFINITY ? 0.0f : -ref;
#pragma unroll
      for (int n = 0; n < 16; ++n) next[n] = 0.0f;
      __builtin_amdgcn_sched_barrier(0);
      // Behind matrix instruction k the scores from 16 k / KS on become
      // probabilities, and the pairs of the step before are rounded.
#pragma unroll
      for (int k = 0; k <= KS; ++k) {
        if (k + DT < KS) kf[k + DT] = key_operand(kn, k + DT);
        if (k < KS) next = mfma_32x32x16<T>(kf[k], qf[k], next);
#pragma unroll
        for (int n = 16 * k / KS; n < 16 && n < 16 * (k + 1) / KS; ++n) weight(s, n, base);
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (k > 0 && (n & 1) && n >= 16 * (k - 1) / KS && n < 16 * k / KS) weights_of(s, n >> 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      page = lookup(i + 3);   // waited for with the next unit's copies
    };
    int i = u0;
    while (i < end) {
      unit(i, even, odd_s, k1, k0, v1, v0);
      if (++i >= end) break;
      unit(i, odd_s, even, k0, k1, v0, v1);
      ++i;
    }
    // The last product; then the wavefront only copies, and waits, for the
    // others.
    auto rest = [&](bool last, char* kfree, char* vp, char* vn) __attribute__((always_inline)) {
      arrived(std::integral_constant<int, 0>{});
      if (last) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int d = 0; d < DT; ++d)
            o[d] = mfma_32x32x16<T>(value_operand(vp, u, d), pf[u], o[d]);
      }
      if (i < u1) {
        copies(i, kfree, vn);
        page = lookup(i + 3);
      }
      ++i;
    };
    const int stop = i;
    while (i <= u1) {
      if (((i - u0) & 1) == 0)
        rest(i == stop && i > u0, k0, v1, v0);
      else
        rest(i == stop, k1, v0, v1);
    }
    // No load into LDS outlives the workgroup.
    __builtin_amdgcn_s_waitcnt(0x0f70);
  }

  l += __shfl_xor(l, 32);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * p.cut + piece;
  bool finite = fabsf(l) < INFINITY;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) finite = finite && fabsf(o[d][i]) < INFINITY;
  const uint64_t odd = __ballot(live && !finite);
  const uint32_t bad_rows = static_cast<uint32_t>(odd) | static_cast<uint32_t>(odd >> 32);
  const bool mine = live && !((bad_rows >> c) & 1);
  if (pieces == 1) {
    // Registers 4 j .. 4 j + 3 of O^T tile d are elements 32 d + 8 j + 4 h .. + 3:
    // of two such fours the lanes of a row swap one, and store 16 bytes each.
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* dst = out_row<T>(a, at.start, token, head);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int i = 4 * j + 2 * k;
          w[0][k] = pack2_bits<T>(o[d][i] * inv, o[d][i + 1] * inv);
          w[1][k] = pack2_bits<T>(o[d][i + 4] * inv, o[d][i + 5] * inv);
          swap_halves(w[0][k], w[1][k]);
        }
        const int e = 32 * d + 8 * (j + h);
        if (mine && e < D)
          *reinterpret_cast<u32x4*>(dst + e) = u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
      }
  } else if (mine) {
    const int64_t r = item * kRows + 32 * wave + c;
    if (h == 0) p.part_rl[r] = f32x2{ref, l};
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 32 * d + 8 * j + 4 * h;
        if (e < D)
          *reinterpret_cast<f32x4*>(p.part_o + r * D + e) =
              f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
      }
  }
  if (bad_rows != 0)
    careful_rows<T, DP>(p, at, kvh, wave_row, bad_rows, u0 * kKeys, min(u1 * kKeys, at.keys), item,
                        pieces == 1);
}

// Adds up the pieces of a row tile that was cut: four elements of a row per
// thread, kJoinAhead pieces of them in flight (32 pieces of 16 rows and 8 key
// heads: 6.0 us, one after the other 13.4).
template <typename T, int DP>
__global__ __launch_bounds__(kJoinThreads) void prefill_join_kernel(PrefillParams p) {
  constexpr int C = DP / 4;             // threads of a row
  constexpr int R = kJoinThreads / C;   // rows of a workgroup
  const PagedAttention& a = p.a;
  const int kvh = blockIdx.x % a.kv_heads;
  const Place at = find_tile(p, blockIdx.x / a.kv_heads);
  if (at.seq < 0) return;
  const int pieces = pieces_of(p, key_units(p, at));
  if (pieces == 1) return;
  const int c = threadIdx.x % C;
  const int in_tile = blockIdx.y * R + threadIdx.x / C;
  const int row = at.row0 + in_tile;
  const int D = a.head_dim;
  if (in_tile >= kRows || row >= at.count * p.group) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.cut * kRows + in_tile;
  // Thread c of a row weighs pieces c, c + C, ...
  constexpr int M = (kMaxCut + C - 1) / C;
  f32x2 rl[M];
  float top = -INFINITY;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    rl[m] = f32x2{-INFINITY, 0.0f};
    if (c + m * C < pieces) rl[m] = p.part_rl[r0 + (c + m * C) * kRows];
    top = fmaxf(top, rl[m][0]);
  }
#pragma unroll
  for (int w = 1; w < C; w <<= 1) top = fmaxf(top, __shfl_xor(top, w));
  const float base = top == -INFINITY ? 0.0f : top;
  float weight[M], l = 0.0f;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    weight[m] = exp2_hw(rl[m][0] - base);
    l += rl[m][1] * weight[m];
  }
#pragma unroll
  for (int w = 1; w < C; w <<= 1) l += __shfl_xor(l, w);
  const float* src = p.part_o + r0 * D + 4 * c;
  const int64_t step = static_cast<int64_t>(kRows) * D;
  const bool inside = 4 * c < D;
  f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int m = 0; m < M; ++m)
    for (int i0 = m * C; i0 < min(pieces, (m + 1) * C); i0 += kJoinAhead) {
      f32x4 x[kJoinAhead];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        x[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (inside && i0 + k < pieces)
          x[k] = *reinterpret_cast<const f32x4*>(src + (i0 + k) * step);
      }
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) o += x[k] * __shfl(weight[m], i0 + k, C);
    }
  if (!inside) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int token = divide_rows(row, p.group);
  T* dst = out_row<T>(a, at.start, token, kvh * p.group + row - token * p.group) + 4 * c;
  *reinterpret_cast<u32x2*>(dst) =
      u32x2{pack2_bits<T>(o[0] * inv, o[1] * inv), pack2_bits<T>(o[2] * inv, o[3] * inv)};
}

// Row tiles of a call at most: each sequence's last one may lack kRows - 1 rows.
int64_t max_tiles(int64_t tokens, int64_t batch, int64_t group) {
  return (tokens * group + batch * (kRows - 1)) / kRows;
}

// Pieces of a row tile at most: of kMinUnits while two workgroups per CU are not
// there, of kFewUnits while one is not (few).
int64_t few_of(int64_t items, int64_t max_keys) {
  return std::max<int64_t>(
      1, std::min<int64_t>({kCus / items, ceil_div(max_keys, kKeys) / kFewUnits, kMaxCut}));
}
int64_t cut_of(int64_t items, int64_t max_keys) {
  const int64_t most = ceil_div(max_keys, kKeys) / kMinUnits;
  return std::max(few_of(items, max_keys),
                  std::min<int64_t>({kSlots / items, most, kMaxCut}));
}

int64_t pairs_bytes(int64_t rows) { return ceil_div(rows * 8, 256) * 256; }

template <typename T, int DP, int DU>
hipError_t launch_d(const PrefillParams& p, int64_t items, hipStream_t st) {
  // To clear rows, at least one workgroup per key head without a row tile.
  const dim3 grid(static_cast<uint32_t>(items + (p.clear ? p.a.kv_heads : 0)),
                  static_cast<uint32_t>(p.cut));
  const bool dma = p.a.page_shift >= 3 && (p.a.c_tok << p.a.page_shift) < (int64_t{1} << 30);
  if (dma)
    hipLaunchKernelGGL((prefill_kernel<T, DP, DU, true>), grid, dim3(64 * kWaves), 0, st, p);
  else
    hipLaunchKernelGGL((prefill_kernel<T, DP, DU, false>), grid, dim3(64 * kWaves), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.cut == 1) return e;
  hipLaunchKernelGGL((prefill_join_kernel<T, DP>),
                     dim3(static_cast<uint32_t>(items), kRows * DP / 4 / kJoinThreads),
                     dim3(kJoinThreads), 0, st, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const PrefillParams& p, int64_t items, hipStream_t st) {
  if (p.a.head_dim <= 64) return launch_d<T, 64, 64>(p, items, st);
  if (p.a.head_dim <= 96) return launch_d<T, 128, 96>(p, items, st);
  if (p.a.head_dim <= 128) return launch_d<T, 128, 128>(p, items, st);
  return launch_d<T, 256, 256>(p, items, st);
}

}  // namespace

int64_t paged_prefill_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                int64_t head_dim, int64_t max_keys) {
  if (tokens == 0 || batch == 0) return 0;
  const int64_t items = max_tiles(tokens, batch, q_heads / kv_heads) * kv_heads;
  const int64_t cut = cut_of(items, max_keys);
  if (cut == 1) return 0;
  const int64_t rows = items * cut * kRows;
  return pairs_bytes(rows) + rows * head_dim * 4;
}

hipError_t launch_paged_prefill(const PagedAttention& a, bool clear, int dtype, hipStream_t st) {
  PrefillParams p;
  p.a = a;
  p.clear = clear;
  p.group = a.q_heads / a.kv_heads;
  const int64_t items = max_tiles(a.tokens, a.batch, p.group) * a.kv_heads;
  p.cut = static_cast<int>(cut_of(items, a.max_keys));
  p.few = static_cast<int>(few_of(items, a.max_keys));
  p.sorted = a.batch <= 64 && items <= kSortedItems;
  char* ws = static_cast<char*>(a.workspace);
  p.part_rl = reinterpret_cast<f32x2*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + pairs_bytes(items * p.cut * kRows));
  return dtype == kF16 ? launch_t<__half>(p, items, st) : launch_t<__hip_bfloat16>(p, items, st);
}

}  // namespace w8a8
