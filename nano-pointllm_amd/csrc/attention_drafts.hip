// Attention of small trees of drafted tokens over a paged key-value cache (gfx950):
// up to 64 rows (token, query head) of a sequence and key head on average.
//
// Mathematics.  As attention_decode.hip: S^T = K Q^T, P = 2^(S^T c - r), O^T = V^T P,
// l = sum P, with the rows as columns; a masked key's score is -inf.  P enters the
// second product as two 16-bit parts (split2), so that the result's own rounding is
// the only one that shows: rounded once, in O and l alike, it leaves 1.4 times that
// error (of the norm 2.9e-4 and 2.1e-4 in binary16, 2.3e-3 and 1.7e-3 in bfloat16), and
// the second part's products cost little next to the loads: 8 trees of 25 to 64 35.2
// instead of 34.6 us, 4 of 64 behind 4032 59.8 and 59.4, 32 of 30 to 60 72 and 68, heads
// of 64 55.6 and 52.4.
//
// Bound by memory: every key and value is read once per workgroup's 16 W rows, for up
// to 64 rows.  4 trees of 64 behind 4032 keys of 32 heads (268 MB): 50 us and a join of
// 12, 5.4 TB/s; one of 64 behind 16320: 50 us and a join of 5, back to back 52.5.  8 of
// 25 to 64 behind 630 to 1590 keys (169 MB) are 256 workgroups, of which the longest
// walks 26 steps: 35 to 40 us.  A small call is bound by its launches: 26 rows of 32
// heads behind 601 keys take 9 us and the join 4.  The comparisons below were made
// while more than 32 rows rounded P once.
//
// Design:
//   * A workgroup takes 16 rows per wavefront of one key head, and a piece of the
//     sequence's keys.  Units of 32 keys and values pass through a ring of kStages
//     buffers in LDS, filled by LDS-DMA buffer loads straight from the pages, so that
//     64 KiB per workgroup are in flight without a register (a wavefront that loads
//     its keys itself, as decode does, has no room for 32 rows and the next keys: 54
//     us for the 8 trees).  16-byte chunks are permuted by key (in the source
//     address), which leaves the reads of both operands without bank conflicts.
//   * Two sets of wavefronts (kParts) take every other unit for the same rows, and add
//     up their sums at the end: alone on its SIMD a wavefront waits for each unit's
//     operands, scores and sums in turn (8 trees: 43 us; one of 64 behind 16320 keys:
//     57).
//   * The scores' registers are the second product's operand as they are: its inner
//     index is summed over, so the values are read (transposing) in the key order
//     that the scores have.
//   * Only the units that hold drafted keys have masks: 32 bits per row, loaded a unit
//     ahead.
//   * Work is cut by the keys there are, on the device, into kSlots workgroups and a
//     few, one per CU (512: 66 instead of 57 us for the 4 trees), and joined in a
//     second launch in a fixed order.  Batches that give every CU a workgroup are not
//     cut while their tables are short (the 8 trees cut: 54 us), nor are short
//     sequences.
//   * Keys behind the sequence and of unknown pages arrive as zeros and are masked.  A
//     masked key's probability is 0, but 0 times an infinite or NaN value is NaN: a
//     row whose sums are not finite is computed again key by key.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"

namespace w8a8 {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const int32_t __attribute__((address_space(4))) const_i32;   // scalar loads

constexpr int kTile = 32;          // keys of a unit
constexpr int kParts = 2;          // wavefronts of the same rows, on every other unit
constexpr int kStages = 3;
constexpr int kOutside = 0x7ffffff0;   // a buffer offset past every range
constexpr int kBufferWord3 = 0x00020000;
constexpr int kMinTiles = 4;       // least units of a workgroup of several
constexpr int kWholeTiles = 10;    // sequences up to here are not cut
constexpr int64_t kCus = 256;
constexpr int64_t kWholeKeys = 2048;
constexpr int kSlots = 256;        // workgroups aimed at
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 8;

struct TreeParams {
  PagedAttention a;
  const uint32_t* masks;   // [tokens, ld_masks], bit j of word w: drafted token 32 w + j
  int64_t ld_masks;
  int words;
  int group;               // query heads per key head
  bool whole;              // no sequence is cut
  bool clear;              // rows of no sequence become zeros
  int items;               // that the workspace has room for
  int resident;            // workgroups that the card holds at a time
  float* part_o;           // [items x kv_heads, rows of a block, head_dim]
  f32x2* part_rl;          // [items x kv_heads, rows of a block]
};

// A block of rows of a sequence, and the piece of its keys.
struct Item {
  int seq;      // or -1: `start` is then how many items there are
  int start;    // the sequence's first row of q
  int count;    // its drafted tokens
  int keys;
  int tiles;
  int pieces;   // of each of the sequence's blocks
  int piece;    // which
  int block;    // its number among the sequence's
  int blocks;
  int first;    // the sequence's first item
};

// Item number `at`, pieces of a block side by side, or (join) block number `at`.
// Every lane gets the same answer.
__device__ inline Item find_item(const TreeParams& p, int rows, int at, bool join) {
  const int lane = threadIdx.x & 63;
  const PagedAttention& a = p.a;
  struct Seq {
    int start, count, keys, tiles, blocks;
  };
  auto read = [&](int b) {
    Seq s{0, 0, 0, 0, 0};
    if (b < a.batch) {
      s.start = max(a.q_starts[b], 0);
      s.count = max(min(a.q_starts[b + 1], a.tokens) - s.start, 0);
      s.keys = max(0, min(a.lengths[b], a.max_keys));
      s.tiles = static_cast<int>(static_cast<uint32_t>(s.keys + kTile - 1) / kTile);
      s.blocks = static_cast<int>((static_cast<uint32_t>(s.count) * p.group + rows - 1) / rows);
    }
    return s;
  };
  auto pieces_of = [](uint32_t tiles, uint32_t cut) {
    return tiles <= kWholeTiles ? 1u : (tiles + cut - 1) / cut;
  };
  const Seq first = read(lane);
  uint32_t cut = INT32_MAX;
  if (!p.whole) {
    // A lane's share is kept below 2^25, so that 64 of them fit 32 bits; work
    // beyond that fills the card without being cut.
    int64_t total = 0;
    bool much = false;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const Seq s = b0 == 0 ? first : read(b0 + lane);
      const uint64_t share = static_cast<uint64_t>(s.tiles) * static_cast<uint32_t>(s.blocks);
      much |= __any(share >= 1u << 25);
      total += static_cast<uint32_t>(
          lane_value(scan64(static_cast<uint32_t>(min(share, uint64_t{1} << 25))), 63));
    }
    total = (total * a.kv_heads + kSlots - 1) / kSlots;
    if (!much) {
      cut = static_cast<uint32_t>(max(int64_t{kMinTiles}, min(total, int64_t{1} << 30)));
      // Pieces rounded up may be more workgroups than the card holds, of which the last
      // few would run by themselves: larger ones then, up to twice (3 trees of 40 behind
      // 5960 keys of 32 heads: 59 us, else 83; 2 of 24 behind 9258 of 40 heads of 80: 66
      // and 92; where lengths are uneven it may cost, 5 of 12 to 40 behind 3606 to 8960:
      // 157 and 137).
      const uint32_t least = cut;
      for (int i = 0;; ++i) {
        int64_t all = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 64) {
          const Seq s = b0 == 0 ? first : read(b0 + lane);
          all += static_cast<uint32_t>(lane_value(
              scan64(pieces_of(s.tiles, cut) * static_cast<uint32_t>(s.blocks)), 63));
        }
        if (all * a.kv_heads <= p.resident) break;
        if (i == 3) {
          cut = least;
          break;
        }
        cut += (cut + 3) / 4;
      }
    }
  }
  int items = 0, blocks = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const Seq s = b0 == 0 ? first : read(b0 + lane);
    const int pieces = static_cast<int>(pieces_of(s.tiles, cut));
    const uint32_t own = pieces * s.blocks;
    const uint32_t upto = scan64(own);
    const uint32_t upto_blocks = scan64(s.blocks);
    const uint64_t found = __ballot(join ? blocks + static_cast<int>(upto_blocks) > at
                                         : items + static_cast<int>(upto) > at);
    if (found != 0) {
      const int l = __ffsll(static_cast<unsigned long long>(found)) - 1;
      Item x;
      x.seq = b0 + l;
      x.start = lane_value(s.start, l);
      x.count = lane_value(s.count, l);
      x.keys = lane_value(s.keys, l);
      x.tiles = lane_value(s.tiles, l);
      x.pieces = lane_value(pieces, l);
      x.blocks = lane_value(s.blocks, l);
      x.first = items + lane_value(upto, l) - x.pieces * x.blocks;
      const int in = join ? at - blocks - (lane_value(upto_blocks, l) - x.blocks) : at - x.first;
      x.block = join ? in : in / x.pieces;
      x.piece = join ? 0 : in % x.pieces;
      return x;
    }
    items += lane_value(upto, 63);
    blocks += lane_value(upto_blocks, 63);
  }
  return Item{-1, items, 0, 0, 0, 0, 0, 0, 0, 0};
}

template <typename T>
__device__ inline T* out_row(const PagedAttention& a, int64_t row, int head) {
  return static_cast<T*>(a.out) + row * a.o_st + head * a.o_sh;
}

// Zeros in the rows of no sequence: workgroup i of n of a key head.
__device__ inline void clear_rows(const TreeParams& p, int kvh, int i, int n) {
  const PagedAttention& a = p.a;
  const int first = max(0, min(a.q_starts[0], a.tokens));
  const int end = max(first, min(a.q_starts[a.batch], a.tokens));
  const int chunks = a.head_dim / 8;
  for (int64_t r = i; r < first + (a.tokens - end); r += n) {
    uint16_t* row = static_cast<uint16_t*>(a.out) + (r < first ? r : r - first + end) * a.o_st;
    for (int c = threadIdx.x; c < p.group * chunks; c += blockDim.x)
      *reinterpret_cast<u32x4*>(row + (kvh * p.group + c / chunks) * a.o_sh + c % chunks * 8) =
          u32x4{0, 0, 0, 0};
  }
}

// Row `row` of a sequence and key head over keys k0 .. k1 - 1, key by key: lane i
// holds elements i and i + 64.  Masked and unknown keys are not read.
template <typename T>
__device__ inline void careful_row(const TreeParams& p, const Item& x, int kvh, int row, int k0,
                                   int k1, int64_t part) {
  const PagedAttention& a = p.a;
  const int lane = threadIdx.x & 63;
  const int D = a.head_dim, cached = x.keys - x.count;
  const int token = row / p.group, head = kvh * p.group + row % p.group;
  const int32_t* table = a.table + x.seq * a.ld_table;
  const uint32_t* mask = p.masks + (x.start + token) * p.ld_masks;
  const T* q = static_cast<const T*>(a.q) + (x.start + token) * a.q_st + head * a.q_sh;
  const float sc = a.scale * kLog2e;
  float qv[2], o[2] = {0.0f, 0.0f}, ref = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) qv[i] = lane + 64 * i < D ? to_f32(q[lane + 64 * i]) : 0.0f;
  for (int j = k0; j < k1; ++j) {
    const int n = j - cached;
    if (n >= 0 && (n / 32 >= p.words || !((mask[n / 32] >> (n & 31)) & 1))) continue;
    const int page = table[j >> a.page_shift];
    if (page < 0 || page >= a.pages) continue;
    const int64_t off = page * a.c_page + kvh * a.c_head +
                        (j & ((1 << a.page_shift) - 1)) * a.c_tok;
    float s = 0.0f, v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
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
    for (int i = 0; i < 2; ++i) o[i] = o[i] * f + w * v[i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = lane + 64 * i;
    if (d >= D) continue;
    if (x.pieces == 1)
      out_row<T>(a, x.start + token, head)[d] = from_f32<T>(o[i] * inv);
    else
      p.part_o[part * D + d] = o[i];
  }
  if (x.pieces > 1 && lane == 0) p.part_rl[part] = f32x2{ref, l};
}

// Chunk permutations of a key's row of DP / 8 chunks of 16 bytes (position = chunk ^
// swizzle): the 16 keys that an operand reads at one chunk, and the 16 that a
// transposing read takes at two, spread over all banks.
template <int DP> __device__ inline int swizzle_k(int key) {
  return DP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int DP> __device__ inline int swizzle_v(int key) {
  return DP == 64 ? ((key >> 1) & 1) << 2 | ((key >> 2) & 3) : (key & 3) << 2 | ((key >> 2) & 3);
}

// DP: head_dim rounded up to 64 or 128.  W: wavefronts of each part, of 16 rows each.
// DMA: pages of at least 8 keys; else each chunk is copied through registers.
template <typename T, int DP, int W, bool DMA>
__global__ __launch_bounds__(64 * W * kParts, W == 4 ? 2 : 1) void tree_kernel(TreeParams p) {
  constexpr int KS = DP / 32;               // first product: steps over the head
  constexpr int DV = DP / 16;               // second product: row tiles of O^T
  constexpr int R = 16 * W;
  constexpr int RB = DP * 2;                // bytes of a key's row
  constexpr int UB = kTile * RB;            // bytes of a unit of one operand
  constexpr int GN = kTile / 8 / W;         // groups of 8 keys that a wavefront copies
  constexpr int GL = 8 * RB / 1024;         // loads of a group and operand
  // Arrays of their own, so that the compiler sees that one is read while loads into
  // the others are in flight.
  constexpr int SB = UB * kParts;           // a unit of each part
  __shared__ __align__(16) char k0[SB], k1[SB], k2[SB], v0[SB], v1[SB], v2[SB];
  __shared__ int odd_pages[W * kParts];

  const PagedAttention& a = p.a;
  const int lane = threadIdx.x & 63;
  const int all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = all_waves % W, part_no = all_waves / W;
  const int r = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.kv_heads;
  const int slot = blockIdx.x / a.kv_heads;
  const Item x = find_item(p, R, slot, false);
  if (x.seq < 0) {
    if (p.clear) clear_rows(p, kvh, slot - x.start, gridDim.x / a.kv_heads - x.start);
    return;
  }
  if (slot >= p.items) return;   // starts that decrease: more rows than the batch has
  const int keys = x.keys, cached = x.keys - x.count;
  const int t0 = static_cast<int>(static_cast<int64_t>(x.tiles) * x.piece / x.pieces);
  const int t1 = static_cast<int>(static_cast<int64_t>(x.tiles) * (x.piece + 1) / x.pieces);
  const int D = a.head_dim;
  const int row0 = x.block * R + 16 * wave;         // the wavefront's first row
  const int total = x.count * p.group;
  const bool works = row0 < total;                  // else it only copies
  const bool live = row0 + r < total;
  const int row = min(row0 + r, total - 1);
  const int token = row / p.group, head = kvh * p.group + row % p.group;

  const_i32* table = (const_i32*)(a.table + x.seq * a.ld_table);
  const int page_mask = (1 << a.page_shift) - 1;
  const int ctok = static_cast<int>(a.c_tok);   // DMA: a page stays below 2^31 elements
  const int pages = static_cast<int>(a.pages);
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + kvh * a.c_head;
  const uint16_t* vb = static_cast<const uint16_t*>(a.v) + kvh * a.c_head;
  const int lk = lane / (RB / 16), lp = lane % (RB / 16);   // a load's key and chunk
  const int first_key = wave * GN * 8;
  int off_k[GN][GL], off_v[GN][GL];
#pragma unroll
  for (int i = 0; i < GN; ++i)
#pragma unroll
    for (int m = 0; m < GL; ++m) {
      const int in = m * (8 / GL) + lk, key = first_key + 8 * i + in;
      const int ck = (lp ^ swizzle_k<DP>(key)) * 8, cv = (lp ^ swizzle_v<DP>(key)) * 8;
      off_k[i][m] = ck < D ? (in * ctok + ck) * 2 : kOutside;
      off_v[i][m] = cv < D ? (in * ctok + cv) * 2 : kOutside;
    }
  struct Entries {
    int page[GN];
  };
  auto lookup = [&](int t) __attribute__((always_inline)) {
    Entries e;
#pragma unroll
    for (int i = 0; i < GN; ++i)
      e.page[i] = DMA && keys > 0
                      ? table[min(min(t, t1 - 1) * kTile + first_key + 8 * i, keys - 1) >>
                              a.page_shift]
                      : 0;
    return e;
  };
  auto dma = [](__amdgpu_buffer_rsrc_t rsrc, char* lds, int offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)lds, 16, offset, 0, 0, 0);
  };
  // The wavefront's part of unit t, keys then values; nothing is read from behind the
  // piece.
  auto copy = [&](int t, const Entries& e, char* kd, char* vd) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < GN; ++i) {
      const int key = t * kTile + first_key + 8 * i;
      char* to_k = kd + part_no * UB + (wave * GN + i) * GL * 1024;
      char* to_v = vd + part_no * UB + (wave * GN + i) * GL * 1024;
      if constexpr (DMA) {
        const int left = t < t1 ? keys - key : 0;
        const int page = __builtin_amdgcn_readfirstlane(e.page[i]);
        const bool known = left > 0 && static_cast<uint32_t>(page) < static_cast<uint32_t>(pages);
        const int64_t offset = known ? page * a.c_page + (key & page_mask) * ctok : int64_t{0};
        const int range = __builtin_amdgcn_readfirstlane(
            known ? ((left < 8 ? left : 8) - 1) * (2 * ctok) + 2 * D : 0);
        const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(offset));
        const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(offset >> 32));
        const int64_t at = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(kb + at), 0, range, kBufferWord3);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(vb + at), 0, range, kBufferWord3);
#pragma unroll
        for (int m = 0; m < GL; ++m) dma(rk, to_k + m * 1024, off_k[i][m]);
#pragma unroll
        for (int m = 0; m < GL; ++m) dma(rv, to_v + m * 1024, off_v[i][m]);
      } else {
#pragma unroll
        for (int m = 0; m < GL; ++m) {
          const int in = m * (8 / GL) + lk, j = key + in, unit = first_key + 8 * i + in;
          int page = -1;
          if (t < t1 && j < keys) page = table[j >> a.page_shift];
          const bool there = page >= 0 && page < pages;
          const int64_t at = there ? page * a.c_page + (j & page_mask) * a.c_tok : int64_t{0};
          const int ck = (lp ^ swizzle_k<DP>(unit)) * 8, cv = (lp ^ swizzle_v<DP>(unit)) * 8;
          u32x4 y{0, 0, 0, 0}, z{0, 0, 0, 0};
          if (there && ck < D) y = *reinterpret_cast<const u32x4*>(kb + at + ck);
          if (there && cv < D) z = *reinterpret_cast<const u32x4*>(vb + at + cv);
          *reinterpret_cast<u32x4*>(to_k + m * 1024 + lane * 16) = y;
          *reinterpret_cast<u32x4*>(to_v + m * 1024 + lane * 16) = z;
        }
      }
    }
  };
  // At most N of this wavefront's loads are in flight, so are the others', and every
  // wavefront has read what it was reading.  The wait is the builtin, which the
  // compiler's own insertion of waits follows.
  auto arrived = [&]() __attribute__((always_inline)) {
    constexpr int N = DMA ? (kStages - 2) * 2 * GN * GL : 0;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));   // lgkmcnt(0) too
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x4 o[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float ref = -INFINITY, l = 0.0f;
  const float sc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;

  if (t0 < t1) {
    const int tf = t0 + part_no;   // the part's first unit
    copy(tf, lookup(tf), k0, v0);
    copy(tf + kParts, lookup(tf + kParts), k1, v1);
    Entries ahead = lookup(tf + 2 * kParts);

    // Whether a page of these keys is unknown: then every unit looks its keys up.
    int odd = 0;
    {
      const int n = ((min(t1 * kTile, keys) - 1) >> a.page_shift) + 1;
      for (int i = (t0 * kTile >> a.page_shift) + threadIdx.x; i < n; i += 64 * W * kParts) {
        const int page = a.table[x.seq * a.ld_table + i];
        odd |= page < 0 || page >= pages;
      }
      const bool any = __any(odd);
      if (lane == 0) odd_pages[all_waves] = any;
    }
    u32x4 qf[KS];
    {
      // Negated for a negative scale, so that the one below is not, and zeros for a
      // scale of zero.
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + (x.start + token) * a.q_st +
                          head * a.q_sh + 8 * g;
      const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[s] = u32x4{0, 0, 0, 0};
        if (live && a.scale != 0.0f && 32 * s + 8 * g < D)
          qf[s] = *reinterpret_cast<const u32x4*>(q + 32 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[s][i] ^= flip;
      }
    }
    // Units from here on hold drafted keys: word n / 32 of the masks and the next,
    // cached keys are seen.
    auto masked = [&](int t) { return (t + 1) * kTile > cached; };
    const uint32_t* mask_row = p.masks + (x.start + token) * p.ld_masks;
    uint32_t words[2] = {0, 0};
    auto load_mask = [&](int t) __attribute__((always_inline)) {
      const int word = (t * kTile - cached) >> 5;
      words[0] = word < 0 ? ~0u : 0u;
      words[1] = 0u;
      if (word >= 0 && word < p.words) words[0] = mask_row[word];
      if (word + 1 < p.words) words[1] = mask_row[word + 1];
    };
    if (tf < t1 && masked(tf)) load_mask(tf);

    int read_k[2][KS], read_v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        read_k[h][s] = (16 * h + r) * RB + (((4 * s + g) ^ swizzle_k<DP>(16 * h + r)) * 16);
    // Lane i of 16 takes element 4 (i % 4) of row i / 4, and gets element i of the four
    // rows.  Row tile d is two chunks further than the one before: its permuted
    // position is formed where it is read.
    const int vkey[2] = {4 * g + (r >> 2), 16 + 4 * g + (r >> 2)};
#pragma unroll
    for (int b = 0; b < 2; ++b) read_v[b] = vkey[b] * RB + 8 * (r & 1);
    auto value_operand = [&](char* vt, int d) __attribute__((always_inline)) {
      u32x2 y[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
        y[b] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds_s16x4*)(vt + read_v[b] +
                                    (((2 * d + ((r & 3) >> 1)) ^ swizzle_v<DP>(vkey[b])) * 16))));
      return u32x4{y[0][0], y[0][1], y[1][0], y[1][1]};
    };

    auto unit = [&](int t, char* kt, char* vt, char* kfree, char* vfree)
        __attribute__((always_inline)) {
      kt += part_no * UB;
      vt += part_no * UB;
      arrived();
      if (t == tf) {
#pragma unroll
        for (int w = 0; w < W * kParts; ++w) odd |= odd_pages[w];
        odd = __builtin_amdgcn_readfirstlane(odd);
      }
      copy(t + (kStages - 1) * kParts, ahead, kfree, vfree);
      ahead = lookup(t + kStages * kParts);
      if (!works || t >= t1) return;
      // All operands are read ahead, the values' while the scores become
      // probabilities.
      u32x4 kf[KS][2], vf[DV];
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) kf[k][h] = *reinterpret_cast<const u32x4*>(kt + read_k[h][k]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DV; ++d) vf[d] = value_operand(vt, d);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 s[2];
      s[0] = s[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = mfma_16x16x32<T>(kf[k][h], qf[k], s[h]);
      const bool cut = (t + 1) * kTile > keys;
      if (masked(t) || cut || odd != 0) {
        uint32_t bits = ~0u;
        if (masked(t))
          bits = __builtin_amdgcn_alignbit(words[1], words[0], (t * kTile - cached) & 31);
        if (cut) bits &= (1u << (keys - t * kTile)) - 1u;
        if (odd != 0) {
#pragma unroll 1
          for (int i = 0; i < kTile; ++i) {
            const int j = t * kTile + i;
            int page = 0;
            if (j < keys) page = table[j >> a.page_shift];
            if (page < 0 || page >= pages) bits &= ~(1u << i);
          }
        }
        bits >>= 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s[i >> 2][i & 3] =
              shown_or_minus_infinity(s[i >> 2][i & 3], bits, (i < 4 ? 0 : 16) + (i & 3));
      }
      if (t + kParts < t1 && masked(t + kParts)) load_mask(t + kParts);
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
      top *= sc;
      if (__any(top > ref + Reference<T>::kSlack)) {
        // Raise the reference of the columns that need it; all four lanes of a
        // column agree.
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (top > ref + Reference<T>::kSlack) {
          const float next = top - Reference<T>::kBelow;
          const float f = ref == -INFINITY ? 1.0f : exp2_hw(ref - next);
          ref = next;
          l *= f;
#pragma unroll
          for (int i = 0; i < DV; ++i) o[i] *= f;
        }
      }
      const float base = ref == -INFINITY ? 0.0f : -ref;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = exp2_hw(__builtin_fmaf(s[i >> 2][i & 3], sc, base));
      l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t y, z;
        split2<T>(w[2 * i], w[2 * i + 1], y, z);
        hi[i] = y;
        lo[i] = z;
      }
#pragma unroll
      for (int d = 0; d < DV; ++d) o[d] = mfma_16x16x32<T>(vf[d], hi, o[d]);
#pragma unroll
      for (int d = 0; d < DV; ++d) o[d] = mfma_16x16x32<T>(vf[d], lo, o[d]);
    };
    // Both parts take as many steps, for their barriers.
    int t = tf;
    const int end = t1 + part_no;
    while (true) {
      unit(t, k0, v0, k2, v2);
      if ((t += kParts) >= end) break;
      unit(t, k1, v1, k0, v0);
      if ((t += kParts) >= end) break;
      unit(t, k2, v2, k1, v1);
      if ((t += kParts) >= end) break;
    }
    // No load into LDS outlives the workgroup, nor meets what follows.
    __builtin_amdgcn_s_waitcnt(0x0f70);

    // The second part's sums to the first, lane by lane.
    __shared__ f32x2 rl[W][64];
    __syncthreads();
    if (part_no > 0) {
#pragma unroll
      for (int d = 0; d < DV; ++d)
        *reinterpret_cast<f32x4*>((d < DV / 2 ? k0 : k1) +
                                  ((wave * (DV / 2) + d % (DV / 2)) * 64 + lane) * 16) = o[d];
      rl[wave][lane] = f32x2{ref, l};
    }
    __syncthreads();
    if (part_no > 0) return;
    const f32x2 other = rl[wave][lane];
    const float next = fmaxf(ref, other[0]);
    const float base = next == -INFINITY ? 0.0f : next;
    const float f0 = exp2_hw(ref - base), f1 = exp2_hw(other[0] - base);
    ref = next;
    l = l * f0 + other[1] * f1;
#pragma unroll
    for (int d = 0; d < DV; ++d) {
      const f32x4 y =
          *reinterpret_cast<const f32x4*>((d < DV / 2 ? k0 : k1) +
                                          ((wave * (DV / 2) + d % (DV / 2)) * 64 + lane) * 16);
      o[d] = o[d] * f0 + y * f1;
    }
  } else if (part_no > 0) {
    return;
  }
  if (!works) return;

  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  bool finite = fabsf(l) < INFINITY;
#pragma unroll
  for (int d = 0; d < DV; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) finite = finite && fabsf(o[d][i]) < INFINITY;
  uint64_t bad = __ballot(live && !finite);
  bad |= bad >> 32;
  bad = (bad | bad >> 16) & 0xffffu;
  const int64_t part =
      (static_cast<int64_t>(x.first + x.block * x.pieces + x.piece) * a.kv_heads + kvh) * R +
      16 * wave;
  if (live && !((bad >> r) & 1)) {
    // o[d][i]: element 16 d + 4 g + i of the lane's row.
    if (x.pieces == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      T* dst = out_row<T>(a, x.start + token, head) + 4 * g;
#pragma unroll
      for (int d = 0; d < DV; ++d)
        if (16 * d + 4 * g < D)
          *reinterpret_cast<u32x2*>(dst + 16 * d) = u32x2{
              pack2_bits<T>(o[d][0] * inv, o[d][1] * inv), pack2_bits<T>(o[d][2] * inv, o[d][3] * inv)};
    } else {
      float* dst = p.part_o + (part + r) * D + 4 * g;
#pragma unroll
      for (int d = 0; d < DV; ++d)
        if (16 * d + 4 * g < D) *reinterpret_cast<f32x4*>(dst + 16 * d) = o[d];
      if (g == 0) p.part_rl[part + r] = f32x2{ref, l};
    }
  }
  while (bad != 0) {
    const int i = __ffsll(static_cast<unsigned long long>(bad)) - 1;
    bad &= bad - 1;
    careful_row<T>(p, x, kvh, row0 + i, t0 * kTile, min(t1 * kTile, keys), part + i);
  }
}

// Adds up what the pieces of a block of rows left: a row per wavefront, four elements
// of every second (D = 128) piece per lane, kJoinAhead of them in flight.
template <typename T, int DP, int R>
__global__ __launch_bounds__(kJoinThreads) void tree_join_kernel(TreeParams p) {
  constexpr int C = DP / 4;              // threads of a row's elements
  constexpr int P = 64 / C;              // pieces at a time
  constexpr int G = kJoinThreads / 64;   // rows of a workgroup
  const PagedAttention& a = p.a;
  const int D = a.head_dim;
  const int kvh = blockIdx.x % a.kv_heads;
  const Item x = find_item(p, R, blockIdx.x / a.kv_heads, true);
  const int lane = threadIdx.x % 64, c = lane % C, first = lane / C;
  const int in = blockIdx.y * G + threadIdx.x / 64;
  const int n = x.pieces, row = x.block * R + in;
  if (x.seq < 0 || n <= 1 || row >= x.count * p.group || x.first + (x.block + 1) * n > p.items)
    return;
  const int64_t step = static_cast<int64_t>(a.kv_heads) * R;
  const int64_t at = static_cast<int64_t>(x.first + x.block * n) * step + kvh * R + in;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, p.part_rl[at + i * step][0]);
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w));
  const float base = top == -INFINITY ? 0.0f : top;
  const bool inside = 4 * c < D;
  const float* src = p.part_o + at * D + (inside ? 4 * c : 0);
  f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
  float l = 0.0f;
  for (int i0 = first; i0 < n; i0 += P * kJoinAhead) {
    f32x4 y[kJoinAhead];
    f32x2 rl[kJoinAhead];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      const int64_t i = min(i0 + P * k, n - 1) * step;
      y[k] = *reinterpret_cast<const f32x4*>(src + i * D);
      rl[k] = p.part_rl[at + i];
    }
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      const float w = i0 + P * k < n ? exp2_hw(rl[k][0] - base) : 0.0f;
      if (w != 0.0f) {   // what a weight of 0 leaves out may be anything
        o += y[k] * w;
        l += rl[k][1] * w;
      }
    }
  }
#pragma unroll
  for (int w = C; w < 64; w <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], w);
    l += __shfl_xor(l, w);
  }
  if (!inside || first > 0) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* dst = out_row<T>(a, x.start + row / p.group, kvh * p.group + row % p.group) + 4 * c;
  *reinterpret_cast<u32x2*>(dst) =
      u32x2{pack2_bits<T>(o[0] * inv, o[1] * inv), pack2_bits<T>(o[2] * inv, o[3] * inv)};
}

// Blocks of rows of a call at most: each sequence's last one may lack all but one.
int64_t max_blocks(int64_t tokens, int64_t batch, int64_t group, int64_t rows) {
  return (tokens * group + batch * (rows - 1)) / rows;
}

// How a call runs.
struct Plan {
  int rows;       // of a workgroup
  bool whole;
  int64_t row_blocks;   // at most
  int64_t items;        // (block, piece) pairs at most
};
Plan plan_of(int64_t tokens, int64_t batch, int64_t group, int64_t kv_heads, int64_t max_keys) {
  Plan x;
  const int64_t rows = ceil_div(tokens * group, batch);
  x.rows = rows <= 32 ? 32 : 64;
  x.row_blocks = max_blocks(tokens, batch, group, x.rows);
  x.whole = ceil_div(max_keys, kTile) <= kWholeTiles ||
            (x.row_blocks * kv_heads >= kCus && max_keys <= kWholeKeys);
  x.items = x.row_blocks + (x.whole ? 0 : kSlots / kv_heads);
  return x;
}

int64_t pairs_bytes(int64_t rows) { return ceil_div(rows * 8, 256) * 256; }

template <typename T, int DP, int W>
hipError_t launch_w(const TreeParams& p, const Plan& x, hipStream_t st) {
  const int64_t heads = p.a.kv_heads;
  // To clear rows, a workgroup per key head without an item.
  const dim3 grid(static_cast<uint32_t>((x.items + (p.clear ? 1 : 0)) * heads));
  if (p.a.page_shift >= 3 && (p.a.c_tok << p.a.page_shift) < (int64_t{1} << 30))
    hipLaunchKernelGGL((tree_kernel<T, DP, W, true>), grid, dim3(64 * W * kParts), 0, st, p);
  else
    hipLaunchKernelGGL((tree_kernel<T, DP, W, false>), grid, dim3(64 * W * kParts), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || x.whole) return e;
  hipLaunchKernelGGL((tree_join_kernel<T, DP, 16 * W>),
                     dim3(static_cast<uint32_t>(x.row_blocks * heads), 16 * W * 64 / kJoinThreads),
                     dim3(kJoinThreads), 0, st, p);
  return hipGetLastError();
}

template <typename T> hipError_t launch_t(const TreeParams& p, const Plan& x, hipStream_t st) {
  if (p.a.head_dim <= 64)
    return x.rows == 32 ? launch_w<T, 64, 2>(p, x, st) : launch_w<T, 64, 4>(p, x, st);
  return x.rows == 32 ? launch_w<T, 128, 2>(p, x, st) : launch_w<T, 128, 4>(p, x, st);
}

}  // namespace

// More rows than that have few keys per operation: they run as a prompt's, 128 rows to
// a key (4 trees of 33 to 45 tokens, 32 heads over 8, behind 32768: 148 us, here 220; 8
// of 48 behind 4048: 58 and 77; one of 64 behind 32704: 81 and 77).
bool small_trees(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                 int64_t head_dim) {
  const int64_t rows = tokens * (q_heads / kv_heads);
  return head_dim <= 128 && rows <= 64 * batch && batch * kv_heads <= (1 << 20);
}

int64_t small_trees_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                              int64_t head_dim, int64_t max_keys) {
  if (tokens == 0 || batch == 0) return 0;
  const Plan x = plan_of(tokens, batch, q_heads / kv_heads, kv_heads, max_keys);
  if (x.whole) return 0;
  const int64_t rows = x.items * kv_heads * x.rows;
  return pairs_bytes(rows) + rows * head_dim * 4;
}

hipError_t launch_small_trees(const PagedAttention& a, const uint64_t* masks, int64_t ld_masks,
                              int words, bool clear, int dtype, hipStream_t st) {
  TreeParams p{};
  p.a = a;
  p.masks = reinterpret_cast<const uint32_t*>(masks);
  p.ld_masks = 2 * ld_masks;
  p.words = 2 * words;
  p.group = a.q_heads / a.kv_heads;
  p.clear = clear;
  const Plan x = plan_of(a.tokens, a.batch, p.group, a.kv_heads, a.max_keys);
  p.whole = x.whole;
  p.items = static_cast<int>(x.items);
  p.resident = static_cast<int>(a.head_dim <= 64 ? 3 * kCus : kCus);   // by their LDS
  char* ws = static_cast<char*>(a.workspace);
  p.part_rl = reinterpret_cast<f32x2*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + pairs_bytes(x.items * a.kv_heads * x.rows));
  return dtype == kF16 ? launch_t<__half>(p, x, st) : launch_t<__hip_bfloat16>(p, x, st);
}

}  // namespace w8a8
