// Attention of one new token per sequence over a paged key-value cache
// (gfx950).
//
// Mathematics.  Per sequence and key head, with the queries q_0 .. q_{G-1}
// that share the head as columns: S^T = K Q^T, P = 2^(S^T c - r) with c = scale
// log2(e) and a running reference r per query (Reference in
// attention_common.h), O^T = V^T P, l = sum P; the result is O / l.
//
// Bound by memory: every key and value is read once, 4 head_dim bytes per key
// and key head against 4 head_dim G operations.  131071 keys of 8 heads (538 MB):
// 89 us, 6.0 TB/s, and 6 to join them; 64 sequences of 229 to 8190 keys of
// 8 heads (1.1 GB): 193 us, 5.7 TB/s; 8 of 775 to 1590 keys of 32 heads (157 MB):
// 31 us, 5.1 TB/s.  A small call is bound by its launches: 601 keys of 32 heads
// take 6.0 us and the join 4.2.
//
// Design:
//   * A wavefront takes tiles of 32 keys through v_mfma_f32_16x16x32 with the
//     queries as the 16 columns, for any G up to 16: with one query 15/16 of
//     the product is unused, and it still costs a tenth of the tile's bytes.
//   * Nothing goes through LDS in the loop.  A lane's 8 scores of a tile are
//     those of the 8 keys whose values it loads, so the probabilities are the
//     second product's operand as they are: the matrix instruction's inner
//     index is summed over, so any order of keys will do that both operands
//     share.  A lane loads 1/16 of the head of each of its 8 values, 16 lanes
//     whole rows, and interleaves them two keys at a time (v_perm_b32) into
//     rows of V^T.
//   * The probabilities enter as two 16-bit parts each (split2): the second
//     product is as exact as binary32 scores are, for a doubled product that
//     the memory time covers.
//   * While a tile is computed the next one's 16 KiB are in flight, in
//     registers; table entries are read a tile further ahead.
//   * Work is cut by the keys there are, on the device: the tiles of all
//     sequences are counted, and a sequence gets as many workgroups as its
//     share of kDecodeSlots asks for, so uneven batches cost nothing.  A
//     sequence of more than one workgroup leaves (O, r, l) per workgroup in the
//     workspace, which join_kernel adds up.  Whether any may be cut the host
//     decides, by the table's width: of one wider than the sequences' lengths the
//     joining launch may find nothing to do, and short sequences are cut that a
//     narrow table would leave whole (kWholeKeys).
//   * With a window and sinks (WINDOW) a sequence's tiles are those that hold a seen
//     key, the sinks' and then the window's; the keys of the first and last of them that
//     are not seen are masked like keys behind the length.  64 sequences of 229 to 8190
//     keys of 8 heads, a window of 1024 (258 MB): 44 us, 5.9 TB/s; one of 131071 with a
//     window of 4096: 8.0 us and 5.6 to join them.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"

namespace w8a8 {

namespace {

constexpr int kTile = 32;            // keys of a wavefront's step
constexpr int kMinTiles = 4;         // least tiles of a workgroup of several
// Sequences up to here are not cut: joining costs a launch (300 keys, 10 tiles,
// of 32 heads: 8.5 us whole, 5.5 + 4.4 us in pieces; 601 keys: 13 and 6.0 + 4.2).
constexpr int kWholeTiles = 10;
constexpr int kDecodeSlots = 768;    // workgroups aimed at
// Keys and values past the last-level cache's 256 MB are loaded without being
// kept in any (131071 keys of 8 heads: 89 against 95 us; 76 MB in 33 sequences:
// 19 against 17.5).
constexpr int64_t kCached = int64_t{256} << 20;
// A batch that gives every CU a workgroup by itself is not cut while its
// sequences may be no longer than this, by the table's width: nothing is joined
// then, and uneven lengths leave CUs idle for little time (8 sequences of 775 to
// 1590 keys, 32 heads: 30 us against 36 cut, which is also what they take over a
// table of 4096 keys; of 925 to 4000: 75 against 65).
// With fewer than two workgroups per CU they have 8 wavefronts, else 4 (32
// sequences of 1000 keys, 256 workgroups: 17.4 against 20.4 us; 64 of 2000, 512
// workgroups: 85 against 73).
constexpr int64_t kCus = 256;
constexpr int64_t kWholeKeys = 2048;
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 4;        // rows a thread loads before the weights are known

struct DecodeParams {
  PagedAttention a;
  int units;       // workgroups of one piece of a sequence: kv_heads x blocks of 16 queries
  int blocks;      // blocks of 16 queries per key head
  int group;       // queries per key head
  int rows;        // query rows of a workgroup: min(group, 16)
  bool whole;      // no sequence is cut
  bool large;      // with whole: the batch's keys and values may pass kCached
  int window, sinks;   // of a windowed call
  float* part_o;   // [pieces x units, rows, head_dim]
  f32x2* part_rl;  // [pieces x units, rows]
};

// Pieces that all sequences are cut into at most: each gets one, and the cut
// itself adds at most slots / units.
inline int64_t max_pieces(int64_t batch, int64_t units, int64_t max_keys) {
  const int64_t tiles = ceil_div(max_keys, kTile);
  if (batch * units >= kCus && max_keys <= kWholeKeys) return batch;
  const int64_t cut = batch + kDecodeSlots / units;
  return tiles <= kWholeTiles ? batch : std::min(cut, batch * ceil_div(tiles, kMinTiles));
}

struct Piece {
  int seq;     // the sequence, or -1
  int first;   // its first piece
  int count;   // its pieces
  int tiles;   // its tiles, of a windowed call those that are seen
  int keys;    // its keys
  bool large;  // the batch's keys and values pass kCached
};

// Of a windowed call: the tiles of a sequence that hold a seen key, in order: its
// first `head` tiles and, from tile head + skip on, the others.
struct Tiles {
  int low;    // the first key of the window
  int head;
  int skip;
  int count;
};
__device__ inline Tiles window_tiles(const DecodeParams& p, int keys) {
  const int low = max(keys - p.window, 0);
  const int all = (keys + kTile - 1) / kTile;
  const int head = (min(p.sinks, low) + kTile - 1) / kTile;
  const int from = max(low / kTile, head);
  return Tiles{low, head, from - head, all - from + head};
}

// The sequence of piece `slot`, or the pieces of sequence `seq` (slot < 0).
// Every lane of the wavefront takes part and gets the same answer, in scalar
// registers.  A lane's tiles stay below 2^26, so 64 of them fit 32 bits.
template <bool WINDOW>
__device__ inline Piece find_piece(const DecodeParams& p, int slot, int seq) {
  const int lane = threadIdx.x & 63;
  const int batch = p.a.batch;
  auto keys_of = [&](int b) { return b < batch ? max(0, min(p.a.lengths[b], p.a.max_keys)) : 0; };
  auto tiles_of = [&](int keys) {
    if constexpr (WINDOW) return static_cast<uint32_t>(window_tiles(p, keys).count);
    return static_cast<uint32_t>(keys + kTile - 1) / kTile;
  };
  if (p.whole) {
    const int at = slot >= 0 ? slot : seq;
    const int keys = max(0, min(p.a.lengths[at], p.a.max_keys));
    return Piece{at, at, 1, static_cast<int>(tiles_of(keys)), keys, p.large};
  }
  const int keys0 = keys_of(lane);
  int64_t total = static_cast<uint32_t>(lane_value(scan64(tiles_of(keys0)), 63));
  for (int b0 = 64; b0 < batch; b0 += 64)
    total += static_cast<uint32_t>(lane_value(scan64(tiles_of(keys_of(b0 + lane))), 63));
  const bool large = total > kCached / (int64_t{4} * kTile * p.a.kv_heads * p.a.head_dim);
  total *= p.units;
  const int64_t share = min((total + kDecodeSlots - 1) / kDecodeSlots, int64_t{INT32_MAX / 2});
  const uint32_t cut = max(static_cast<uint32_t>(kMinTiles), static_cast<uint32_t>(share));
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int keys = b0 == 0 ? keys0 : keys_of(b0 + lane);
    const uint32_t tiles = tiles_of(keys);
    const uint32_t pieces = tiles <= kWholeTiles ? 1u : (tiles + cut - 1) / cut;
    const uint32_t count = b0 + lane < batch ? pieces : 0u;
    const uint32_t upto = scan64(count);
    const bool mine = slot >= 0 ? before + static_cast<int>(upto) > slot : b0 + lane == seq;
    const uint64_t found = __ballot(mine);
    if (found != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(found)) - 1;
      const int n = lane_value(count, at);
      return Piece{b0 + at, before + lane_value(upto, at) - n, n, lane_value(tiles, at),
                   lane_value(static_cast<uint32_t>(keys), at), large};
    }
    before += lane_value(upto, 63);
  }
  return Piece{-1, 0, 0, 0, 0, false};
}

template <typename T>
__device__ inline void write_out(const DecodeParams& p, int seq, int head, int d, float o,
                                 float l) {
  const float y = o * (l == 0.0f ? 0.0f : 1.0f / l);
  static_cast<T*>(p.a.out)[seq * p.a.o_st + head * p.a.o_sh + d] = from_f32<T>(y);
}

// DP: head_dim rounded up to 64, 128 or 256; FULL: head_dim == DP.  SMALL:
// pages of fewer than 4 keys, so that each key has a table entry of its own.
// W: wavefronts.  WINDOW: the keys between the sinks and the window are not seen.
template <typename T, int DP, bool FULL, bool SMALL, int W, bool WINDOW>
__global__ __launch_bounds__(64 * W, DP == 256 ? 1 : 2) void decode_kernel(DecodeParams p) {
  constexpr int KS = DP / 32;   // first product: steps over the head
  constexpr int DV = DP / 16;   // elements of a value row per lane
  constexpr int VW = DV / 2;    // ... dwords
  constexpr int NV = SMALL ? 8 : 2;  // table entries of a lane's 8 values
  __shared__ float red_o[W][16][DP];
  __shared__ float red_r[W][16], red_l[W][16];

  const PagedAttention& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / p.units, unit = blockIdx.x % p.units;
  const Piece piece = find_piece<WINDOW>(p, slot, -1);
  const int seq = piece.seq, count = piece.count;
  const int tiles = __builtin_amdgcn_readfirstlane(piece.tiles);
  const int keys = __builtin_amdgcn_readfirstlane(piece.keys);
  if (seq < 0) return;
  Tiles seen{0, tiles, 0, tiles};
  if constexpr (WINDOW) seen = window_tiles(p, keys);
  // The first key of the piece's tile t, and whether key j is seen.
  auto key_of = [&](int t) { return (WINDOW && t >= seen.head ? t + seen.skip : t) * kTile; };
  auto is_seen = [&](int j) { return j < keys && (!WINDOW || j >= seen.low || j < p.sinks); };
  const int part = slot - piece.first;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / count);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / count);
  const int kvh = unit / p.blocks;
  const int head0 = kvh * p.group + (unit % p.blocks) * 16;
  const int rows = min(16, (kvh + 1) * p.group - head0);
  const int D = a.head_dim;

  u32x4 qf[KS];
  bool live[KS];   // whether the head has elements 32 s + 8 g
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    live[s] = FULL || 32 * s + 8 * g < D;
    qf[s] = u32x4{0, 0, 0, 0};
    if (live[s] && r < rows)
      qf[s] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + seq * a.q_st +
                                              (head0 + r) * a.q_sh + 32 * s + 8 * g);
  }
  const int vd = FULL || r * DV < D ? r * DV : 0;   // rows past the head are not written
  const int32_t* table = a.table + seq * a.ld_table;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + kvh * a.c_head + 8 * g;
  const uint16_t* vb = static_cast<const uint16_t*>(a.v) + kvh * a.c_head + vd;
  const int page_mask = (1 << a.page_shift) - 1;
  const int pages = static_cast<int>(a.pages);

  struct Entries {
    int k[2];    // of keys 16 t + r
    int v[NV];   // of keys 4 g and 16 + 4 g (SMALL: 4 g + i, then 16 + 4 g + i)
  };
  struct Tile {
    u32x4 k[2][KS];
    uint32_t v[8][VW];
    uint32_t ok;   // bit i: the lane's key i is there
  };
  auto entry = [&](int j) {
    int e = -1;
    if (is_seen(j)) e = table[j >> a.page_shift];
    return e;
  };
  // Of the page of keys j .. j + 3, any of which may be the first of the window.
  auto entry_of_four = [&](int j) {
    int e = -1;
    if (j < keys && (!WINDOW || j + 3 >= seen.low || j < p.sinks)) e = table[j >> a.page_shift];
    return e;
  };
  auto lookup = [&](int t, Entries& e) {
#pragma unroll
    for (int h = 0; h < 2; ++h) e.k[h] = entry(key_of(t) + 16 * h + r);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      e.v[i] = SMALL ? entry(key_of(t) + (i < 4 ? 0 : 16) + 4 * g + (i & 3))
                     : entry_of_four(key_of(t) + 16 * i + 4 * g);
  };
  // A key that is not there reads row 0 of page 0 instead.
  auto row_of = [&](int e, int j) {
    return e >= 0 && e < pages ? e * a.c_page + (j & page_mask) * a.c_tok : int64_t{0};
  };
  auto load = [](auto once, const auto* src) {
    if constexpr (decltype(once)::value)
      return __builtin_nontemporal_load(src);
    else
      return *src;
  };
  auto issue = [&](auto once, int t, const Entries& e, Tile& x) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* src = kb + row_of(e.k[h], key_of(t) + 16 * h + r);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (FULL) {
          x.k[h][s] = load(once, reinterpret_cast<const u32x4*>(src + 32 * s));
        } else {
          x.k[h][s] = u32x4{0, 0, 0, 0};
          if (live[s]) x.k[h][s] = load(once, reinterpret_cast<const u32x4*>(src + 32 * s));
        }
      }
    }
    x.ok = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = key_of(t) + (i < 4 ? 0 : 16) + 4 * g + (i & 3);
      const int ev = e.v[SMALL ? i : i >> 2];
      const bool there = is_seen(j) && ev >= 0 && ev < pages;
      x.ok |= static_cast<uint32_t>(there) << i;
      const uint16_t* src = vb + row_of(there ? ev : -1, j);
      if constexpr (VW == 2) {
        const u32x2 w = load(once, reinterpret_cast<const u32x2*>(src));
        x.v[i][0] = w[0];
        x.v[i][1] = w[1];
      } else {
#pragma unroll
        for (int c = 0; c < VW; c += 4) {
          // head_dim is a multiple of 8: a lane's second half may lie past it.
          const int more = FULL || c == 0 || vd + 2 * c < D ? 2 * c : 0;
          const u32x4 w = load(once, reinterpret_cast<const u32x4*>(src + more));
#pragma unroll
          for (int k = 0; k < 4; ++k) x.v[i][c + k] = w[k];
        }
      }
    }
  };

  f32x4 o[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float ref = -INFINITY, l = 0.0f;
  const float sc = a.scale * kLog2e;

  auto compute = [&](Tile& x) __attribute__((always_inline)) {
    f32x4 s0{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      s0 = mfma_16x16x32<T>(x.k[0][s], qf[s], s0);
      s1 = mfma_16x16x32<T>(x.k[1][s], qf[s], s1);
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = s0[i] * sc;
      w[4 + i] = s1[i] * sc;
    }
    if (!__all(x.ok == 0xffu)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool there = (x.ok >> i) & 1;
        w[i] = there ? w[i] : -INFINITY;
#pragma unroll
        for (int c = 0; c < VW; ++c) x.v[i][c] = there ? x.v[i][c] : 0u;
      }
    }
    float top = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, w[i]);
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
    // Without a score above -inf so far the reference is 0: -inf gives 0, NaN
    // stays.
    const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = exp2_hw(w[i] - base);
    l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h, m;
      split2<T>(w[2 * i], w[2 * i + 1], h, m);
      hi[i] = h;
      lo[i] = m;
    }
#pragma unroll
    for (int i = 0; i < DV; ++i) {
      u32x4 vt;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        vt[k] = __builtin_amdgcn_perm(x.v[2 * k + 1][i >> 1], x.v[2 * k][i >> 1],
                                      (i & 1) ? 0x07060302u : 0x05040100u);
      o[i] = mfma_16x16x32<T>(vt, hi, o[i]);
      o[i] = mfma_16x16x32<T>(vt, lo, o[i]);
    }
  };

  auto run = [&](auto once) __attribute__((always_inline)) {
    int t = t0 + wave;
    Entries e;
    Tile x0, x1;
    if (t < t1) {
      lookup(t, e);
      issue(once, t, e, x0);
      lookup(min(t + W, t1 - 1), e);
    }
    while (t < t1) {
      const int tn = t + W;
      if (tn < t1) {
        issue(once, tn, e, x1);
        lookup(min(tn + W, t1 - 1), e);
      }
      compute(x0);
      if (tn >= t1) break;
      const int tm = tn + W;
      if (tm < t1) {
        issue(once, tm, e, x0);
        lookup(min(tm + W, t1 - 1), e);
      }
      compute(x1);
      t = tm;
    }
  };
  if (piece.large)
    run(std::true_type{});
  else
    run(std::false_type{});

  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (r < rows) {
    if (g == 0) {
      red_r[wave][r] = ref;
      red_l[wave][r] = l;
    }
    // o[i][k]: element DV (4 g + k) + i of the head.
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < DV; ++i) red_o[wave][r][DV * (4 * g + k) + i] = o[i][k];
  }
  __syncthreads();
  // What infinities and NaNs among the piece's values make of element d: an
  // infinity times a part of its weight that is 0 must not make it NaN.  0
  // without any (the sum itself passed binary32).  16 values are in flight: a
  // NaN among 131071 keys adds 0.11 ms to 0.09, one after the other 0.30.
  auto not_finite = [&](int d) {
    constexpr int N = 16;
    bool up = false, down = false, nan = false;
    const T* v = static_cast<const T*>(a.v) + kvh * a.c_head + d;
    const int last = t1 > t0 ? min(key_of(t1 - 1) + kTile, keys) : 0;
    for (int i0 = t0 * kTile; i0 < t1 * kTile; i0 += N) {
      const int j0 = key_of(i0 / kTile) + i0 % kTile;
      if (j0 >= last) break;
      int e[N];
      T y[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = min(j0 + i, last - 1);
        e[i] = !WINDOW || is_seen(j) ? table[j >> a.page_shift] : -1;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = v[row_of(e[i], min(j0 + i, last - 1))];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool there = e[i] >= 0 && e[i] < pages;
        const float x = to_f32(y[i]);
        up |= there && x == INFINITY;
        down |= there && x == -INFINITY;
        nan |= there && x != x;
      }
    }
    return nan || (up && down) ? NAN : up ? INFINITY : down ? -INFINITY : 0.0f;
  };
  const int64_t item = blockIdx.x;
  bool searched = false;
  float special = 0.0f;
  for (int n = threadIdx.x; n < rows * DP; n += 64 * W) {
    const int q = n / DP, d = n % DP;   // one d per thread
    if (!FULL && d >= D) continue;
    float top = red_r[0][q];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, red_r[w][q]);
    const float base = top == -INFINITY ? 0.0f : top;
    float ov = 0.0f, lv = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2_hw(red_r[w][q] - base);
      ov += red_o[w][q][d] * f;
      lv += red_l[w][q] * f;
    }
    if (!(fabsf(ov) < INFINITY) && fabsf(lv) < INFINITY) {
      if (!searched) special = not_finite(d);
      searched = true;
      ov = special == 0.0f ? ov : special;
    }
    if (count == 1) {
      write_out<T>(p, seq, head0 + q, d, ov, lv);
    } else {
      p.part_o[(item * p.rows + q) * D + d] = ov;
      if (d == 0) p.part_rl[item * p.rows + q] = f32x2{top, lv};
    }
  }
}

// One workgroup per query row: adds up what the pieces of its sequence left.
// A thread takes four elements of every eighth (D = 128) piece, the first
// kJoinAhead of them in flight while the weights are formed.
template <typename T, int DP, bool WINDOW>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(DecodeParams p) {
  constexpr int C = DP / 4;              // threads of a row
  constexpr int R = kJoinThreads / C;    // rows at a time
  constexpr int W = kJoinThreads / 64;
  __shared__ float weight[kDecodeSlots + 1];   // one sequence's pieces at most
  __shared__ f32x4 red_o[R][C];
  __shared__ float red[2][W];
  const int seq = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const int D = p.a.head_dim;
  const Piece piece = find_piece<WINDOW>(p, -1, seq);
  const int n = piece.count;
  if (n <= 1) return;
  const int q = head % p.group;
  const int unit = head / p.group * p.blocks + q / 16;
  const int64_t step = static_cast<int64_t>(p.units) * p.rows;
  const int64_t at = (static_cast<int64_t>(piece.first) * p.units + unit) * p.rows + q % 16;
  const int c = tid % C, row = tid / C;
  const float* src = p.part_o + at * D + 4 * c;
  f32x4 ahead[kJoinAhead];
#pragma unroll
  for (int i = 0; i < kJoinAhead; ++i) {
    ahead[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (row + i * R < n && 4 * c < D)
      ahead[i] = *reinterpret_cast<const f32x4*>(src + (row + i * R) * step * D);
  }
  float top = -INFINITY;
  for (int i = tid; i < n; i += kJoinThreads) {
    weight[i] = p.part_rl[at + i * step][0];
    top = fmaxf(top, weight[i]);
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w));
  if ((tid & 63) == 0) red[0][tid >> 6] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, red[0][w]);
  const float base = top == -INFINITY ? 0.0f : top;
  float l = 0.0f;
  for (int i = tid; i < n; i += kJoinThreads) {
    weight[i] = exp2_hw(weight[i] - base);
    l += weight[i] * p.part_rl[at + i * step][1];
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) l += __shfl_xor(l, w);
  if ((tid & 63) == 0) red[1][tid >> 6] = l;
  __syncthreads();
  f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kJoinAhead; ++i)
    if (row + i * R < n) o += ahead[i] * weight[row + i * R];
  if (4 * c < D) {
#pragma unroll 4
    for (int i = row + kJoinAhead * R; i < n; i += R)
      o += *reinterpret_cast<const f32x4*>(src + i * step * D) * weight[i];
  }
  red_o[row][c] = o;
  __syncthreads();
  if (row == 0 && 4 * c < D) {
    l = red[1][0];
#pragma unroll
    for (int w = 1; w < W; ++w) l += red[1][w];
#pragma unroll
    for (int w = 1; w < R; ++w) o += red_o[w][c];
#pragma unroll
    for (int i = 0; i < 4; ++i) write_out<T>(p, seq, head, 4 * c + i, o[i], l);
  }
}

template <typename T, int DP, bool FULL, bool WINDOW>
hipError_t launch_d(const DecodeParams& p, int64_t pieces, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(pieces * p.units));
  const bool small = p.a.page_shift < 2;
  // Heads past 128 take too many registers for two wavefronts of a SIMD.
  if (DP <= 128 && !small && p.whole && grid.x < 2 * kCus)
    hipLaunchKernelGGL((decode_kernel<T, DP, FULL, false, DP <= 128 ? 8 : 4, WINDOW>), grid,
                       dim3(64 * (DP <= 128 ? 8 : 4)), 0, st, p);
  else if (small)
    hipLaunchKernelGGL((decode_kernel<T, DP, FULL, true, 4, WINDOW>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((decode_kernel<T, DP, FULL, false, 4, WINDOW>), grid, dim3(256), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || pieces == p.a.batch) return e;
  hipLaunchKernelGGL((join_kernel<T, DP, WINDOW>), dim3(p.a.batch, p.a.q_heads), dim3(kJoinThreads), 0, st,
                     p);
  return hipGetLastError();
}

template <typename T, bool WINDOW>
hipError_t launch_t(const DecodeParams& p, int64_t pieces, hipStream_t st) {
  const int d = p.a.head_dim;
  if (d == 64) return launch_d<T, 64, true, WINDOW>(p, pieces, st);
  if (d < 64) return launch_d<T, 64, false, WINDOW>(p, pieces, st);
  if (d == 128) return launch_d<T, 128, true, WINDOW>(p, pieces, st);
  if (d < 128) return launch_d<T, 128, false, WINDOW>(p, pieces, st);
  if (d == 256) return launch_d<T, 256, true, WINDOW>(p, pieces, st);
  return launch_d<T, 256, false, WINDOW>(p, pieces, st);
}

int64_t units_of(int64_t q_heads, int64_t kv_heads) {
  return kv_heads * ceil_div(q_heads / kv_heads, 16);
}

// Bytes of the (r, l) pairs in front of the O rows.
int64_t pairs_bytes(int64_t items, int64_t rows) { return ceil_div(items * rows * 8, 256) * 256; }

int64_t workspace_of(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                     int64_t max_keys) {
  const int64_t units = units_of(q_heads, kv_heads);
  const int64_t pieces = max_pieces(batch, units, max_keys);
  if (pieces <= batch) return 0;
  const int64_t rows = std::min<int64_t>(q_heads / kv_heads, 16), items = pieces * units;
  return pairs_bytes(items, rows) + items * rows * head_dim * 4;
}

// keys: what workspace_of was asked with.
template <bool WINDOW>
hipError_t launch(DecodeParams& p, const PagedAttention& a, int64_t keys, int dtype,
                  hipStream_t st) {
  p.a = a;
  p.group = a.q_heads / a.kv_heads;
  p.blocks = static_cast<int>(ceil_div(p.group, 16));
  p.units = a.kv_heads * p.blocks;
  p.rows = std::min(p.group, 16);
  const int64_t pieces = max_pieces(a.batch, p.units, keys);
  p.whole = pieces == a.batch;
  p.large = 4.0 * a.batch * keys * a.kv_heads * a.head_dim > static_cast<double>(kCached);
  char* ws = static_cast<char*>(a.workspace);
  p.part_rl = reinterpret_cast<f32x2*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + pairs_bytes(pieces * p.units, p.rows));
  return dtype == kF16 ? launch_t<__half, WINDOW>(p, pieces, st)
                       : launch_t<__hip_bfloat16, WINDOW>(p, pieces, st);
}

// The keys of the tiles that a row sees at most: all, or those of the sinks and of
// the window.
int64_t seen_keys(int64_t max_keys, int64_t window, int64_t sinks) {
  return std::min(max_keys, (ceil_div(sinks, kTile) + ceil_div(window, kTile) + 1) * kTile);
}

}  // namespace

int64_t paged_decode_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t max_keys) {
  return workspace_of(batch, q_heads, kv_heads, head_dim, max_keys);
}

int64_t paged_decode_window_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                      int64_t head_dim, int64_t max_keys, int64_t window,
                                      int64_t sinks) {
  return workspace_of(batch, q_heads, kv_heads, head_dim, seen_keys(max_keys, window, sinks));
}

hipError_t launch_paged_decode(const PagedAttention& a, int dtype, hipStream_t st) {
  DecodeParams p{};
  return launch<false>(p, a, a.max_keys, dtype, st);
}

hipError_t launch_paged_decode_window(const PagedAttention& a, int window, int sinks, int dtype,
                                      hipStream_t st) {
  DecodeParams p{};
  p.window = window;
  p.sinks = sinks;
  return launch<true>(p, a, seen_keys(a.max_keys, window, sinks), dtype, st);
}

}  // namespace w8a8
