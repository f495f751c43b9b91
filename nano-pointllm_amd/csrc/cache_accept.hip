// Keys and values of the accepted path of a tree of drafted tokens, moved to the
// places behind the cached ones (gfx950).
//
// A move copies row lengths[b] + path[i] to row lengths[b] + i, path[i] >= i: so
// no later move's source (at or past its own i) is an earlier one's target, and a
// thread that copies 16 bytes of a row for every i in order, a few of them ahead,
// copies what was there before the call.
//
// Bound by latency: three dependent reads (the path, the table, the row) and a
// write, of a few rows per sequence, head and layer: 4.5 us for one path of 5 rows of 32
// heads in 32 layers, 9.3 us for 32 paths of 1 to 8 rows of 8 heads in 32 layers (38 MB
// read and written, 4.0 TB/s); 13.4 us for 32 paths that move seven rows each, every
// one to where the next one was.
#include "w8a8_internal.h"

namespace w8a8 {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 8;   // rows that a thread has in flight

// Workgroup (x, y, z): 16-byte chunks of the heads' rows, layer and cache, sequence.
__global__ __launch_bounds__(kThreads) void accept_kernel(CacheAccept p) {
  const int chunks = p.head_dim / 8;
  const int n = blockIdx.x * kThreads + threadIdx.x;
  const int head = n / chunks, chunk = n % chunks;
  const int seq = blockIdx.z;
  const int32_t* path = p.path + seq * p.ld_path;
  const int32_t* table = p.table + seq * p.ld_table;
  const int64_t base = max(p.lengths[seq], 0);
  uint16_t* cache = static_cast<uint16_t*>(blockIdx.y & 1 ? p.v : p.k) +
                    (blockIdx.y >> 1) * p.c_layer;
  if (head >= p.kv_heads) return;
  cache += head * p.c_head + chunk * 8;
  const int mask = (1 << p.page_shift) - 1;
  // The row of a place, or null.
  auto row_of = [&](int64_t place) -> u32x4* {
    if (place >= p.max_keys) return nullptr;
    const int page = table[place >> p.page_shift];
    if (page < 0 || page >= p.pages) return nullptr;
    return reinterpret_cast<u32x4*>(cache + page * p.c_page + (place & mask) * p.c_tok);
  };
  for (int i0 = 0; i0 < p.steps; i0 += kAhead) {
    u32x4* to[kAhead];
    u32x4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int step = i0 + i;
      const int node = step < p.steps ? path[step] : -1;
      to[i] = nullptr;
      if (node <= step) continue;   // in its place already, or nothing to move
      const u32x4* from = row_of(base + node);
      if (from == nullptr) continue;
      to[i] = row_of(base + step);
      x[i] = *from;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (to[i] != nullptr) *to[i] = x[i];
  }
}

// Workgroups of one layer's keys, for one sequence.
int64_t groups_of(int64_t kv_heads, int64_t head_dim) {
  return ceil_div(kv_heads * (head_dim / 8), kThreads);
}

}  // namespace

int64_t cache_accept_workgroups(int64_t layers, int64_t batch, int64_t kv_heads,
                                int64_t head_dim) {
  return groups_of(kv_heads, head_dim) * 2 * layers * batch;
}

hipError_t launch_cache_accept(const CacheAccept& p, hipStream_t st) {
  hipLaunchKernelGGL(accept_kernel,
                     dim3(static_cast<uint32_t>(groups_of(p.kv_heads, p.head_dim)), 2 * p.layers,
                          p.batch),
                     dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace w8a8
