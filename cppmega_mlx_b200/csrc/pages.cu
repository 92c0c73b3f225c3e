// Movements of a paged cache: whole pages duplicated (a sequence forks, a shared page is about to be written, the pool is put
// in order) and rows moved within sequences (the accepted path of a drafted tree closes up behind the prefix).
//
// Both only move bytes: the bound is reading and writing each of them once at copy bandwidth, and for the usual small call the
// launch itself.  One launch serves every pool of a cache (keys and values, all layers).
#include "sm100.cuh"

namespace cmb {

constexpr int PG_MAX_POOLS = 32;
constexpr int PG_THREADS = 256;
constexpr int PG_UNROLL = 8;               // 16-byte pieces a thread has in flight

struct PagePool {
  uint8_t* base;
  long long page_stride, layer_stride, row_stride;   // bytes
  long long bytes;                                    // copy: of a page; move: of a row
  int layers;
};
struct PagePools {
  PagePool pool[PG_MAX_POOLS];
};

__device__ __forceinline__ void page_error(int* status, int a, int b, int c) {
  if (status != nullptr && atomicCAS(status, 0, ST_BAD_ARGUMENT) == 0) {
    status[1] = a;
    status[2] = b;
    status[3] = c;
  }
}

// grid (chunk of a page, pair, pool); V: the widest type that every address and size is a multiple of
template <typename V>
__global__ void __launch_bounds__(PG_THREADS) copy_pages_kernel(const __grid_constant__ PagePools pools, const int* src, const int* dst,
                                                                int pairs, int num_pages, int* status) {
  const PagePool& pool = pools.pool[blockIdx.z];
  const long long n = pool.bytes / static_cast<long long>(sizeof(V));
  const long long first = static_cast<long long>(blockIdx.x) * (PG_THREADS * PG_UNROLL);
  if (first >= n) return;
  const int pair = blockIdx.y;
  const int s = src[pair], d = dst[pair];
  if (s == -1 && d == -1) return;                    // an unused place of the list
  if (s < 0 || s >= num_pages || d < 0 || d >= num_pages) {
    if (threadIdx.x == 0) page_error(status, pair, s, d);
    return;
  }
  if (blockIdx.x == 0 && blockIdx.z == 0) {          // a page may be written once, and not read beside that
    for (int j = threadIdx.x; j < pairs; j += PG_THREADS)
      if (j != pair && (dst[j] == d || dst[j] == s)) page_error(status, pair, s, d);
  }
  if (s == d) return;
  const V* from = reinterpret_cast<const V*>(pool.base + s * pool.page_stride) + first;
  V* to = reinterpret_cast<V*>(pool.base + d * pool.page_stride) + first;
  const long long left = n - first;
  V v[PG_UNROLL];
#pragma unroll
  for (int i = 0; i < PG_UNROLL; ++i) {
    const int at = i * PG_THREADS + threadIdx.x;
    if (at < left) v[i] = from[at];
  }
#pragma unroll
  for (int i = 0; i < PG_UNROLL; ++i) {
    const int at = i * PG_THREADS + threadIdx.x;
    if (at < left) to[at] = v[i];
  }
}

// Rows start[b] + path[b, i] -> start[b] + i, i < counts[b].  A block holds every row of one sequence, pool and layer for
// `cols` pieces of the row in registers before it writes any of them, so sources and destinations may overlap.
// grid (column chunk, pool * layer, sequence)
template <typename V>
__global__ void __launch_bounds__(PG_THREADS) compact_rows_kernel(const __grid_constant__ PagePools pools, const int* table, int table_w,
                                                                  const int* start, const int* path, const int* counts, int most,
                                                                  int page, int num_pages, int layers, int cols, int* status) {
  const int b = blockIdx.z;
  const PagePool& pool = pools.pool[blockIdx.y / layers];
  const int layer = blockIdx.y % layers;
  const int n = pool.bytes / static_cast<int>(sizeof(V));
  const int c0 = blockIdx.x * cols;
  const int want = counts[b], rows = want < 0 ? 0 : (want < most ? want : most);
  const bool report = blockIdx.x == 0 && blockIdx.y == 0;
  if (want != rows && report && threadIdx.x == 0) page_error(status, b, want, most);
  if (c0 >= n || rows == 0) return;
  const int width = min(cols, n - c0);
  const long long s0 = start[b];
  uint8_t* base = pool.base + layer * pool.layer_stride;
  auto row_at = [&](long long j) -> uint8_t* {       // null for a position that the table does not hold
    if (j < 0 || j >= static_cast<long long>(table_w) * page) return nullptr;
    const int id = table[static_cast<long long>(b) * table_w + j / page];
    if (id < 0 || id >= num_pages) return nullptr;
    return base + id * pool.page_stride + (j % page) * pool.row_stride;
  };
  V v[PG_UNROLL];
  V* to[PG_UNROLL];
  const int total = rows * width;
#pragma unroll
  for (int i = 0; i < PG_UNROLL; ++i) {
    const int at = i * PG_THREADS + threadIdx.x;
    to[i] = nullptr;
    if (at < total) {
      const int r = at / width, c = at - r * width;
      const int p = path[static_cast<long long>(b) * most + r];
      if (p != r) {
        const uint8_t* from = row_at(s0 + p);
        uint8_t* dest = row_at(s0 + r);
        if (p < 0 || from == nullptr || dest == nullptr) {
          if (report && c == 0) page_error(status, b, p, r);
        } else {
          v[i] = reinterpret_cast<const V*>(from)[c0 + c];
          to[i] = reinterpret_cast<V*>(dest) + c0 + c;
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PG_UNROLL; ++i)
    if (to[i] != nullptr) *to[i] = v[i];
}

}  // namespace cmb

namespace {

// The widest access (16, 8, 4, 2 or 1 bytes) that divides every address, stride and size.
int pool_width(const cmb::PagePools& pools, int n, bool rows) {
  unsigned long long all = 16;
  for (int i = 0; i < n; ++i) {
    const cmb::PagePool& p = pools.pool[i];
    all |= reinterpret_cast<uintptr_t>(p.base) | static_cast<unsigned long long>(p.page_stride) | static_cast<unsigned long long>(p.bytes);
    if (rows) all |= static_cast<unsigned long long>(p.layer_stride) | static_cast<unsigned long long>(p.row_stride);
  }
  return static_cast<int>(all & (~all + 1));
}
template <typename V>
int launch_copy(const cmb::PagePools& pools, int n, const int* src, const int* dst, int pairs, int num_pages, int* status, cudaStream_t st) {
  long long most = 0;
  for (int i = 0; i < n; ++i) most = pools.pool[i].bytes > most ? pools.pool[i].bytes : most;
  const long long per = static_cast<long long>(cmb::PG_THREADS) * cmb::PG_UNROLL * sizeof(V);
  const long long chunks = (most + per - 1) / per;
  if (chunks > 0x7fffffffll) return 1;
  cmb::copy_pages_kernel<V><<<dim3(static_cast<unsigned>(chunks), pairs, n), cmb::PG_THREADS, 0, st>>>(pools, src, dst, pairs, num_pages, status);
  return cudaGetLastError() == cudaSuccess ? 0 : 104;
}
template <typename V>
int launch_compact(const cmb::PagePools& pools, int n, const int* table, int table_w, const int* start, const int* path, const int* counts,
                   int B, int most, int page, int num_pages, int layers, int* status, cudaStream_t st) {
  long long row = 0;
  for (int i = 0; i < n; ++i) row = pools.pool[i].bytes > row ? pools.pool[i].bytes : row;
  const long long vecs = row / static_cast<long long>(sizeof(V));
  const int cols = cmb::PG_THREADS * cmb::PG_UNROLL / most;
  const long long chunks = (vecs + cols - 1) / cols;
  if (chunks > 0x7fffffffll) return 1;
  cmb::compact_rows_kernel<V><<<dim3(static_cast<unsigned>(chunks), n * layers, B), cmb::PG_THREADS, 0, st>>>(
      pools, table, table_w, start, path, counts, most, page, num_pages, layers, cols, status);
  return cudaGetLastError() == cudaSuccess ? 0 : 104;
}

}  // namespace

// A pool as callers describe it: sizes and strides in bytes (host memory); bytes: of a page (copy) or of a row (compact).
struct cmb_page_pool {
  unsigned long long base;
  long long page_stride, layer_stride, row_stride, bytes;
};

// src, dst [pairs] page ids on the device (-1, -1: unused).  pairs <= 65535, n <= 32.
extern "C" int cmb_copy_pages(const cmb_page_pool* pool, int n, const int* src, const int* dst, int pairs, int num_pages, int* status,
                              void* stream) {
  if (n < 1 || n > cmb::PG_MAX_POOLS || pairs < 1 || pairs > 65535 || num_pages < 1) return 1;
  cmb::PagePools pools{};
  for (int i = 0; i < n; ++i) {
    if (pool[i].bytes <= 0) return 1;
    pools.pool[i] = {reinterpret_cast<uint8_t*>(pool[i].base), pool[i].page_stride, 0, 0, pool[i].bytes, 1};
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (pool_width(pools, n, false)) {
    case 16: return launch_copy<uint4>(pools, n, src, dst, pairs, num_pages, status, st);
    case 8: return launch_copy<uint2>(pools, n, src, dst, pairs, num_pages, status, st);
    case 4: return launch_copy<uint32_t>(pools, n, src, dst, pairs, num_pages, status, st);
    case 2: return launch_copy<uint16_t>(pools, n, src, dst, pairs, num_pages, status, st);
    default: return launch_copy<uint8_t>(pools, n, src, dst, pairs, num_pages, status, st);
  }
}

// ip = {B, table_w, most, page, num_pages, layers}; table [B, table_w], start [B], path [B, most], counts [B] int32 on the device;
// most <= 2048.
extern "C" int cmb_compact_rows(const cmb_page_pool* pool, int n, const int* table, const int* start, const int* path, const int* counts,
                                const int* ip, int* status, void* stream) {
  const int B = ip[0], table_w = ip[1], most = ip[2], page = ip[3], num_pages = ip[4], layers = ip[5];
  if (n < 1 || n > cmb::PG_MAX_POOLS || B < 1 || B > 65535 || most < 1 || most > cmb::PG_THREADS * cmb::PG_UNROLL || page < 1 ||
      num_pages < 1 || layers < 1 || table_w < 1 || static_cast<long long>(n) * layers > 65535)
    return 1;
  cmb::PagePools pools{};
  for (int i = 0; i < n; ++i) {
    if (pool[i].bytes <= 0 || pool[i].bytes > (1ll << 30)) return 1;
    pools.pool[i] = {reinterpret_cast<uint8_t*>(pool[i].base), pool[i].page_stride, pool[i].layer_stride, pool[i].row_stride, pool[i].bytes,
                     layers};
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (pool_width(pools, n, true)) {
    case 16: return launch_compact<uint4>(pools, n, table, table_w, start, path, counts, B, most, page, num_pages, layers, status, st);
    case 8: return launch_compact<uint2>(pools, n, table, table_w, start, path, counts, B, most, page, num_pages, layers, status, st);
    case 4: return launch_compact<uint32_t>(pools, n, table, table_w, start, path, counts, B, most, page, num_pages, layers, status, st);
    case 2: return launch_compact<uint16_t>(pools, n, table, table_w, start, path, counts, B, most, page, num_pages, layers, status, st);
    default: return launch_compact<uint8_t>(pools, n, table, table_w, start, path, counts, B, most, page, num_pages, layers, status, st);
  }
}
