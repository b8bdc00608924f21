// Pages of a paged KV cache copied on the device: pool[dst[i]] = pool[src[i]] for a list of page
// pairs, in every pool of every layer, in one launch.  What forking a sequence (its partly filled
// last page) and compacting a pool ask for; the reference has a ring buffer per slot and no
// counterpart.
//
// Pure streaming, every byte read once and written once.  A block takes one page pair, a warp of
// it 4 KB pieces of the pair's run in the pools, eight 16-byte loads a lane in flight before the
// first store; how many blocks share a pair is chosen so that a fork of a few pages still
// occupies every SM.  Measured on three sets of pools in turn: 2100 pages in 16 pools of 16 KB pages 178.2 us = 6180 GB/s
// read + written, 0.94 of the copy (180.8 with streaming hints on loads and stores, which gain 0.7 % where one set
// is copied over and over and lose 14 % on 301 pages of 8-bit pools, 8.3 -> 9.5 us; 177.0 with 16 loads in flight,
// but then 4 pages in 48 pools take 3.5 us instead of 2.9).
//
// A pair list can contradict itself (one destination named twice, or a page that is read and
// written in the same call), and what it would do then depended on which block came first.  Every
// block therefore scans the list for its own pair: the lists are a few KB in L2, next to
// the pages they move, and the outcome is the same whatever the order of the blocks.
#include "common.cuh"

namespace g4b {
namespace {

constexpr int kMaxPools = 192;        // per launch: the table travels as a kernel parameter (3 KB)
constexpr int kWarps = 8;
constexpr int kPiece = 4096;          // bytes a warp moves at a time

struct PageCopyParams {
  G4bPagePool pools[kMaxPools];
  const int32_t* src;
  const int32_t* dst;
  int64_t src_stride, dst_stride;
  int num_pools, num_pairs;
  int num_pages;
  int blocks_per_pair;
  int pieces;                         // 4 KB pieces of the largest pool's page
  int32_t* status;
};

enum : int32_t { kErrPage = 0x104, kErrConflict = 0x105 };

template <typename V>
__device__ __forceinline__ void copy_piece(const char* from, char* to, int bytes, int lane) {
  constexpr int kPerLane = 8;
  const int n = bytes / (int)sizeof(V);
  const V* a = reinterpret_cast<const V*>(from);
  V* b = reinterpret_cast<V*>(to);
  for (int at = 0; at < n; at += 32 * kPerLane) {
    V x[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int k = at + i * 32 + lane;
      if (k < n) x[i] = a[k];
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int k = at + i * 32 + lane;
      if (k < n) b[k] = x[i];
    }
  }
}

__global__ void __launch_bounds__(kWarps * 32) page_copy_kernel(const __grid_constant__ PageCopyParams p) {
  const int pair = blockIdx.x / p.blocks_per_pair;
  const int part = blockIdx.x - pair * p.blocks_per_pair;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto in_pool = [&](int page) { return page >= 0 && page < p.num_pages; };
  const int s = p.src[pair * p.src_stride], d = p.dst[pair * p.dst_stride];
  if (s < 0 || d < 0 || s == d) return;               // padding of a list of fixed length, or nothing to do
  if (!in_pool(s) || !in_pool(d)) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kErrPage);
    return;
  }
  bool clash = false;
  for (int j = threadIdx.x; j < p.num_pairs; j += kWarps * 32) {
    if (j == pair) continue;
    const int sj = p.src[j * p.src_stride], dj = p.dst[j * p.dst_stride];
    if (!in_pool(sj) || !in_pool(dj) || sj == dj) continue;
    clash |= dj == s || (dj == d && j < pair);
  }
  if (__syncthreads_or(clash)) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kErrConflict);
    return;
  }
  const int units = p.num_pools * p.pieces;
  for (int u = part * kWarps + warp; u < units; u += p.blocks_per_pair * kWarps) {
    const int pool = u / p.pieces;
    const int64_t at = (int64_t)(u - pool * p.pieces) * kPiece;
    const int64_t size = p.pools[pool].page_bytes;
    if (at >= size) continue;
    char* base = (char*)p.pools[pool].ptr;
    const char* from = base + s * size + at;
    char* to = base + d * size + at;
    const int bytes = (int)(size - at < kPiece ? size - at : kPiece);
    const uint64_t align = (uint64_t)base | (uint64_t)size;
    if ((align & 15) == 0) copy_piece<uint4>(from, to, bytes, lane);
    else if ((align & 3) == 0) copy_piece<uint32_t>(from, to, bytes, lane);
    else copy_piece<uint8_t>(from, to, bytes, lane);
  }
}

int check_pages(const G4bTensor& t, const char* name, int64_t n) {
  if (t.ndim != 1 || t.shape[0] < 0 || (n >= 0 && t.shape[0] != n)) return fail(G4B_ERR_BAD_ARG, "src_pages and dst_pages must be vectors of one length");
  if (t.ptr == nullptr && t.shape[0] > 0) return fail(G4B_ERR_BAD_ARG, "%s: null pointer", name);
  if (t.dtype != G4B_I32) return fail(G4B_ERR_BAD_DTYPE, "%s must be int32", name);
  return G4B_OK;
}

}  // namespace

int launch_page_copy(const G4bPageCopyArgs& a, cudaStream_t st) {
  int rc;
  if (a.num_pools < 0 || (a.num_pools > 0 && a.pools == nullptr)) return fail(G4B_ERR_BAD_ARG, "pools: null pointer");
  if (a.num_pages < 0 || a.num_pages > 0x7fffffffLL) return fail(G4B_ERR_BAD_ARG, "num_pages out of range");
  for (int i = 0; i < a.num_pools; ++i) {
    const G4bPagePool& q = a.pools[i];
    if (q.page_bytes < 0 || q.page_bytes > (1LL << 30)) return fail(G4B_ERR_BAD_ARG, "pool %d: page_bytes out of range", i);
    if (q.ptr == nullptr && q.page_bytes > 0 && a.num_pages > 0) return fail(G4B_ERR_BAD_ARG, "pool %d: null pointer", i);
  }
  if ((rc = check_pages(a.src_pages, "src_pages", -1)) || (rc = check_pages(a.dst_pages, "dst_pages", a.src_pages.shape[0]))) return rc;
  const int64_t n = a.src_pages.shape[0];
  // (every block scans the list: 2^16 pairs read 34 GB from L2 in all, a few milliseconds)
  if (n > 1 << 16) return fail(G4B_ERR_TOO_LARGE, "at most 65536 page pairs in a call");
  G4B_STOP_IF_VALIDATE_ONLY();
  if (n == 0) return G4B_OK;
  for (int first = 0; first < a.num_pools; first += kMaxPools) {
    PageCopyParams p{};
    p.num_pools = a.num_pools - first < kMaxPools ? a.num_pools - first : kMaxPools;
    int64_t largest = 0;
    for (int i = 0; i < p.num_pools; ++i) {
      p.pools[i] = a.pools[first + i];
      if (p.pools[i].page_bytes > largest) largest = p.pools[i].page_bytes;
    }
    if (largest == 0) continue;
    p.src = (const int32_t*)a.src_pages.ptr; p.dst = (const int32_t*)a.dst_pages.ptr;
    p.src_stride = a.src_pages.stride[0]; p.dst_stride = a.dst_pages.stride[0];
    p.num_pairs = (int)n;
    p.num_pages = (int)a.num_pages;
    p.pieces = (int)((largest + kPiece - 1) / kPiece);
    // eight blocks an SM wanted; a block has at least one piece for each of its warps
    const int64_t most = ((int64_t)p.num_pools * p.pieces + kWarps - 1) / kWarps;
    int64_t per = (148 * 8 + n - 1) / n;
    if (per > most) per = most;
    p.blocks_per_pair = (int)(per < 1 ? 1 : per);
    p.status = device_status_ptr();
    if (p.status == nullptr) return G4B_ERR_CUDA;
    page_copy_kernel<<<(unsigned)(n * p.blocks_per_pair), kWarps * 32, 0, st>>>(p);
    G4B_CUDA_CHECK(cudaGetLastError());
  }
  return G4B_OK;
}

}  // namespace g4b

extern "C" int g4b_page_copy(const G4bPageCopyArgs* args, void* cuda_stream) {
  if (args == nullptr) return g4b::fail(G4B_ERR_BAD_ARG, "args is null");
  return g4b::launch_page_copy(*args, (cudaStream_t)cuda_stream);
}
