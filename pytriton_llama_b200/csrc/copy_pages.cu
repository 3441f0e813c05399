// Rows of several tensors copied inside them: dst row <- src row of every tensor, for every (src, dst) pair, in one launch.
// Pages of all cache entries of a group (a request forked, pages moved to the front of a pool) and rows of per-request
// states are copied so.
//
// The tensors and the pairs are arguments of the launch (up to 32 KB of them), so nothing is sent to the device
// beforehand and a captured copy holds its own.  No dst row is a src row of the same call and none comes twice, so the
// copies have no order.  A block takes 16 KB of a row: four packets of 16 bytes a thread, all asked for before one is stored.
//
// What bounds it: the bytes, read and written once.  1,500 pages of 16 KB in 16 tensors: 130 us, 6.06 TB/s (a copy of the device's own kind
// measured 6.45); one page of 32 KB to seven others in 16 tensors: 2.2 us, of which the bytes take 1.1.
#include "common.cuh"

namespace ptl {

constexpr int kCopyThreads = 256;
constexpr int kCopyAhead = 4;                                  // packets a thread asks for at once
constexpr int kCopyMaxTensors = 128;

template <int TENSORS, int PAIRS> struct CopyArgs {
  int tensors, pairs;
  unsigned char* base[TENSORS];
  long long row_bytes[TENSORS];
  int chunk_end[TENSORS];                                      // chunks of one pair's rows up to and with each tensor
  int src[PAIRS], dst[PAIRS];
};

template <typename P>
__device__ __forceinline__ void copy_chunk(unsigned char* to, const unsigned char* from, int packets) {
  P v[kCopyAhead];
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i) {
    const int e = i * kCopyThreads + threadIdx.x;
    if (e < packets) v[i] = reinterpret_cast<const P*>(from)[e];
  }
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i) {
    const int e = i * kCopyThreads + threadIdx.x;
    if (e < packets) reinterpret_cast<P*>(to)[e] = v[i];
  }
}

template <int TENSORS, int PAIRS, typename P>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ CopyArgs<TENSORS, PAIRS> a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kChunk = kCopyThreads * kCopyAhead * (int)sizeof(P);
  const int per_pair = a.chunk_end[a.tensors - 1];
  const long long total = (long long)per_pair * a.pairs;
  for (long long i = blockIdx.x; i < total; i += gridDim.x) {
    const int pair = (int)(i / per_pair), c = (int)(i % per_pair);
    int lo = 0, hi = a.tensors - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.chunk_end[mid] > c) hi = mid; else lo = mid + 1;
    }
    const long long row = a.row_bytes[lo], at = (long long)(c - (lo ? a.chunk_end[lo - 1] : 0)) * kChunk;
    const long long left = row - at;
    copy_chunk<P>(a.base[lo] + a.dst[pair] * row + at, a.base[lo] + a.src[pair] * row + at, (int)(left < kChunk ? left : kChunk) / (int)sizeof(P));
  }
}

template <int TENSORS, int PAIRS, typename P>
static int launch_copy(void* const* tensors, const long long* row_bytes, int n_tensors, const int* src, const int* dst, int n_pairs, void* stream) {
  constexpr int kChunk = kCopyThreads * kCopyAhead * (int)sizeof(P);
  static_assert(sizeof(CopyArgs<TENSORS, PAIRS>) <= 32764, "the arguments of a launch");
  CopyArgs<TENSORS, PAIRS> a;
  for (int p0 = 0; p0 < n_pairs; p0 += PAIRS) {
    a.pairs = n_pairs - p0 < PAIRS ? n_pairs - p0 : PAIRS;
    a.tensors = 0;
    long long chunks = 0;
    for (int i = 0; i < n_tensors; ++i) {
      a.base[i] = (unsigned char*)tensors[i];
      a.row_bytes[i] = row_bytes[i];
      chunks += (row_bytes[i] + kChunk - 1) / kChunk;
      PTL_REQUIRE(chunks <= 0x7fffffffLL, "copy_pages: rows are too large");
      a.chunk_end[i] = (int)chunks;
    }
    a.tensors = n_tensors;
    for (int i = 0; i < a.pairs; ++i) { a.src[i] = src[p0 + i]; a.dst[i] = dst[p0 + i]; }
    const long long total = chunks * a.pairs;
    const int grid = (int)(total < 148 * 16 ? total : 148 * 16);
    if (int rc = launch_kernel("copy_pages", copy_pages_kernel<TENSORS, PAIRS, P>, dim3(grid), dim3(kCopyThreads), 0, as_stream(stream), a)) return rc;
  }
  return 0;
}

}  // namespace ptl

// `tensors`, `row_bytes`, `src` and `dst` are host arrays: the tensors' addresses, the bytes of a row of each, and the rows, which
// the caller has checked to lie in every tensor, with no dst twice and none among the src.  *launches: kernels launched.
PTL_EXPORT int ptl_copy_pages(void* const* tensors, const long long* row_bytes, int n_tensors, const int* src, const int* dst, int n_pairs,
                              int* launches, void* stream) {
  using namespace ptl;
  PTL_REQUIRE(n_tensors >= 0 && n_pairs >= 0, "copy_pages: bad sizes");
  *launches = 0;
  for (int i = 0; i < n_tensors; ++i) PTL_REQUIRE(tensors[i] && row_bytes[i] > 0, "copy_pages: tensor %d has no rows", i);
  if (n_pairs == 0) return 0;
  for (int t0 = 0; t0 < n_tensors; t0 += kCopyMaxTensors) {
    const int n = n_tensors - t0 < kCopyMaxTensors ? n_tensors - t0 : kCopyMaxTensors;
    uintptr_t mixed = 0;
    for (int i = t0; i < t0 + n; ++i) mixed |= reinterpret_cast<uintptr_t>(tensors[i]) | (uintptr_t)row_bytes[i];
    void* const* t = tensors + t0;
    const long long* b = row_bytes + t0;
    const bool few = n <= 32 && n_pairs <= 128;
    int rc;
    if (mixed % 16 == 0)
      rc = few ? launch_copy<32, 128, uint4>(t, b, n, src, dst, n_pairs, stream) : launch_copy<kCopyMaxTensors, 3700, uint4>(t, b, n, src, dst, n_pairs, stream);
    else if (mixed % 4 == 0)
      rc = few ? launch_copy<32, 128, uint32_t>(t, b, n, src, dst, n_pairs, stream) : launch_copy<kCopyMaxTensors, 3700, uint32_t>(t, b, n, src, dst, n_pairs, stream);
    else
      rc = launch_copy<kCopyMaxTensors, 3700, unsigned char>(t, b, n, src, dst, n_pairs, stream);
    if (rc) return rc;
    *launches += few ? 1 : (n_pairs + 3699) / 3700;
  }
  return 0;
}
