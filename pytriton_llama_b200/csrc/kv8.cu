// Writing keys and values into an 8-bit cache (kv8.cuh), and reading them back.
//
// Write.  qkv is a step's projection [tokens, (nq + 2 nkv) d] as in rope_kv.cu: q is turned by position * inv_freq
// in place; k, turned likewise and rounded to the step's type, and v go into the blocks that `slots` name.  The k and v columns of
// qkv stay as they are.  The rows of one block of 16 positions stand next to each other in the step (a request's tokens do);
// the first row of such a run does the work for all of it, one warp per (head, k or v): the largest magnitude and the marks of the
// new values, then, where the block's exponent grows, the codes that are there made coarser, then the new codes.  A run
// that holds the block's first position starts the block anew.
#include "kv8.cuh"

namespace ptl {

constexpr int kKv8Threads = 256;

// Packet `i` (of Vec16<T>::N values) of k (part 0, turned) or v (part 1) of one head in one row.
template <typename T>
__device__ __forceinline__ void kv8_values_of(float (&x)[Vec16<T>::N], const T* head, int i, int half, int rot, bool turned,
                                              const float* cs /* cos[half], sin[half] of the row */) {
  constexpr int N = Vec16<T>::N;
  const Vec16<T> a = load16(head + i * N);
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = a.get(j);
  if (!turned || i * N >= rot) return;
  if (half % N == 0) {
    const bool first = i * N < half;
    const Vec16<T> b = load16(head + i * N + (first ? half : -half));
    const int c0 = i * N - (first ? 0 : half);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float o1, o2;
      rope_rotate(first ? x[j] : b.get(j), first ? b.get(j) : x[j], cs[c0 + j], cs[half + c0 + j], o1, o2);
      x[j] = to_f32(from_f32<T>(first ? o1 : o2));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = i * N + j;
    if (e >= rot) break;
    const bool first = e < half;
    const int c = first ? e : e - half;
    float o1, o2;
    rope_rotate(to_f32(head[c]), to_f32(head[c + half]), cs[c], cs[half + c], o1, o2);
    x[j] = to_f32(from_f32<T>(first ? o1 : o2));
  }
}

template <int N> struct Kv8Packet;
template <> struct Kv8Packet<8> { using type = uint2; };
template <> struct Kv8Packet<4> { using type = uint32_t; };

template <typename T>
__global__ void __launch_bounds__(kKv8Threads)
rope_kv8_write_kernel(T* __restrict__ qkv, const int* __restrict__ positions, const float* __restrict__ inv_freq,
                      const int* __restrict__ slots, unsigned char* __restrict__ codes, uint32_t* __restrict__ words, int tokens,
                      int nq, int nkv, int d, int rot, int page_size, long long num_slots) {
  extern __shared__ float cs[];                  // [up to 16 rows][cos[half], sin[half]]
  constexpr int N = Vec16<T>::N;
  const int t = blockIdx.x;
  const int row_len = (nq + 2 * nkv) * d, half = rot / 2;
  // positions, slots and frequencies are inputs of the step, not results of the kernel before this one
  auto block_of = [&](int row) -> long long {
    const int s = row >= 0 && row < tokens ? __ldg(slots + row) : -1;
    return s >= 0 && s < num_slots ? s / kKv8Block : -1;
  };
  const long long block = block_of(t);
  const bool leads = block >= 0 && block_of(t - 1) != block;
  int rows = 0;                                  // of the run (counted up to 16 at a time)
  auto count_rows = [&](int first) {
    int n = 0;
    while (n < kKv8Block && block_of(first + n) == block) ++n;
    return n;
  };
  if (leads) rows = count_rows(t);
  if (!leads && (nq == 0 || !inv_freq)) return;
  auto angles = [&](int first, int n) {
    for (int e = threadIdx.x; e < n * half; e += kKv8Threads) {
      const int r = e / half, j = e % half;
      float s, c;
      sincosf((float)__ldg(positions + first + r) * inv_freq[j], &s, &c);
      cs[r * rot + j] = c;
      cs[r * rot + half + j] = s;
    }
  };
  if (inv_freq) angles(t, max(rows, 1));
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  if (inv_freq) {                                // q of this row, in place
    T* row = qkv + (size_t)t * row_len;
    for (int e = threadIdx.x; e < nq * half; e += kKv8Threads) {
      T* head = row + (size_t)(e / half) * d;
      const int j = e % half;
      float o1, o2;
      rope_rotate(to_f32(head[j]), to_f32(head[j + half]), cs[j], cs[half + j], o1, o2);
      head[j] = from_f32<T>(o1);
      head[j + half] = from_f32<T>(o2);
    }
  }
  if (!leads) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks_per_page = page_size / kKv8Block;
  const long long page = block / blocks_per_page;
  const int sub = (int)(block % blocks_per_page);
  const int packets = d / N;
  int first = t;
  while (true) {
    for (int unit = warp; unit < 2 * nkv; unit += kKv8Threads / 32) {
      const int g = unit >> 1, part = unit & 1;
      const T* src = qkv + (size_t)first * row_len + (size_t)(nq + part * nkv + g) * d;
      const bool turned = part == 0 && inv_freq != nullptr;
      unsigned char* dst = codes + (((size_t)page * 2 + part) * nkv + g) * page_size * d + (size_t)sub * kKv8Block * d;
      uint32_t* word = words + ((size_t)page * nkv + g) * blocks_per_page * 2 + sub * 2 + part;
      const uint32_t had = *word;
      uint32_t amax = 0u, here = 0u, bad = 0u;    // bits of the largest magnitude; tokens of the run, and the marked ones among them
      float x[N];
      for (int e = lane; e < rows * packets; e += 32) {
        const int r = e / packets;
        const uint32_t bit = 1u << (__ldg(slots + first + r) % kKv8Block);
        kv8_values_of<T>(x, src + (size_t)r * row_len, e % packets, half, rot, turned, cs + r * rot);
        here |= bit;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint32_t mag = __float_as_uint(x[j]) & 0x7fffffffu;
          if (mag >= 0x7f800000u) bad |= bit;
          else amax = max(amax, mag);
        }
      }
      amax = __reduce_max_sync(0xffffffffu, amax);
      here = __reduce_or_sync(0xffffffffu, here);
      bad = __reduce_or_sync(0xffffffffu, bad);
      const bool anew = here & 1u;
      const int e_old = anew ? 0 : (int)(had & 255u);
      const int e_new = max(e_old, kv8_exponent(amax));
      if (!anew && e_new > e_old) {
        const int n = e_old == 0 ? 7 : e_new - e_old;
        for (int i = lane; i < kKv8Block * d / 16; i += 32) {
          uint4 v = reinterpret_cast<uint4*>(dst)[i];
          v.x = kv8_coarser(v.x, n); v.y = kv8_coarser(v.y, n); v.z = kv8_coarser(v.z, n); v.w = kv8_coarser(v.w, n);
          reinterpret_cast<uint4*>(dst)[i] = v;
        }
        __syncwarp();
      }
      const float inverse = e_new ? kv8_inverse_step(e_new) : 0.f;
      for (int e = lane; e < rows * packets; e += 32) {
        const int r = e / packets, i = e % packets;
        kv8_values_of<T>(x, src + (size_t)r * row_len, i, half, rot, turned, cs + r * rot);
        uint32_t out[N / 4];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const bool finite = (__float_as_uint(x[j]) & 0x7fffffffu) < 0x7f800000u;
          const uint32_t u = finite && e_new ? kv8_code(x[j], inverse) : 128u;
          out[j / 4] = j % 4 ? out[j / 4] | u << (8 * (j % 4)) : u;
        }
        *reinterpret_cast<typename Kv8Packet<N>::type*>(dst + (size_t)(__ldg(slots + first + r) % kKv8Block) * d + i * N) =
            *reinterpret_cast<typename Kv8Packet<N>::type*>(out);
      }
      if (lane == 0) *word = (uint32_t)e_new | ((((anew ? 0u : had >> 16) & ~here) | bad) << 16);
      __syncwarp();
    }
    first += rows;
    rows = count_rows(first);                    // more rows than positions: the same ones again
    if (rows == 0) break;
    __syncthreads();
    if (inv_freq) angles(first, rows);
    __syncthreads();
  }
}

// Keys and values of the first length[r] tokens of the requests as numbers, request after request: out [tokens][2][heads][d].
constexpr int kKv8ReadRequests = 960;
struct Kv8ReadArgs {
  long long first_row;                     // of the output
  int requests, first_request;
  int end[kKv8ReadRequests];               // tokens of this launch's requests up to and with each
};

template <typename T>
__global__ void __launch_bounds__(kKv8Threads)
read_kv8_kernel(T* __restrict__ out, const unsigned char* __restrict__ codes, const uint32_t* __restrict__ words,
                const int* __restrict__ block_table, const __grid_constant__ Kv8ReadArgs args, int bt_stride, int nkv, int d, int page_size,
                int num_pages) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int N = 8;                     // codes a thread takes
  const int per_token = 2 * nkv * d / N;
  const long long total = (long long)args.end[args.requests - 1] * per_token;
  for (long long i = (long long)blockIdx.x * kKv8Threads + threadIdx.x; i < total; i += (long long)gridDim.x * kKv8Threads) {
    const int t = (int)(i / per_token), e = (int)(i % per_token) * N;
    int lo = 0, hi = args.requests - 1;    // the first request that ends behind t
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (args.end[mid] > t) hi = mid; else lo = mid + 1;
    }
    const int pos = t - (lo ? args.end[lo - 1] : 0);
    const int page = block_table[(size_t)(args.first_request + lo) * bt_stride + pos / page_size];
    const int part = e / (nkv * d), g = e / d % nkv, off = pos % page_size;
    float v[N];
    if (page >= 0 && page < num_pages) {
      const uint2 c = *reinterpret_cast<const uint2*>(codes + ((((size_t)page * 2 + part) * nkv + g) * page_size + off) * d + e % d);
      const uint32_t w = words[(((size_t)page * nkv + g) * (page_size / kKv8Block) + off / kKv8Block) * 2 + part];
      const float half_step = kv8_half_step(w & 255u);
      const bool bad = w >> (16 + off % kKv8Block) & 1u;
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] = bad ? __uint_as_float(0x7fc00000u) : (float)(2 * (int)(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 255u) - 255) * half_step;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = 0.f;          // a position that has no page
    }
    T* dst = out + (args.first_row + t) * 2 * nkv * d + e;
    Vec16<T> p;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      p.set(j % Vec16<T>::N, v[j]);
      if (j % Vec16<T>::N == Vec16<T>::N - 1) store16(dst + j + 1 - Vec16<T>::N, p);
    }
  }
}

template <typename T>
static int rope_kv8_write(T* qkv, const int* positions, const float* inv_freq, const int* slots, void* codes, void* words, int tokens, int nq,
                          int nkv, int d, int rot, int page_size, long long num_slots, void* stream) {
  PTL_REQUIRE(tokens >= 0 && nq >= 0 && nkv > 0 && d > 0 && page_size > 0 && num_slots >= 0, "rope_kv8_write: bad sizes");
  PTL_REQUIRE(d % 16 == 0 && d <= 1024, "rope_kv8_write: head size %d is no multiple of 16 up to 1,024", d);
  PTL_REQUIRE(page_size % kKv8Block == 0, "rope_kv8_write: pages of %d positions are not whole blocks of %d", page_size, kKv8Block);
  PTL_REQUIRE(rot % 2 == 0 && rot >= 0 && rot <= d, "rope_kv8_write: rotary width %d of head size %d", rot, d);
  PTL_REQUIRE(aligned16(qkv) && aligned16(codes), "rope_kv8_write: qkv and codes must be 16-byte aligned");
  if (tokens == 0) return 0;
  if (rot == 0) inv_freq = nullptr;
  const size_t smem = inv_freq ? (size_t)kKv8Block * rot * sizeof(float) : 0;
  static SmemRaised raised = {};
  if (smem > 48 * 1024)
    if (int rc = raise_shared_memory("rope_kv8_write", rope_kv8_write_kernel<T>, kKv8Block * 1024 * 4, raised)) return rc;
  return launch_kernel("rope_kv8_write", rope_kv8_write_kernel<T>, dim3(tokens), dim3(kKv8Threads), smem, as_stream(stream), qkv, positions,
                       inv_freq, slots, (unsigned char*)codes, (uint32_t*)words, tokens, nq, nkv, d, rot, page_size, num_slots);
}

template <typename T>
static int read_kv8(T* out, const void* codes, const void* words, const int* block_table, const int* lengths, int requests, int bt_stride,
                    int nkv, int d, int page_size, int num_pages, void* stream) {
  PTL_REQUIRE(requests >= 0 && nkv > 0 && d > 0 && page_size > 0 && num_pages > 0 && bt_stride > 0, "read_kv8: bad sizes");
  PTL_REQUIRE(d % 16 == 0 && page_size % kKv8Block == 0, "read_kv8: head size %d and pages of %d must be multiples of 16", d, page_size);
  PTL_REQUIRE(aligned16(out) && aligned16(codes), "read_kv8: out and codes must be 16-byte aligned");
  Kv8ReadArgs args;
  args.first_row = 0;
  for (int r0 = 0; r0 < requests; r0 += kKv8ReadRequests) {
    args.first_request = r0;
    args.requests = requests - r0 < kKv8ReadRequests ? requests - r0 : kKv8ReadRequests;
    long long sum = 0;
    for (int i = 0; i < args.requests; ++i) {
      const int n = lengths[r0 + i];
      PTL_REQUIRE(n >= 0 && n <= (long long)bt_stride * page_size, "read_kv8: request %d of %d tokens does not fit its row of the table", r0 + i, n);
      sum += n;
      PTL_REQUIRE(sum <= 0x7fffffffLL, "read_kv8: too many tokens");
      args.end[i] = (int)sum;
    }
    if (sum > 0) {
      const long long blocks = (sum * (2 * nkv * d / 8) + kKv8Threads - 1) / kKv8Threads;
      const int grid = (int)(blocks < 148 * 16 ? blocks : 148 * 16);
      if (int rc = launch_kernel("read_kv8", read_kv8_kernel<T>, dim3(grid), dim3(kKv8Threads), 0, as_stream(stream), out,
                                 (const unsigned char*)codes, (const uint32_t*)words, block_table, args, bt_stride, nkv, d, page_size, num_pages))
        return rc;
    }
    args.first_row += sum;
  }
  return 0;
}

}  // namespace ptl

// See the top of the file.  `inv_freq` null or `rot` 0: nothing is turned.  A slot that is negative or not below num_slots is not written.
#define PTL_KV8_ENTRIES(NAME, T)                                                                                                        \
  PTL_EXPORT int ptl_rope_kv8_write_##NAME(void* qkv, const int* positions, const float* inv_freq, const int* slots, void* codes,       \
                                           void* words, int tokens, int nq, int nkv, int d, int rot, int page_size, long long num_slots, \
                                           void* stream) {                                                                              \
    return ptl::rope_kv8_write<T>((T*)qkv, positions, inv_freq, slots, codes, words, tokens, nq, nkv, d, rot, page_size, num_slots, stream); \
  }                                                                                                                                     \
  PTL_EXPORT int ptl_read_kv8_##NAME(void* out, const void* codes, const void* words, const int* block_table, const int* lengths,       \
                                     int requests, int bt_stride, int nkv, int d, int page_size, int num_pages, void* stream) {         \
    return ptl::read_kv8<T>((T*)out, codes, words, block_table, lengths, requests, bt_stride, nkv, d, page_size, num_pages, stream);    \
  }
PTL_KV8_ENTRIES(f32, float)
PTL_KV8_ENTRIES(bf16, __nv_bfloat16)
