// Writing keys and values into an 8-bit cache (kv8.cuh), and reading them back.
//
// Write.  qkv is a step's projection [tokens, (nq + 2 nkv) d] as in rope_kv.cu: q is turned by position * inv_freq
// in place; k, turned likewise and rounded to the step's type, and v go into the blocks that `slots` name.  The k and v columns of
// qkv stay as they are.  The rows of one block of 16 positions stand next to each other in the step (a request's tokens do): a
// run.  One warp does a run's work for one head's k or v: it reads the values once, into registers, for the largest magnitude
// and the marks; then, where the block's exponent grows, the codes that are there are made coarser; then come the new codes.  A run
// that holds the block's first position starts the block anew.  A block of threads looks at one row of the step, or, in steps
// of many rows, at 16, and takes the runs that begin there.
//
// What bounds it: three loads that wait for one another (slots, then the run's values and the word, then, where the exponent grows, the codes) and
// the launch; one rounding a code, by fma.rd.  Four prompts of 301 to 1,021 tokens (8 heads of 128) are written and read back in 13.2 us,
// of which the bytes take 5.2; 64 single tokens in 8.2 of 1.5.  That is without turning; a model's step turns q and k.  With 32 query heads of 64
// and 128, bfloat16: 8 tokens 4.4 and 5.7 us, 64 4.6 and 5.9, the four prompts 36 and 75, 8,000 tokens 89 and 192.  There q bounds it, turned in place an
// element at a time (8,000 tokens without q 26 and 58), and a write into the other cache, two elements at a time, takes 24 and 43.
// Five blocks an SM (up to 96 registers): over steps of 8 to 8,000 rows, heads of 64 and 128, both types, turned and not, it is on average within
// 2 to 10 % of the best of three to six for each instance; three is 3 to 24 % off, four 6 to 18, six 0 to 9 and for float32 heads of 128, unturned, which
// then spill, 28.  (With five the heads of 128 spill 16 to 28 bytes, but bfloat16 unturned.)  Reading back and making pages bfloat16 are
// given up to 80 registers, so that a thread's four packets are asked for at once (the compiler keeps to 64: 9.4 and 15.4 us).
#include "kv8.cuh"
#include <cstring>

namespace ptl {

constexpr int kKv8Threads = 256;
constexpr int kKv8WriteThreads = 128;

template <int N> struct Kv8Packet;
template <> struct Kv8Packet<8> { using type = uint2; };
template <> struct Kv8Packet<4> { using type = uint32_t; };

// (cos, sin) of an angle: a call, so that the kernel holds it once.
__device__ __noinline__ float2 kv8_angle(float a) {
  float2 r;
  sincosf(a, &r.y, &r.x);
  return r;
}

struct Kv8WriteParams {
  void* qkv;
  const int* positions;
  const float* inv_freq;
  const int* slots;
  unsigned char* codes;
  uint32_t* words;
  int tokens, nq, nkv, d, rot, page_size, rows_per_block, early;      // early: see the kernel
  long long num_slots;

  // The block of 16 positions that a row goes to, -1: none.
  __device__ __forceinline__ int block_of(int row) const {
    const int s = row >= 0 && row < tokens ? __ldg(slots + row) : -1;
    return s >= 0 && s < num_slots ? s / kKv8Block : -1;
  }
  __device__ __forceinline__ float2 angle(int row, int j) const { return kv8_angle((float)__ldg(positions + row) * inv_freq[j]); }
};

// The turned values of packet `i` of a k head in `row`; cs: cos[half], sin[half] of the row, or null.
template <typename T>
__device__ __forceinline__ void kv8_turn(const Kv8WriteParams& p, float (&x)[Vec16<T>::N], const T* head, int i, int row, const float* cs) {
  constexpr int N = Vec16<T>::N;
  const int half = p.rot / 2;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = i * N + j;
    if (e >= p.rot) break;
    const bool low = e < half;
    const int a = low ? e : e - half;
    float o1, o2;
    const float2 cos_sin = cs ? make_float2(cs[a], cs[half + a]) : p.angle(row, a);
    const float other = to_f32(head[low ? e + half : a]);
    rope_rotate(low ? x[j] : other, low ? other : x[j], cos_sin.x, cos_sin.y, o1, o2);
    x[j] = to_f32(from_f32<T>(low ? o1 : o2));
  }
}

// D: the head size, or 0 for any (then the values are read twice).  TURN: there are frequencies.
template <typename T, int D, bool TURN>
__global__ void __launch_bounds__(kKv8WriteThreads, 5)
rope_kv8_write_kernel(const Kv8WriteParams p) {
  extern __shared__ float cs[];                  // [rows staged][cos[half], sin[half]]
  constexpr int N = Vec16<T>::N;
  constexpr int kPackets = D ? kKv8Block * D / N / 32 : 1;     // a lane has of a run's 16 rows
  const int d = D ? D : p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_len = (p.nq + 2 * p.nkv) * d, half = p.rot / 2;
  const int t0 = blockIdx.x * p.rows_per_block, t1 = min(p.tokens, t0 + p.rows_per_block);
  T* qkv = static_cast<T*>(p.qkv);
  // positions, slots and frequencies may be results of the kernel before this one, unless the caller says that they are not (a model's
  // step, whose integers were there before its first kernel)
  if (!p.early) pdl_wait();
  const int mine = p.block_of(t0 - 1 + lane);                  // (rows t0 - 1 .. t0 + 30)
  const int before = __shfl_up_sync(0xffffffffu, mine, 1);
  const unsigned leads = __ballot_sync(0xffffffffu, lane >= 1 && t0 - 1 + lane < t1 && mine >= 0 && mine != before) >> 1;      // bit i: row t0 + i begins a run
  if (!leads && (p.nq == 0 || !TURN)) {
    pdl_wait();                                  // (what comes after this kernel counts on the one before it being through)
    return;
  }
  int staged = 0;                                              // rows from t0 on whose angles are in shared memory
  if constexpr (TURN) {
    const int last = 31 - __clz(leads | 1u);                   // the last run's first row, and up to 16 of its rows
    const int of_last = __shfl_sync(0xffffffffu, mine, last + 1);
    const unsigned same = __ballot_sync(0xffffffffu, lane > last && mine == of_last) >> (last + 1);
    staged = max(t1 - t0, leads ? last + min(kKv8Block, __ffs(~same) - 1) : 0);
    for (int e = threadIdx.x; e < staged * half; e += kKv8WriteThreads) {
      if (t0 + e / half >= p.tokens) break;
      const float2 cos_sin = p.angle(t0 + e / half, e % half);
      cs[e / half * p.rot + e % half] = cos_sin.x;
      cs[e / half * p.rot + half + e % half] = cos_sin.y;
    }
  }
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  if constexpr (TURN) {                          // q of these rows, in place
    for (int e = blockIdx.y * kKv8WriteThreads + threadIdx.x; e < (t1 - t0) * p.nq * half; e += gridDim.y * kKv8WriteThreads) {
      const int r = e / (p.nq * half), j = e % half;
      T* head = qkv + (size_t)(t0 + r) * row_len + (size_t)(e / half % p.nq) * d;
      float o1, o2;
      rope_rotate(to_f32(head[j]), to_f32(head[j + half]), cs[r * p.rot + j], cs[r * p.rot + half + j], o1, o2);
      head[j] = from_f32<T>(o1);
      head[j + half] = from_f32<T>(o2);
    }
  }
  const int blocks_per_page = p.page_size / kKv8Block, units = 2 * p.nkv, packets = d / N;
  for (int task = blockIdx.y * (kKv8WriteThreads / 32) + warp; task < __popc(leads) * units; task += gridDim.y * (kKv8WriteThreads / 32)) {
    const int unit = task % units, g = unit >> 1, part = unit & 1;
    int first = t0 + __fns(leads, 0, task / units + 1);
    const int block = p.block_of(first);
    const int page = block / blocks_per_page, sub = block % blocks_per_page;
    unsigned char* dst = p.codes + (((size_t)page * 2 + part) * p.nkv + g) * p.page_size * d + (size_t)sub * kKv8Block * d;
    uint32_t* word = p.words + ((size_t)page * p.nkv + g) * blocks_per_page * 2 + sub * 2 + part;
    const bool turned = TURN && part == 0;
    while (true) {                               // up to 16 rows at a time (more: the same positions again)
      const int slot = lane < kKv8Block && first + lane < p.tokens ? __ldg(p.slots + first + lane) : -1;
      const unsigned others = __ballot_sync(0xffffffffu, slot < 0 || slot >= p.num_slots || slot / kKv8Block != block);
      const int rows = __ffs(others) - 1;        // (lanes 16 to 31 are others)
      if (rows == 0) break;
      const int off = slot % kKv8Block;
      const uint32_t here = __reduce_or_sync(0xffffffffu, lane < rows ? 1u << off : 0u);
      const T* src = qkv + (size_t)first * row_len + (size_t)(p.nq + part * p.nkv + g) * d;
      const uint32_t had = *word;
      Vec16<T> raw[kPackets];                    // (turned, once they have been looked at)
      auto fetch = [&](int e) { return load16(src + (size_t)(e / packets) * row_len + e % packets * N); };
      auto turn = [&](int e, Vec16<T>& v) {
        if constexpr (TURN) {
          if (!turned) return;
          float x[N];
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = v.get(j);
          const int row = first + e / packets;
          kv8_turn<T>(p, x, src + (size_t)(e / packets) * row_len, e % packets, row, row - t0 < staged ? cs + (row - t0) * p.rot : nullptr);
#pragma unroll
          for (int j = 0; j < N; ++j) v.set(j, x[j]);
        }
      };
      // Bits of the largest magnitude, marked values among them: those of infinity and NaN are larger than all others, so one look at
      // the largest of the run tells whether there is one, and only then the tokens are looked through.
      uint32_t amax = 0u, bad = 0u;
      auto look = [&](const Vec16<T>& v) {
#pragma unroll
        for (int j = 0; j < N; ++j) amax = max(amax, __float_as_uint(v.get(j)) & 0x7fffffffu);
      };
      constexpr uint32_t kInf = 0x7f800000u;
      auto look_closely = [&](const Vec16<T>& v, int row_off) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint32_t mag = __float_as_uint(v.get(j)) & 0x7fffffffu;
          if (mag >= kInf) bad |= 1u << row_off;
          else amax = max(amax, mag);
        }
      };
      int offs[kPackets];                        // of the packets' rows in the block of 16
      if constexpr (D != 0) {
#pragma unroll
        for (int i = 0; i < kPackets; ++i) {
          if (lane + 32 * i < rows * packets) raw[i] = fetch(lane + 32 * i);
          offs[i] = __shfl_sync(0xffffffffu, off, (lane + 32 * i) / packets);
        }
#pragma unroll
        for (int i = 0; i < kPackets; ++i)
          if (lane + 32 * i < rows * packets) { turn(lane + 32 * i, raw[i]); look(raw[i]); }
      } else {
        for (int e = lane; e < rows * packets; e += 32) {
          Vec16<T> v = fetch(e);
          turn(e, v);
          look(v);
        }
      }
      amax = __reduce_max_sync(0xffffffffu, amax);
      if (amax >= kInf) {
        amax = 0u;
        if constexpr (D != 0) {
#pragma unroll
          for (int i = 0; i < kPackets; ++i)
            if (lane + 32 * i < rows * packets) look_closely(raw[i], offs[i]);
        } else {
          for (int e = lane; e < rows * packets; e += 32) {
            Vec16<T> v = fetch(e);
            turn(e, v);
            look_closely(v, __ldg(p.slots + first + e / packets) % kKv8Block);
          }
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
        bad = __reduce_or_sync(0xffffffffu, bad);
      }
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
      }
      __syncwarp();
      const float inverse = e_new ? kv8_inverse_step(e_new) : 0.f;
      auto store = [&](int e, const Vec16<T>& v, int row_off) {
        uint32_t out[N / 4];
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          uint32_t u[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) u[k] = kv8_code(v.get(j + k), inverse);
          if (bad) {                             // (what is no finite number is kept as 128)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((__float_as_uint(v.get(j + k)) & 0x7fffffffu) >= kInf) u[k] = 128u;
          }
          out[j / 4] = __byte_perm(__byte_perm(u[0], u[1], 0x0040u), __byte_perm(u[2], u[3], 0x0040u), 0x5410u);
        }
        *reinterpret_cast<typename Kv8Packet<N>::type*>(dst + (size_t)row_off * d + e % packets * N) = *reinterpret_cast<typename Kv8Packet<N>::type*>(out);
      };
      if constexpr (D != 0) {
#pragma unroll
        for (int i = 0; i < kPackets; ++i)
          if (lane + 32 * i < rows * packets) store(lane + 32 * i, raw[i], offs[i]);
      } else {
        for (int e = lane; e < rows * packets; e += 32) {
          Vec16<T> v = fetch(e);
          turn(e, v);
          store(e, v, __ldg(p.slots + first + e / packets) % kKv8Block);
        }
      }
      if (lane == 0) *word = (uint32_t)e_new | ((((anew ? 0u : had >> 16) & ~here) | bad) << 16);
      __syncwarp();
      first += rows;
      if (rows < kKv8Block) break;
    }
  }
}

// Keys and values of the first length[r] tokens of the requests as numbers, request after request: out [tokens][2][heads][d].  A block of
// threads takes packets of 16 codes, four a thread, of 16 positions of a request, which lie in one page, in the order in which they lie there.
constexpr int kKv8ReadAhead = 4;
template <int REQUESTS> struct Kv8ReadArgs {
  long long first_row;                     // of the output
  int requests, first_request;
  int end[REQUESTS];                       // tokens of this launch's requests up to and with each
};

template <typename T, int REQUESTS>
__global__ void __launch_bounds__(kKv8Threads, 3)
read_kv8_kernel(T* __restrict__ out, const unsigned char* __restrict__ codes, const uint32_t* __restrict__ words,
                const int* __restrict__ block_table, const __grid_constant__ Kv8ReadArgs<REQUESTS> args, int bt_stride, int nkv, int d, int page_size,
                int num_pages) {
  const int r = blockIdx.y, pos0 = blockIdx.x * kKv8Block;
  const int t0 = r ? args.end[r - 1] : 0, tokens = min(kKv8Block, args.end[r] - t0 - pos0);
  if (tokens <= 0) return;
  pdl_wait();                              // (the table may be a result of the kernel before this one)
  pdl_launch_dependents();
  const int page = __ldg(block_table + (size_t)(args.first_request + r) * bt_stride + pos0 / page_size), sub = pos0 % page_size / kKv8Block;
  const bool here = page >= 0 && page < num_pages;           // (a position that has no page reads as 0)
  const unsigned per_row = d / 16, total = 2u * nkv * d;     // packets of a row, and of the 16 positions
  const unsigned char* src = codes + (size_t)(here ? page : 0) * 2 * nkv * page_size * d + (size_t)sub * kKv8Block * d;
  const uint32_t* word0 = words + (size_t)(here ? page : 0) * nkv * (page_size / kKv8Block) * 2 + sub * 2;
  T* dst0 = out + (args.first_row + t0 + pos0) * 2 * nkv * d;
  for (unsigned x0 = blockIdx.z * kKv8Threads * kKv8ReadAhead + threadIdx.x; x0 < total; x0 += gridDim.z * kKv8Threads * kKv8ReadAhead) {
    uint4 c[kKv8ReadAhead];
    uint32_t w[kKv8ReadAhead];
#pragma unroll
    for (int i = 0; i < kKv8ReadAhead; ++i) {
      const unsigned x = x0 + i * kKv8Threads, head = x / d, part = head >= (unsigned)nkv, in_head = x - head * d;
      if (x >= total || !here) continue;
      c[i] = __ldg(reinterpret_cast<const uint4*>(src + (size_t)head * page_size * d) + in_head);
      w[i] = __ldg(word0 + (head - part * nkv) * (page_size / kKv8Block) * 2 + part);
    }
#pragma unroll
    for (int i = 0; i < kKv8ReadAhead; ++i) {
      const unsigned x = x0 + i * kKv8Threads, head = x / d, in_head = x - head * d, off = in_head / per_row, col = (in_head - off * per_row) * 16;
      if (x >= total || off >= (unsigned)tokens) continue;
      const float half_step = here ? kv8_half_step(w[i] & 255u) : 0.f;
      const bool bad = here && ((w[i] >> (16 + off)) & 1u);
      T* dst = dst0 + (size_t)off * 2 * nkv * d + head * d + col;
      Vec16<T> p;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t four = j < 4 ? c[i].x : j < 8 ? c[i].y : j < 12 ? c[i].z : c[i].w;
        const float v = here ? (float)(2 * (int)((four >> (8 * (j & 3))) & 255u) - 255) * half_step : 0.f;
        p.set(j % Vec16<T>::N, bad ? __uint_as_float(0x7fc00000u) : v);
        if (j % Vec16<T>::N == Vec16<T>::N - 1) store16(dst + j + 1 - Vec16<T>::N, p);
      }
    }
  }
}

// The pages that a step's portions see, made bfloat16 (which holds every value exactly) in a place of their own, for the attention
// of portions on the fifth-generation tensor cores: the tiles of a prompt multiply the same keys for every query head and 256 rows, and
// making numbers of codes there cost more than the products (2,048 tokens of 32 heads of 64: 76 us with warps of their own for it, 133 on
// mma.sync, 44 from bfloat16).  The j-th request with portions, counted in the order of the tiles (pairs of {request, first row,
// rows, first position}, as the attention takes them), has pages j * width .. of `pages` in the order of its positions;
// table[request] says so, -1 where it has no page.  Page slots * width is zeros.  A marked token's key is NaN and its value
// the finite part, so that it reaches the rows that see it and no other.  Blocks of threads a page (a thread has four
// packets of 16 codes of it) and pair; a request's first pair works.
struct Kv8ExpandParams {
  __nv_bfloat16* pages;
  int* table;
  const unsigned char* codes;
  const uint32_t* words;
  const int* block_table;
  const int* tiles;
  int pairs, slots, width, nkv, d, page_size, num_pages, window, early;      // early: as for a write
};

constexpr int kKv8ExpandChunk = kKv8Threads * kKv8ReadAhead;      // packets of a page a block takes

__global__ void __launch_bounds__(kKv8Threads, 3)
kv8_expand_kernel(const Kv8ExpandParams p) {
  if (!p.early) pdl_wait();                // (tiles and the block table)
  const int page_codes = 2 * p.nkv * p.page_size * p.d, lane = threadIdx.x & 31;
  const int pair = blockIdx.y, chunk = blockIdx.z * kKv8ExpandChunk;      // of the page's packets of 16 codes
  auto request = [&](int i) { return i >= 0 && i < p.pairs && __ldg(p.tiles + 8 * i + 2) > 0 ? __ldg(p.tiles + 8 * i) : -1; };
  const int r = request(pair);
  const bool works = r >= 0 && request(pair - 1) != r;
  int before = 0, lo = 0, hi = 0;
  if (works) {
    // requests before this one, and the end of this one's last portion (every warp for itself)
    int end = 0;
    for (int i = lane; i < p.pairs; i += 32) {
      const int ri = request(i);
      if (i < pair && ri >= 0 && request(i - 1) != ri) ++before;
      if (i >= pair && ri == r) end = max(end, __ldg(p.tiles + 8 * i + 3) + __ldg(p.tiles + 8 * i + 2) + max(0, __ldg(p.tiles + 8 * i + 6)));
    }
    before = __reduce_add_sync(0xffffffffu, before);
    end = __reduce_max_sync(0xffffffffu, end);
    const int pos0 = __ldg(p.tiles + 8 * pair + 3);
    lo = p.window > 0 && pos0 + 1 > p.window ? (pos0 + 1 - p.window) / p.page_size : 0;
    hi = before < p.slots ? min((end + p.page_size - 1) / p.page_size, p.width) : 0;      // (there are as many slots as such requests)
  }
  auto page_at = [&](int b) { return b < hi ? __ldg(p.block_table + (size_t)r * p.width + b) : -1; };
  int b = lo + blockIdx.x, page = page_at(b);
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = 2 * chunk + threadIdx.x; i < min(page_codes / 8, 2 * (chunk + kKv8ExpandChunk)); i += kKv8Threads)
      reinterpret_cast<uint4*>(p.pages + (size_t)p.slots * p.width * page_codes)[i] = make_uint4(0u, 0u, 0u, 0u);
  const int blocks = p.page_size / kKv8Block, per_row = p.d / 16;
  for (; b < hi; b += gridDim.x) {
    const int to = before * p.width + b;
    const bool here = page >= 0 && page < p.num_pages;
    if (threadIdx.x == 0 && blockIdx.z == 0) p.table[(size_t)r * p.width + b] = here ? to : -1;
    const uint4* src = reinterpret_cast<const uint4*>(p.codes + (size_t)(here ? page : 0) * page_codes);
    uint4* dst = reinterpret_cast<uint4*>(p.pages + (size_t)to * page_codes);
    const uint2* words = reinterpret_cast<const uint2*>(p.words) + (size_t)(here ? page : 0) * p.nkv * blocks;
    uint4 c[kKv8ReadAhead];
    uint2 w[kKv8ReadAhead];
#pragma unroll
    for (int k = 0; k < kKv8ReadAhead; ++k) {
      const int i = chunk + k * kKv8Threads + threadIdx.x, row = i / per_row, g = row / p.page_size % p.nkv, off = row % p.page_size;
      if (!here || i >= page_codes / 16) continue;
      c[k] = __ldg(src + i);
      w[k] = __ldg(words + g * blocks + off / kKv8Block);
    }
    page = page_at(b + gridDim.x);
#pragma unroll
    for (int k = 0; k < kKv8ReadAhead; ++k) {
      const int i = chunk + k * kKv8Threads + threadIdx.x, row = i / per_row, part = row / (p.nkv * p.page_size), off = row % p.page_size;
      if (!here || i >= page_codes / 16) continue;
      // Values' exponents are 0 or 16 to 254.  A block that nothing was written to may say what it likes: its keys are masked, but its values are
      // multiplied by 0 and so must be numbers.
      const int e = min(254, (int)((part ? w[k].y : w[k].x) & 255u));
      const float step = 2.0f * kv8_half_step(e < kKv8MinExponent ? 0 : e);
      const bool marked = part == 0 && (((w[k].x | w[k].y) >> (16 + off % kKv8Block)) & 1u);
      uint32_t out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t four = j < 2 ? c[k].x : j < 4 ? c[k].y : j < 6 ? c[k].z : c[k].w;
        const float lo2 = (float)((four >> (16 * (j & 1))) & 255u) - 127.5f, hi2 = (float)((four >> (16 * (j & 1) + 8)) & 255u) - 127.5f;
        const __nv_bfloat162 two = __floats2bfloat162_rn(lo2 * step, hi2 * step);
        out[j] = marked ? 0x7fc07fc0u : *reinterpret_cast<const uint32_t*>(&two);
      }
      dst[2 * i] = make_uint4(out[0], out[1], out[2], out[3]);
      dst[2 * i + 1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

template <typename T>
static int rope_kv8_write(T* qkv, const int* positions, const float* inv_freq, const int* slots, void* codes, void* words, int tokens, int nq,
                          int nkv, int d, int rot, int page_size, int early, long long num_slots, void* stream) {
  PTL_REQUIRE(tokens >= 0 && nq >= 0 && nkv > 0 && d > 0 && page_size > 0 && num_slots >= 0, "rope_kv8_write: bad sizes");
  PTL_REQUIRE(d % 16 == 0 && d <= 256, "rope_kv8_write: head size %d is no multiple of 16 up to 256", d);
  PTL_REQUIRE(nkv <= 65535, "rope_kv8_write: too many heads");
  PTL_REQUIRE(page_size % kKv8Block == 0, "rope_kv8_write: pages of %d positions are not whole blocks of %d", page_size, kKv8Block);
  PTL_REQUIRE(rot % 2 == 0 && rot >= 0 && rot <= d, "rope_kv8_write: rotary width %d of head size %d", rot, d);
  PTL_REQUIRE(aligned16(qkv) && aligned16(codes), "rope_kv8_write: qkv and codes must be 16-byte aligned");
  if (tokens == 0) return 0;
  if (rot == 0) inv_freq = nullptr;
  Kv8WriteParams p{qkv, positions, inv_freq, slots, (unsigned char*)codes, (uint32_t*)words, tokens, nq, nkv, d, rot, page_size, 1, early, num_slots};
  // Steps of many rows are mostly prompts, whose runs are long: a block a row asks for every row's slot many times over there.  Written and read
  // back (before reading was faster), us, by one row and by 16 a block: 64 single tokens (8 heads of 64) 9.5 and 25.8; one prompt (8 heads of 128) of 500 8.7 and 9.0, of
  // 1,024 10.4 and 8.5, of 1,500 13.0 and 9.6.
  p.rows_per_block = tokens > 512 ? kKv8Block : 1;
  const size_t smem = inv_freq ? (size_t)(p.rows_per_block + kKv8Block - 1) * rot * sizeof(float) : 0;
  auto kernel = inv_freq ? (d == 64 ? rope_kv8_write_kernel<T, 64, true> : d == 128 ? rope_kv8_write_kernel<T, 128, true> : rope_kv8_write_kernel<T, 0, true>)
                         : (d == 64 ? rope_kv8_write_kernel<T, 64, false> : d == 128 ? rope_kv8_write_kernel<T, 128, false> : rope_kv8_write_kernel<T, 0, false>);
  return launch_kernel("rope_kv8_write", kernel, dim3((tokens + p.rows_per_block - 1) / p.rows_per_block, (2 * nkv + kKv8WriteThreads / 32 - 1) / (kKv8WriteThreads / 32)),
                       dim3(kKv8WriteThreads), smem,
                       as_stream(stream), p);
}

template <typename T, int REQUESTS>
static int launch_read_kv8(T* out, const void* codes, const void* words, const int* block_table, const int* lengths, int requests, int bt_stride,
                           int nkv, int d, int page_size, int num_pages, void* stream) {
  Kv8ReadArgs<REQUESTS> args;
  args.first_row = 0;
  for (int r0 = 0; r0 < requests; r0 += REQUESTS) {
    args.first_request = r0;
    args.requests = requests - r0 < REQUESTS ? requests - r0 : REQUESTS;
    long long sum = 0;
    int longest = 0;
    for (int i = 0; i < args.requests; ++i) {
      const int n = lengths[r0 + i];
      longest = n > longest ? n : longest;
      PTL_REQUIRE(n >= 0 && n <= (long long)bt_stride * page_size, "read_kv8: request %d of %d tokens does not fit its row of the table", r0 + i, n);
      sum += n;
      PTL_REQUIRE(sum <= 0x7fffffffLL, "read_kv8: too many tokens");
      args.end[i] = (int)sum;
    }
    if (sum > 0) {
      const int chunks = (2 * nkv * d + kKv8Threads * kKv8ReadAhead - 1) / (kKv8Threads * kKv8ReadAhead);
      if (int rc = launch_kernel("read_kv8", read_kv8_kernel<T, REQUESTS>,
                                 dim3((longest + kKv8Block - 1) / kKv8Block, args.requests, chunks < 64 ? chunks : 64), dim3(kKv8Threads), 0,
                                 as_stream(stream), out, (const unsigned char*)codes, (const uint32_t*)words, block_table, args, bt_stride, nkv, d,
                                 page_size, num_pages))
        return rc;
    }
    args.first_row += sum;
  }
  return 0;
}

template <typename T>
static int read_kv8(T* out, const void* codes, const void* words, const int* block_table, const int* lengths, int requests, int bt_stride,
                    int nkv, int d, int page_size, int num_pages, void* stream) {
  PTL_REQUIRE(requests >= 0 && nkv > 0 && d > 0 && page_size > 0 && num_pages > 0 && bt_stride > 0, "read_kv8: bad sizes");
  PTL_REQUIRE(d % 16 == 0 && page_size % kKv8Block == 0, "read_kv8: head size %d and pages of %d must be multiples of 16", d, page_size);
  PTL_REQUIRE(aligned16(out) && aligned16(codes), "read_kv8: out and codes must be 16-byte aligned");
  // (the host copies the arguments of a launch, however many are used)
  return (requests <= 64 ? launch_read_kv8<T, 64> : launch_read_kv8<T, 960>)(out, codes, words, block_table, lengths, requests, bt_stride, nkv, d, page_size,
                                                                             num_pages, stream);
}

// pages: bfloat16 [slots * width + 1, 2, nkv, page_size, d]; table: int32 [requests, width]; slots: at least the requests with portions.
int kv8_expand_bf16(void* pages, int* table, const void* codes, const void* words, const int* block_table, const int* tiles, int n_tiles, int slots,
                    int width, int nkv, int d, int page_size, int num_pages, int window, int early, void* stream) {
  PTL_REQUIRE(n_tiles >= 0 && n_tiles % 2 == 0 && slots > 0 && width > 0 && nkv > 0 && page_size > 0 && num_pages > 0, "kv8_expand: bad sizes");
  PTL_REQUIRE(d % 16 == 0 && d > 0 && page_size % kKv8Block == 0, "kv8_expand: head size %d and pages of %d must be multiples of 16", d, page_size);
  PTL_REQUIRE(aligned16(pages) && aligned16(codes) && (reinterpret_cast<uintptr_t>(words) & 7u) == 0 && n_tiles / 2 <= 65535, "kv8_expand: alignment");
  if (n_tiles == 0) return 0;
  const int x = width < 1024 ? width : 1024, chunks = (nkv * page_size * d / 8 + kKv8ExpandChunk - 1) / kKv8ExpandChunk;
  PTL_REQUIRE(chunks <= 65535, "kv8_expand: pages are too large");
  return launch_kernel("kv8_expand", kv8_expand_kernel, dim3(x, n_tiles / 2, chunks), dim3(kKv8Threads), 0, as_stream(stream),
                       Kv8ExpandParams{(__nv_bfloat16*)pages, table, (const unsigned char*)codes, (const uint32_t*)words, block_table, tiles,
                                       n_tiles / 2, slots, width, nkv, d, page_size, num_pages, window, early});
}

}  // namespace ptl

// The arguments as the caller packs them: the host converts fourteen of a call's own in 1.4 us, and packs them in 0.3.
struct Kv8WriteArgs {
  void* qkv;
  const int* positions;
  const float* inv_freq;
  const int* slots;
  void *codes, *words, *stream;
  long long num_slots;
  int tokens, nq, nkv, d, rot, page_size;
};
static_assert(sizeof(Kv8WriteArgs) == 8 * 8 + 6 * 4, "as it is packed");
struct Kv8ReadCall {
  void* out;
  const void *codes, *words;
  const int *block_table, *lengths;
  void* stream;
  int requests, bt_stride, nkv, d, page_size, num_pages;
};
static_assert(sizeof(Kv8ReadCall) == 6 * 8 + 6 * 4, "as it is packed");

// See the top of the file.  `inv_freq` null or `rot` 0: nothing is turned.  A slot that is negative or not below num_slots is not written.  The second entry
// is for callers whose positions, inv_freq and slots no kernel that is still under way writes.  `lengths` is a host array.
#define PTL_KV8_WRITE_ENTRY(NAME, T, EARLY)                                                                                               \
  PTL_EXPORT int ptl_rope_kv8_write_##NAME(const void* args) {                                                                            \
    Kv8WriteArgs a;                                                                                                                       \
    memcpy(&a, args, sizeof a);                                                                                                           \
    return ptl::rope_kv8_write<T>((T*)a.qkv, a.positions, a.inv_freq, a.slots, a.codes, a.words, a.tokens, a.nq, a.nkv, a.d, a.rot,        \
                                  a.page_size, EARLY, a.num_slots, a.stream);                                                             \
  }
#define PTL_KV8_ENTRIES(NAME, T)                                                                                                          \
  PTL_KV8_WRITE_ENTRY(NAME, T, 0)                                                                                                         \
  PTL_KV8_WRITE_ENTRY(early_##NAME, T, 1)                                                                                                 \
  PTL_EXPORT int ptl_read_kv8_##NAME(const void* args) {                                                                                  \
    Kv8ReadCall a;                                                                                                                        \
    memcpy(&a, args, sizeof a);                                                                                                           \
    return ptl::read_kv8<T>((T*)a.out, a.codes, a.words, a.block_table, a.lengths, a.requests, a.bt_stride, a.nkv, a.d, a.page_size,      \
                            a.num_pages, a.stream);                                                                                       \
  }
PTL_KV8_ENTRIES(f32, float)
PTL_KV8_ENTRIES(bf16, __nv_bfloat16)
