// Attention over an 8-bit cache (kv8.cuh) with mma.sync tensor products: head sizes 64 and 128, up to 16 query heads a kv head.
//
// A code u counts u - 128 = c steps and a half, and c is a half float exactly, so with a query row q = 2^e x, |x| < 2,
//   q . k = s_k 2^e (x . c + sum(x) / 2),        sum_j p_j v_j = sum over blocks of s_v (sum p_j c_j + sum p_j / 2):
// the two products run on half floats with float32 sums, a block's step is a float32 factor of its 16 keys' scores and of its 16
// keys' part of the output, and the halves cost one float32 sum a row.  x is a half float exactly for bfloat16 q (but for entries
// below 2^-14 of the row's largest, which lose bits below 2^-24 of it); weights are rounded to half floats, 2^-11 of each.
// float32 rows take two half floats each, x = x1 + x2 and p = p1 + p2, and twice the products.
//
// Keys and values are the rows of m16n8k16's first operand (S^T = C_k X^T, O^T = C_v^T P^T): 8 query rows fill the other side, where
// they would leave half of the first one empty, and what is made of the codes serves as many tiles of 8 rows as a warp has.
// The 16 dimensions of a step and the 16 rows of a value product may be any, as long as both sides agree, so they are chosen for the
// loads: lane (g, c) reads 16 bytes of key rows g and g + 8 at 16 c, which are its operand of four steps, and D / 8 bytes of value
// rows 2c, 2c + 1, 2c + 8, 2c + 9 at g D / 8, which are its operand of D / 16 products.  A pair of bytes becomes 1024 + u by one
// byte permutation, and 1024 + u - 1152 = c exactly.  Weights come out of the scores' layout by an 8 x 8 transposition.
//
// Warps of several tiles of rows sum the output in units of the largest value step so far, 2^(E - 133), by the products themselves: weights
// carry 2^(E_b - E) of their block.  A block whose step is more than 2^8 smaller, where such a weight would leave the half floats'
// normal numbers, is multiplied by itself and added with its step, as every block of a warp of one tile is.
//
// A row's reference maximum only moves when a score is above it by more than 2^8: the comparison is one vote a turn, and
// the reduction over the keys' lanes and the rescaling of the output happen a few times a row.  Weights count in units of 2^-7, so that
// the largest are 2^15, and those that half floats hold with fewer bits are below 2^-21 of e^reference (2^-13 in a block of small steps).
//
// Keys and values of 16 positions and a head are 16 D bytes each in one piece, and come by bulk copies into rings of slots in shared memory.
// Waits for them are bounded: one that gives up says so in *status, and the block ends once its copies have.
#include "kv8.cuh"
#include "tcgen05_utils.cuh"
#include <cstring>

namespace ptl {

constexpr int kA8Warps = 4;
constexpr int kA8Turn = 2;                                    // blocks of 16 keys a turn
constexpr float kA8Lift = 7.0f;                               // weights are 2^7 e^(score - reference), at most 2^15

struct A8Params {
  void* out;
  float* part_acc;            // [blocks][G][D]
  float* part_ml;             // [blocks][G][2], in units of log2
  int* counters;              // a zero per (row, kv head)
  const void* q;
  const unsigned char* codes;
  const uint32_t* words;
  const int* block_table;
  const int* items;           // singles: token rows, null for 0..; portions: tiles {request, first row, rows, first position}
  const int* tok_req;
  const int* positions;
  const int4* units;
  int* status;
  int q_stride, out_stride, bt_stride, nq, nkv, blocks_per_page, page_shift, num_pages, window, splits, cluster;      // (portions: splits of their keys)
  float scale_log2;

  __device__ __forceinline__ int page_of(const int* table, int block) const {
    const int pg = page_shift >= 0 ? block >> page_shift : block / blocks_per_page;
    const int page = pg < bt_stride ? __ldg(table + pg) : -1;
    return page < num_pages ? page : -1;
  }
  __device__ __forceinline__ int sub_of(int block) const { return page_shift >= 0 ? block & (blocks_per_page - 1) : block % blocks_per_page; }
  template <int D> __device__ __forceinline__ const unsigned char* keys(int page, int kvh, int sub) const {
    return codes + (((size_t)page * 2 * nkv + kvh) * blocks_per_page + sub) * (kKv8Block * D);
  }
  template <int D> __device__ __forceinline__ size_t plane() const { return (size_t)nkv * blocks_per_page * (kKv8Block * D); }
  __device__ __forceinline__ uint2 word(int page, int kvh, int sub) const {
    return __ldg(reinterpret_cast<const uint2*>(words) + ((size_t)page * nkv + kvh) * blocks_per_page + sub);
  }
};

__device__ __forceinline__ float a8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^k, 0 below the normal numbers.
__device__ __forceinline__ float a8_power(int k) { return k < -126 ? 0.f : __uint_as_float((uint32_t)(127 + k) << 23); }
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same, to `c` and not to what is in d.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t a8_prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t x;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(x) : "r"(a), "r"(b), "r"(sel));
  return x;
}
// Bytes 0 and 1 (HIGH: 2 and 3), as half floats u - 128.
template <bool HIGH> __device__ __forceinline__ uint32_t a8_pair(uint32_t bytes) {
  uint32_t y;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a8_prmt(bytes, 0x64646464u, HIGH ? 0x4342u : 0x4140u)), "r"(0x64806480u));
  return y;
}
__device__ __forceinline__ uint32_t a8_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void a8_unpack(uint32_t v, float& lo, float& hi) {
  asm("{\n.reg .f16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(lo), "=f"(hi) : "r"(v));
}
// The transposed 8 x 8 matrix of 16-bit elements of a warp.
__device__ __forceinline__ uint32_t a8_transpose(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ld_peer_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// NT tiles of 8 query rows in a warp.  Lane (g, c) holds, of the rows 8 n + 2c and 8 n + 2c + 1 (j = 0, 1), their statistics and the output's
// dimensions g D / 8 .. (g + 1) D / 8 - 1.
template <int D, typename T, int NT> struct A8Rows {
  static constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr int kSteps = D / 16;
  uint32_t qb[kParts][kSteps][NT][2];
  float half_sum[NT][2];                                     // sum(x) / 2
  float factor[NT][2];                                       // 2^e scale log2(e)
  int first[NT][2], last[NT][2];                             // positions a row sees
  float o[kSteps][NT][4];                                    // dimension 2 i + (e >> 1) of the lane's, row j = e & 1
  float m[NT][2], l[NT][2], w[NT][2];                        // reference maximum (log2), and the lane's sums of p and of p s_v
  static constexpr bool kUnits = NT > 1;
  int unit;                                                  // kUnits: E of the step that o and w are counted in

  // Row `row` of the warp's is query head kvh * group + row % group of token t0 + row / group.  `fetch` asks for what `load` works on.
  static constexpr int kRaw = D / 4 / Vec16<T>::N;           // packets of a row a lane holds
  struct Raw { Vec16<T> v[NT][kRaw]; };
  __device__ __forceinline__ static void fetch(Raw& raw, const A8Params& p, int t0, int tokens, int kvh, int group) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = 8 * n + g;
      const bool here = row < tokens * group;
      const T* src = static_cast<const T*>(p.q) + (size_t)(t0 + (here ? row / group : 0)) * p.q_stride + (size_t)(kvh * group + (here ? row % group : 0)) * D + 16 * c;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        constexpr int kPer = 16 / Vec16<T>::N;
        if (here) raw.v[n][i] = load16(src + 64 * (i / kPer) + i % kPer * Vec16<T>::N);
        else
#pragma unroll
          for (int j = 0; j < Vec16<T>::N; ++j) raw.v[n][i].set(j, 0.f);
      }
    }
  }
  __device__ __forceinline__ void load(const Raw& raw, const A8Params& p, int tokens, int pos0, int group) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    unit = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < kRaw; ++i)
#pragma unroll
        for (int j = 0; j < Vec16<T>::N; ++j) big = fmaxf(big, fabsf(raw.v[n][i].get(j)));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // 2^e with |x| < 2, within the powers of two whose inverse is a normal number
      const uint32_t e = min(max(__float_as_uint(big) >> 23, 2u), 252u);
      const float inverse = __uint_as_float((254u - e) << 23);
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = 4 * k + 2 * j;                       // of the lane's entries, 16 for each 64 dimensions
          float a = raw.v[n][i / Vec16<T>::N].get(i % Vec16<T>::N) * inverse, b = raw.v[n][i / Vec16<T>::N].get(i % Vec16<T>::N + 1) * inverse;
          const uint32_t half = a8_pack(a, b);
          qb[0][k][n][j] = half;
          if (kParts == 2) {
            float fa, fb;
            a8_unpack(half, fa, fb);
            qb[kParts - 1][k][n][j] = a8_pack(a - fa, b - fb);
          }
        }
      // sum(x) of rows 2c and 2c + 1, where the scores will be: the products with ones
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int k = 0; k < kSteps; ++k) mma_f16_16816(sum, ones, qb[part][k][n][0], qb[part][k][n][1]);
      const float f = __uint_as_float(e << 23) * p.scale_log2;
#pragma unroll
      for (int j = 0; j < 2; ++j) {                          // row 8 n + 2c + j is held by the lanes of g = 2c + j here
        half_sum[n][j] = 0.5f * sum[j];
        factor[n][j] = __shfl_sync(0xffffffffu, f, 4 * (2 * c + j));
        const int r = 8 * n + 2 * c + j;
        last[n][j] = r < tokens * group ? pos0 + r / group : -1;
        first[n][j] = p.window > 0 && last[n][j] + 1 > p.window ? last[n][j] + 1 - p.window : 0;
        m[n][j] = -INFINITY; l[n][j] = 0.f; w[n][j] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int x2 = 0; x2 < 4; ++x2) o[i][n][x2] = 0.f;
    }
  }

  // kA8Turn blocks of 16 keys: their keys at slot[b], their values 16 D bytes further, their words, and their first positions.  Positions
  // of [all_first, all_last] are in every row's sight.
  __device__ __forceinline__ void turn(const unsigned char* const (&slot)[kA8Turn], const bool (&have)[kA8Turn], const uint2 (&word)[kA8Turn],
                                       const int (&key0)[kA8Turn], int all_first, int all_last) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float s[kA8Turn][NT][4];
    float f[kA8Turn][NT][2];
#pragma unroll
    for (int b = 0; b < kA8Turn; ++b) {
      const float step = 2.0f * kv8_half_step(word[b].x & 255u);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) f[b][n][j] = fmaxf(factor[n][j] * step, 1e-37f);       // (0 times the -inf of a masked key is none)
      if (have[b]) {
        const uint4* k = reinterpret_cast<const uint4*>(slot[b]);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const uint4 k0 = k[g * (D / 16) + 4 * h + c], k1 = k[(g + 8) * (D / 16) + 4 * h + c];
          const uint32_t x0[4] = {k0.x, k0.y, k0.z, k0.w}, x1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {a8_pair<false>(x0[i]), a8_pair<false>(x1[i]), a8_pair<true>(x0[i]), a8_pair<true>(x1[i])};
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (h == 0 && i == 0 && part == 0)
                  mma_f16_16816(s[b][n], a, qb[0][0][n][0], qb[0][0][n][1], half_sum[n][0], half_sum[n][1], half_sum[n][0], half_sum[n][1]);
                else
                  mma_f16_16816(s[b][n], a, qb[part][4 * h + i][n][0], qb[part][4 * h + i][n][1]);
              }
          }
        }
      }
      const uint32_t marks = (word[b].x | word[b].y) >> 16;
      if (!have[b] || key0[b] < all_first || key0[b] + kKv8Block - 1 > all_last || marks) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int off = g + 8 * (e >> 1), key = key0[b] + off;
            if ((marks >> off) & 1u) s[b][n][e] = __uint_as_float(0x7fc00000u);
            if (!have[b] || key < first[n][e & 1] || key > last[n][e & 1]) s[b][n][e] = -INFINITY;      // (without its keys a block has no scores yet)
          }
      }
    }
    // the largest score of the lane's keys above a row's reference by more than 8 moves the reference
    float top[NT][2];
    bool above = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        top[n][j] = -INFINITY;
#pragma unroll
        for (int b = 0; b < kA8Turn; ++b) top[n][j] = fmaxf(top[n][j], fmaxf(s[b][n][j], s[b][n][2 + j]) * f[b][n][j]);
        above |= top[n][j] > m[n][j] + 8.0f;
      }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float alpha[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(top[n][j], m[n][j]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          alpha[j] = mx == -INFINITY ? 1.0f : a8_exp2(m[n][j] - mx);
          m[n][j] = mx;
          l[n][j] *= alpha[j];
          w[n][j] *= alpha[j];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][n][e] *= alpha[e & 1];
      }
    }
    int ev[kA8Turn];
#pragma unroll
    for (int b = 0; b < kA8Turn; ++b) ev[b] = (int)(word[b].y & 255u);
    if constexpr (kUnits) {
      // the unit follows the largest value step; a block far below it keeps its own
      int e_max = unit;
#pragma unroll
      for (int b = 0; b < kA8Turn; ++b) e_max = max(e_max, ev[b]);
      if (e_max > unit) {
        const float f2 = unit == 0 ? 0.f : a8_power(unit - e_max);      // (nothing but zeros so far: o and w are 0)
        unit = e_max;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          w[n][0] *= f2; w[n][1] *= f2;
#pragma unroll
          for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][n][e] *= f2;
        }
      }
    }
    uint32_t pb[kParts][kA8Turn][NT][2];
    float apart[kA8Turn];                                    // the factor of a block that is multiplied by itself
    bool own[kA8Turn];
#pragma unroll
    for (int b = 0; b < kA8Turn; ++b) {
      own[b] = !kUnits || ev[b] + 8 < unit;
      apart[b] = !kUnits ? 2.0f * kv8_half_step(ev[b]) : ev[b] == 0 ? 0.f : a8_power(ev[b] - unit);
      const float up = own[b] ? 1.0f : a8_power(unit - ev[b]), down = own[b] ? apart[b] : 1.0f, shift = own[b] ? 0.f : (float)(ev[b] - unit);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float pr[4];
        const float use[2] = {(m[n][0] == -INFINITY ? 0.f : m[n][0]) - (shift + kA8Lift), (m[n][1] == -INFINITY ? 0.f : m[n][1]) - (shift + kA8Lift)};
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = a8_exp2(fmaf(s[b][n][e], f[b][n][e & 1], -use[e & 1]));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float sum = pr[j] + pr[2 + j];
          l[n][j] = kUnits ? fmaf(sum, up, l[n][j]) : l[n][j] + sum;
          w[n][j] = fmaf(sum, down, w[n][j]);
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t half = a8_pack(pr[2 * x], pr[2 * x + 1]);
            pb[part][b][n][x] = a8_transpose(half);
            if (part + 1 < kParts) {
              float fa, fb;
              a8_unpack(half, fa, fb);
              pr[2 * x] -= fa; pr[2 * x + 1] -= fb;
            }
          }
      }
    }
#pragma unroll
    for (int b = 0; b < kA8Turn; ++b) {
      if (!have[b]) continue;
      uint32_t v[4][D / 32];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned char* row = slot[b] + kKv8Block * D + ((r >> 1) * 8 + 2 * c + (r & 1)) * D + g * (D / 8);
        if constexpr (D == 64) {
          const uint2 x = *reinterpret_cast<const uint2*>(row);
          v[r][0] = x.x; v[r][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(row);
          v[r][0] = x.x; v[r][1] = x.y; v[r][2] = x.z; v[r][3] = x.w;
        }
      }
      // two bytes of each of the four rows: rows 2c and 2c + 1 side by side, then the other two
      auto operand = [&](int x, int y, uint32_t (&a)[4]) {
        const uint32_t lo = a8_prmt(v[0][x], v[1][x], y ? 0x7362u : 0x5140u), hi = a8_prmt(v[2][x], v[3][x], y ? 0x7362u : 0x5140u);
        a[0] = a8_pair<false>(lo); a[1] = a8_pair<true>(lo); a[2] = a8_pair<false>(hi); a[3] = a8_pair<true>(hi);
      };
      if (kUnits && !own[b]) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t a[4];
          operand(i / 2, i % 2, a);
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(o[i][n], a, pb[part][b][n][0], pb[part][b][n][1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t a[4];
          operand(i / 2, i % 2, a);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float acc[4];
            mma_f16_16816(acc, a, pb[0][b][n][0], pb[0][b][n][1], 0.f, 0.f, 0.f, 0.f);
            if (kParts == 2) mma_f16_16816(acc, a, pb[kParts - 1][b][n][0], pb[kParts - 1][b][n][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][n][e] = fmaf(acc[e], apart[b], o[i][n][e]);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void finish() {
    const float step = kUnits ? 2.0f * kv8_half_step(unit) : 1.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
          w[n][j] += __shfl_xor_sync(0xffffffffu, w[n][j], x);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          o[i][n][j] = (o[i][n][j] + 0.5f * w[n][j]) * step;
          o[i][n][2 + j] = (o[i][n][2 + j] + 0.5f * w[n][j]) * step;
        }
      }
  }
  // Entry `i` of the lane's D / 8 dimensions of row 8 n + 2c + j.
  __device__ __forceinline__ float entry(int n, int j, int i) const { return o[i / 2][n][2 * (i % 2) + j]; }
};

// What a row's weight sum l and a part's (m, l) give: parts without keys count nothing, a sum that is no number stays one.
__device__ __forceinline__ float a8_weight(float m, float l, float M) { return l == 0.f ? 0.f : a8_exp2(m - M); }
__device__ __forceinline__ float a8_inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }

template <int D, int NT, int WARPS> struct A8Single {
  static constexpr int kRing = 4;                                          // slots a warp has
  static constexpr int kSlot = 2 * kKv8Block * D;
  static constexpr int kRingBytes = WARPS * kRing * kSlot;
  static constexpr int kJoinBytes = WARPS * 8 * NT * (D + 2) * 4;          // the warps' rows, where the rings were
  static constexpr int kPartBytes = 8 * NT * D * 12 + 8 * 12;              // what a cluster's blocks send: (output, maximum, sum) of a share's entries
  static constexpr int kSmem = kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes;
};

// Single tokens: the warps of a block take turns through the keys of one (token, kv head), or of a part of them, and join
// through shared memory.  The parts of a (token, kv head) join in a cluster, or, where the contexts are cut into parts of equal
// length (the list of attention8_units_kernel), in the block that ends last.  Every warp fetches its own keys, kRing blocks ahead.  Eight warps
// halve the turns; four leave more blocks side by side (the choice and its figures: CudaOps._kv8_single_form).
//
// What bounds it: instructions and their latencies, 0.53 of the issue slots at 24 % of the warps an SM holds, tensor pipe 0.11.  A turn has about
// 410, of which 144 make operands out of codes (two a pair of codes), and a warp 1,400 outside of its turns: its query, its tables, the join.  32 heads
// over 8, bfloat16: one token of 4,000 7.8 us (bytes: 0.64; two turns a warp), 64 of 256 to 2,560 27.4 (14.4; 3.4 TB/s; six turns on average), eight of
// 20,011 to 30,011 with heads of 128 84 (64; 4.9 TB/s); float32, eight of 1,000 to 4,096 16.8 (3.3; up to eight turns of twice the products).  Fewer
// registers for half as many blocks more were slower everywhere (64 tokens 33.5 us: 80 registers, spills).
template <int D, typename T, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 && sizeof(T) == 2 && WARPS == 4 ? (D == 64 ? 4 : 3) : 1)
attention8_single_kernel(const A8Params p) {
  using Cfg = A8Single<D, NT, WARPS>;
  constexpr int kRows = 8 * NT, kRing = Cfg::kRing;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t s_full[WARPS][kRing];
  __shared__ int s_last;
  __shared__ volatile int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint32_t full0 = smem_addr(&s_full[warp][0]);
  if (lane == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(full0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) s_abort = 0;
  __syncthreads();
  if (p.cluster) cluster_arrive();                           // (waited for before anything is sent: every block runs by then)
  pdl_wait();
  pdl_launch_dependents();
  const int group = p.nq / p.nkv;
  T* out = static_cast<T*>(p.out);
  int t, r, pos, kvh, split, splits, pair;
  if (p.units) {
    const int4 a = p.units[2 * blockIdx.x], b = p.units[2 * blockIdx.x + 1];
    t = a.x; r = a.y; pos = a.z; kvh = a.w; split = b.x; splits = b.y;
    if (b.z >= 0)                                            // a row without a request: zeros
      for (int e = tid; e < group * D; e += WARPS * 32) out[(size_t)b.z * p.out_stride + (size_t)b.w * group * D + e] = from_f32<T>(0.f);
    if (t < 0) return;
    pair = t * p.nkv + kvh;
  } else {
    splits = p.splits;
    split = blockIdx.x % splits;
    pair = blockIdx.x / splits;
    kvh = pair % p.nkv;
    t = p.items ? p.items[pair / p.nkv] : pair / p.nkv;
    r = p.tok_req[t];
    pos = p.positions[t];
    if (r < 0) {                                             // (every block of a cluster alike)
      if (split == 0)
        for (int e = tid; e < group * D; e += WARPS * 32) out[(size_t)t * p.out_stride + (size_t)kvh * group * D + e] = from_f32<T>(0.f);
      if (p.cluster) cluster_wait();
      return;
    }
  }
  const int lo = p.window > 0 && pos + 1 > p.window ? pos + 1 - p.window : 0;
  const int b0 = lo / kKv8Block, blocks = pos < 0 ? 0 : pos / kKv8Block - b0 + 1;
  const int per = (blocks + splits - 1) / splits;
  const int begin = b0 + min(blocks, split * per), end = b0 + min(blocks, (split + 1) * per);
  // ---- this warp's blocks: begin + warp + 4 i, i < count.  Lane l looks after blocks l, l + 32, ...: where they lie, their words, and their copies
  static_assert(kRing == 4 && kA8Turn == 2, "blocks i + 4 and i + 5 follow blocks i and i + 1 into their slots");
  const int count = max(0, (end - begin - warp + WARPS - 1) / WARPS);
  const int* table = p.block_table + (size_t)r * p.bt_stride;
  auto page_at = [&](int i) { return i < count ? p.page_of(table, begin + warp + WARPS * i) : -1; };
  auto source = [&](int i, int page) { return page >= 0 ? p.keys<D>(page, kvh, p.sub_of(begin + warp + WARPS * i)) : nullptr; };
  auto word_at = [&](int i, int page) { return page >= 0 ? p.word(page, kvh, p.sub_of(begin + warp + WARPS * i)) : make_uint2(0u, 0u); };
  const uint32_t slot0 = smem_addr(smem) + warp * (kRing * Cfg::kSlot);
  const size_t plane = p.plane<D>();
  auto fetch = [&](int slot, const unsigned char* src) {
    const uint32_t bar = full0 + 8 * slot, dst = slot0 + slot * Cfg::kSlot;
    if (!src) { mbar_arrive(bar); return; }
    mbar_expect_tx(bar, Cfg::kSlot);
    bulk_load(dst, src, Cfg::kSlot / 2, bar);
    bulk_load(dst + Cfg::kSlot / 2, src + plane, Cfg::kSlot / 2, bar);
  };
  const int page0 = page_at(lane);
  int page_nxt = page_at(32 + lane);
  A8Rows<D, T, NT> rows;
  typename A8Rows<D, T, NT>::Raw raw;
  rows.fetch(raw, p, t, 1, kvh, group);                       // (asked for beside the pages)
  uint2 word_cur = word_at(lane, page0);                      // (before the copies, behind which it would wait)
  const unsigned char* src_cur = source(lane, page0);
  if (lane < min(kRing, count)) fetch(lane, src_cur);
  __syncwarp();
  rows.load(raw, p, 1, pos, group);
  int gave_up = -1;                                           // the block whose wait ran out
  for (int base = 0; base < count; base += 32) {
    const uint2 word_nxt = word_at(base + 32 + lane, page_nxt);
    const unsigned char* src_nxt = source(base + 32 + lane, page_nxt);
    page_nxt = page_at(base + 64 + lane);
    const int stop = min(32, count - base);
    const unsigned there = __ballot_sync(0xffffffffu, src_cur != nullptr);      // blocks with a page (none behind the last)
    for (int i = 0; i < stop; i += kA8Turn) {
      const unsigned char* slot[kA8Turn];
      bool have[kA8Turn];
      uint2 word[kA8Turn];
      int key0[kA8Turn];
#pragma unroll
      for (int b = 0; b < kA8Turn; ++b) {
        word[b].x = __shfl_sync(0xffffffffu, word_cur.x, i + b);
        word[b].y = __shfl_sync(0xffffffffu, word_cur.y, i + b);
        have[b] = (there >> (i + b)) & 1u;
        key0[b] = (begin + warp + WARPS * (base + i + b)) * kKv8Block;
        slot[b] = smem + warp * (kRing * Cfg::kSlot) + ((i + b) % kRing) * Cfg::kSlot;
        if (i + b < stop && gave_up < 0 &&
            !__all_sync(0xffffffffu, mbar_wait(full0 + 8 * ((i + b) % kRing), ((base + i + b) / kRing) & 1, &s_abort, p.status, 9))) gave_up = base + i + b;
      }
      if (gave_up >= 0) break;
      rows.turn(slot, have, word, key0, lo, pos);
      __syncwarp();                                           // the slots are read: their next blocks
      const int ahead = i + kRing + (lane & 1);
      if ((lane & 30) == ((i + kRing) & 31) && base + ahead < count) fetch(ahead % kRing, ahead < 32 ? src_cur : src_nxt);
    }
    if (gave_up >= 0) break;
    src_cur = src_nxt; word_cur = word_nxt;
  }
  if (gave_up >= 0)                                           // this warp's copies still under way end before the memory is used for something else
    for (int i = gave_up; i < min(gave_up + kRing, count); ++i) mbar_drain(full0 + 8 * (i % kRing), (i / kRing) & 1);
  rows.finish();
  __syncthreads();                                            // the rings are read
  float(*s_o)[kRows][D] = reinterpret_cast<float(*)[kRows][D]>(smem);
  float(*s_m)[kRows] = reinterpret_cast<float(*)[kRows]>(smem + WARPS * kRows * D * 4);
  float(*s_l)[kRows] = s_m + WARPS;
  // behind them, what the cluster's blocks send: [part][entry of this block's share] outputs, then maxima, then sums
  float* s_part = reinterpret_cast<float*>(smem + Cfg::kSmem);
  const int share = p.cluster ? (group * D + splits - 1) / splits : 0, shares = share * splits;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * c + j;
#pragma unroll
      for (int i = 0; i < D / 8; i += 4)
        *reinterpret_cast<float4*>(&s_o[warp][row][g * (D / 8) + i]) =
            make_float4(rows.entry(n, j, i), rows.entry(n, j, i + 1), rows.entry(n, j, i + 2), rows.entry(n, j, i + 3));
      if (g == 0) { s_m[warp][row] = rows.m[n][j]; s_l[warp][row] = rows.l[n][j]; }
    }
  __syncthreads();
  const bool whole = splits == 1;
  if (p.cluster) cluster_wait();                             // (every block of the cluster runs)
  for (int e = tid; e < group * D; e += WARPS * 32) {
    const int row = e / D, col = e % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) M = fmaxf(M, s_m[i][row]);
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float f = a8_weight(s_m[i][row], s_l[i][row], M);
      if (s_l[i][row] == 0.f) continue;
      L = fmaf(f, s_l[i][row], L);
      acc = fmaf(f, s_o[i][row][col], acc);
    }
    if (whole) {
      out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + col] = from_f32<T>(acc * a8_inverse(L));
    } else if (p.cluster) {
      const uint32_t to = map_to_peer(smem_addr(s_part + split * share + e % share), e / share);
      st_peer_f32(to, acc);
      st_peer_f32(to + 4 * shares, M);
      st_peer_f32(to + 8 * shares, L);
    } else {
      const size_t at = (size_t)blockIdx.x * group + row;
      p.part_acc[at * D + col] = acc;
      if (col == 0) { p.part_ml[2 * at] = M; p.part_ml[2 * at + 1] = L; }
    }
  }
  if (whole) return;
  if (p.cluster) {
    // every block of the cluster finishes its share of the outputs
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    for (int e = tid; e < min(share, group * D - split * share); e += WARPS * 32) {
      const int row = (split * share + e) / D, col = (split * share + e) % D;
      float M = -INFINITY, L = 0.f, acc = 0.f;
      for (int z = 0; z < splits; ++z) M = fmaxf(M, s_part[shares + z * share + e]);
      for (int z = 0; z < splits; ++z) {
        const float m = s_part[shares + z * share + e], l = s_part[2 * shares + z * share + e];
        if (l == 0.f) continue;
        const float f = a8_weight(m, l, M);
        L = fmaf(f, l, L);
        acc = fmaf(f, s_part[z * share + e], acc);
      }
      out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + col] = from_f32<T>(acc * a8_inverse(L));
    }
    return;
  }
  // ---- the block that ends last among the parts joins them; nobody waits
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.counters + pair, 1) == splits - 1;
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) p.counters[pair] = 0;                        // ready for the next layer
  __threadfence();
  const size_t at0 = (size_t)(blockIdx.x - split) * group;   // the parts of a (token, kv head) lie side by side
  for (int e = tid; e < group * D; e += WARPS * 32) {
    const int row = e / D, col = e % D;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + at0 + row;
    const float* acc_of = p.part_acc + (at0 + row) * D + col;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int z0 = 0; z0 < splits; z0 += 8) {                 // eight parts are asked for at once
      float2 part[8];
      float a[8], top = M;
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        part[z] = z0 + z < splits ? __ldcg(ml + (size_t)(z0 + z) * group) : make_float2(-INFINITY, 0.f);
        a[z] = z0 + z < splits ? __ldcg(acc_of + (size_t)(z0 + z) * group * D) : 0.f;
        top = fmaxf(top, part[z].x);
      }
      const float before = a8_weight(M, L, top);
      M = top;
      L *= before;
      acc *= before;
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        const float f = a8_weight(part[z].x, part[z].y, top);
        if (part[z].y == 0.f) continue;
        L = fmaf(f, part[z].y, L);
        acc = fmaf(f, a[z], acc);
      }
    }
    out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + col] = from_f32<T>(acc * a8_inverse(L));
  }
}

// Portions: a warp has rows of its own, the heads of the group for as many neighbouring tokens as fit 8 NT rows; the block's warps have
// neighbouring ones and read the same keys out of one ring of slots, a turn's kA8Turn blocks each.  For float32, and for bfloat16 where
// the fifth-generation tensor cores do not pay (CudaOps._attention8_tensor_cores has the figures); mma.sync bounds it: a prompt of 2,048 tokens
// takes 133 us here and 50 there.  The warps take turns at fetching: turn i's
// one refills the slot that turn i - kLag left, which the others are through with by then (but for the slowest, which it waits for).
template <int D, typename T> struct A8Portion {
  static constexpr int kTiles = D == 64 ? (sizeof(T) == 2 ? 4 : 2) : 2;
  static constexpr int kRing = 6, kLag = 2;
  static constexpr int kSlot = kA8Turn * 2 * kKv8Block * D;
  static constexpr int kSmem = kRing * kSlot;
};

template <int D, typename T>
__global__ void __launch_bounds__(kA8Warps * 32)
attention8_portion_kernel(const A8Params p) {
  using Cfg = A8Portion<D, T>;
  constexpr int NT = Cfg::kTiles, kRing = Cfg::kRing, kLag = Cfg::kLag;
  static_assert(32 % kA8Turn == 0 && kRing * kA8Turn <= 32, "pages are looked up for 32 blocks at a time, and the 32 after them");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t s_full[kRing], s_empty[kRing];
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t full0 = smem_addr(s_full), empty0 = smem_addr(s_empty);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) { mbar_init(full0 + 8 * i, 1); mbar_init(empty0 + 8 * i, kA8Warps); }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int group = p.nq / p.nkv, per_warp = 8 * NT / group, per_block = per_warp * kA8Warps;      // tokens
  const int kvh = blockIdx.x % p.nkv;
  const int* tl = p.items + 4 * (gridDim.y - 1 - blockIdx.y);   // the last rows of a portion see the most keys: first
  const int sub = gridDim.x / p.nkv - 1 - blockIdx.x / p.nkv;
  const int tokens = min(per_block, tl[2] - sub * per_block);
  if (tokens <= 0) return;
  const int t0 = tl[1] + sub * per_block, pos0 = tl[3] + sub * per_block;
  const int lo = p.window > 0 && pos0 + 1 > p.window ? pos0 + 1 - p.window : 0;
  const int begin0 = lo / kKv8Block, all = (pos0 + tokens - 1) / kKv8Block + 1 - begin0;
  const int per_split = ((all + p.splits - 1) / p.splits + kA8Turn - 1) / kA8Turn * kA8Turn;
  const int begin = begin0 + min(all, (int)blockIdx.z * per_split), end = begin0 + min(all, ((int)blockIdx.z + 1) * per_split);
  const int turns = (end - begin + kA8Turn - 1) / kA8Turn;
  const int* table = p.block_table + (size_t)tl[0] * p.bt_stride;
  auto page_at = [&](int i) { return begin + i < end ? p.page_of(table, begin + i) : -1; };      // of the block's i-th block of keys
  auto word_at = [&](int i, int page) { return page >= 0 ? p.word(page, kvh, p.sub_of(begin + i)) : make_uint2(0u, 0u); };
  // lanes 0 .. kA8Turn - 1 fetch the turn's blocks, whose pages they are given
  auto fetch = [&](int turn, int page) {
    const int s = turn % kRing;
    const uint32_t bar = full0 + 8 * s;
    const unsigned got = __ballot_sync(0xffffffffu, lane < kA8Turn && page >= 0);
    if (lane == 0) mbar_expect_tx(bar, __popc(got) * 2 * kKv8Block * D);
    __syncwarp();
    if (lane < kA8Turn && page >= 0) {
      const unsigned char* src = p.keys<D>(page, kvh, p.sub_of(begin + turn * kA8Turn + lane));
      const uint32_t dst = smem_addr(smem) + s * Cfg::kSlot + lane * 2 * kKv8Block * D;
      bulk_load(dst, src, kKv8Block * D, bar);
      bulk_load(dst + kKv8Block * D, src + p.plane<D>(), kKv8Block * D, bar);
    }
    __syncwarp();
  };
  const int my_tokens = max(0, min(per_warp, tokens - warp * per_warp));
  const int my_t0 = t0 + warp * per_warp, my_pos0 = pos0 + warp * per_warp, my_last = my_pos0 + my_tokens - 1;
  const int my_lo = p.window > 0 && my_pos0 + 1 > p.window ? my_pos0 + 1 - p.window : 0;
  const int all_first = p.window > 0 && my_last + 1 > p.window ? my_last + 1 - p.window : 0;
  int page_cur = page_at(lane), page_nxt = page_at(32 + lane);
  A8Rows<D, T, NT> rows;
  {
    typename A8Rows<D, T, NT>::Raw raw;
    rows.fetch(raw, p, my_t0, my_tokens, kvh, group);
    for (int i = 0; i < min(kRing - kLag, turns); ++i) {
      const int page = __shfl_sync(0xffffffffu, page_cur, (i * kA8Turn + lane) & 31);
      if (i % kA8Warps == warp) fetch(i, page);
    }
    rows.load(raw, p, my_tokens, my_pos0, group);
  }
  uint2 word_cur = word_at(lane, page_cur), word_nxt = word_at(32 + lane, page_nxt);
  int page_nn = page_at(64 + lane);
  for (int i = 0; i < turns; ++i) {
    const int at = i * kA8Turn % 32;
    if (at == 0 && i > 0) {
      page_cur = page_nxt; word_cur = word_nxt; page_nxt = page_nn;
      word_nxt = word_at(i * kA8Turn + 32 + lane, page_nxt);
      page_nn = page_at(i * kA8Turn + 64 + lane);
    }
    bool ok = true;
    const int next = i + kRing - kLag;                        // the turn that takes the slot of turn i - kLag
    if (next < turns) {
      const int ahead = at + (kRing - kLag) * kA8Turn + lane;
      const int near = __shfl_sync(0xffffffffu, page_cur, ahead & 31), far = __shfl_sync(0xffffffffu, page_nxt, ahead & 31);
      if (next % kA8Warps == warp) {
        ok = i < kLag || __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * (next % kRing), ((next / kRing) & 1) ^ 1, &s_abort, p.status, 9));
        if (ok) fetch(next, ahead < 32 ? near : far);
      }
    }
    const int s = i % kRing, first_key = (begin + i * kA8Turn) * kKv8Block;
    if (!ok || !__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (i / kRing) & 1, &s_abort, p.status, 9))) {
      for (int k = i; k < min(i + kRing, turns); ++k) mbar_drain(full0 + 8 * (k % kRing), (k / kRing) & 1);      // (copies that are under way)
      return;
    }
    if (my_tokens > 0 && first_key <= my_last && first_key + kA8Turn * kKv8Block > my_lo) {
      const unsigned char* slot[kA8Turn];
      bool have[kA8Turn];
      uint2 word[kA8Turn];
      int key0[kA8Turn];
#pragma unroll
      for (int b = 0; b < kA8Turn; ++b) {
        slot[b] = smem + s * Cfg::kSlot + b * 2 * kKv8Block * D;
        have[b] = __shfl_sync(0xffffffffu, page_cur, at + b) >= 0;
        word[b].x = __shfl_sync(0xffffffffu, word_cur.x, at + b);
        word[b].y = __shfl_sync(0xffffffffu, word_cur.y, at + b);
        key0[b] = first_key + b * kKv8Block;
      }
      rows.turn(slot, have, word, key0, all_first, my_pos0);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty0 + 8 * s);
  }
  rows.finish();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * c + j;
      if (row >= my_tokens * group) continue;
      if (p.splits > 1) {
        const size_t at = ((size_t)(my_t0 + row / group) * p.nq + kvh * group + row % group) * p.splits + blockIdx.z;
#pragma unroll
        for (int i = 0; i < D / 8; i += 4)
          *reinterpret_cast<float4*>(p.part_acc + at * D + g * (D / 8) + i) =
              make_float4(rows.entry(n, j, i), rows.entry(n, j, i + 1), rows.entry(n, j, i + 2), rows.entry(n, j, i + 3));
        if (g == 0) { p.part_ml[2 * at] = rows.m[n][j]; p.part_ml[2 * at + 1] = rows.l[n][j]; }
        continue;
      }
      const float inv = a8_inverse(rows.l[n][j]);
      T* dst = static_cast<T*>(p.out) + (size_t)(my_t0 + row / group) * p.out_stride + (size_t)(kvh * group + row % group) * D + g * (D / 8);
#pragma unroll
      for (int i = 0; i < D / 8; i += Vec16<T>::N) {
        Vec16<T> v;
#pragma unroll
        for (int x = 0; x < Vec16<T>::N; ++x) v.set(x, rows.entry(n, j, i + x) * inv);
        store16(dst + i, v);
      }
    }
}

// The splits of portions joined: D / 4 lanes a row of the tiles and query head, four dimensions each.
constexpr int kA8JoinThreads = 256;
template <int D, typename T>
__global__ void __launch_bounds__(kA8JoinThreads)
attention8_join_kernel(const A8Params p) {
  const int* tl = p.items + 4 * blockIdx.y;
  const int first = __ldg(tl + 1), rows = __ldg(tl + 2);       // (the kernels before this one have waited for whoever wrote them)
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x * (kA8JoinThreads / (D / 4)) + threadIdx.x / (D / 4), col = threadIdx.x % (D / 4) * 4;
  if (i / p.nq >= rows) return;
  const size_t row = (size_t)(first + i / p.nq), at = (row * p.nq + i % p.nq) * p.splits;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + at;
  const float4* part = reinterpret_cast<const float4*>(p.part_acc + at * D + col);
  constexpr int kAhead = 4;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int z0 = 0; z0 < p.splits; z0 += kAhead) {              // kAhead parts are asked for at once; those without keys hold nothing
    float2 s[kAhead];
    float4 a[kAhead];
    float top = M;
#pragma unroll
    for (int z = 0; z < kAhead; ++z) {
      s[z] = z0 + z < p.splits ? __ldg(ml + z0 + z) : make_float2(-INFINITY, 0.f);
      a[z] = z0 + z < p.splits ? __ldg(part + (size_t)(z0 + z) * (D / 4)) : acc;
      top = fmaxf(top, s[z].x);
    }
    const float before = a8_weight(M, L, top);
    M = top;
    L *= before;
    acc.x *= before; acc.y *= before; acc.z *= before; acc.w *= before;
#pragma unroll
    for (int z = 0; z < kAhead; ++z) {
      if (s[z].y == 0.f) continue;
      const float f = a8_weight(s[z].x, s[z].y, top);
      L = fmaf(f, s[z].y, L);
      acc.x = fmaf(f, a[z].x, acc.x); acc.y = fmaf(f, a[z].y, acc.y); acc.z = fmaf(f, a[z].z, acc.z); acc.w = fmaf(f, a[z].w, acc.w);
    }
  }
  const float inv = a8_inverse(L);
  T* dst = static_cast<T*>(p.out) + row * p.out_stride + (size_t)(i % p.nq) * D + col;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
}
template <int D, typename T> static int launch_a8_join(const A8Params& p, int tiles, cudaStream_t stream) {
  constexpr int kPer = kA8JoinThreads / (D / 4);
  return launch_kernel("attention8_join", attention8_join_kernel<D, T>, dim3((128 * p.nq + kPer - 1) / kPer, tiles), dim3(kA8JoinThreads), 0, stream, p);
}

int attention8_join_bf16(void* out, const float* part_acc, const float* part_ml, const int* tiles, int n_tiles, int out_stride, int nq, int d, int splits,
                         void* stream) {
  A8Params p{};
  p.out = out; p.part_acc = const_cast<float*>(part_acc); p.part_ml = const_cast<float*>(part_ml); p.items = tiles;
  p.out_stride = out_stride; p.nq = nq; p.splits = splits;
  return d == 64 ? launch_a8_join<64, __nv_bfloat16>(p, n_tiles, as_stream(stream)) : launch_a8_join<128, __nv_bfloat16>(p, n_tiles, as_stream(stream));
}

// The units that a step's single tokens are dealt out in: see decode_units_kernel (attention_decode.cu), whose list this is.  c is
// ceil(tiles / (units - tokens)), which always suffices, and not the smallest that does: no search, three barriers in all; and the counters
// that the parts join by are set to zero.  Tiles are 64 keys.  5.6 us by the search (64 tokens), 3 so.
constexpr int kA8PlanItems = 1024;
__global__ void __launch_bounds__(kA8PlanItems)
attention8_units_kernel(int4* __restrict__ units, const int* __restrict__ items, const int* __restrict__ tok_req, const int* __restrict__ positions,
                        int n_items, int nkv, int window, int per_head, int* __restrict__ counters, int n_counters) {
  __shared__ int s_t[kA8PlanItems], s_r[kA8PlanItems], s_p[kA8PlanItems], s_first[kA8PlanItems + 1], s_sum[32], s_units[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  int t = -1, r = -1, p = -1, tiles = 0;
  if (tid < n_items) {
    t = items ? __ldg(items + tid) : tid;
    r = __ldg(tok_req + t);
    p = __ldg(positions + t);
    const int keys = window > 0 && p + 1 > window ? window : p + 1;
    tiles = r < 0 ? 0 : max(1, (keys + 63) / 64);
  }
  for (int i = tid; i < n_counters; i += kA8PlanItems) counters[i] = 0;
  s_t[tid] = t; s_r[tid] = r; s_p[tid] = p;
  const int sum = __reduce_add_sync(0xffffffffu, tiles);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  const int total = __reduce_add_sync(0xffffffffu, s_sum[lane]);
  const int c = max(1, per_head > n_items ? (total + per_head - n_items - 1) / (per_head - n_items) : total);
  const int mine = (tiles + c - 1) / c;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += below;
  }
  if (lane == 31) s_units[warp] = incl;
  __syncthreads();
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_units[lane] : 0);
  s_first[tid] = before + incl - mine;                       // units of the tokens before, per kv head
  if (tid == kA8PlanItems - 1) s_first[kA8PlanItems] = before + incl;
  __syncthreads();
  const int units_per_head = s_first[kA8PlanItems];
  for (int u = tid; u < nkv * per_head; u += kA8PlanItems) {
    int4 a = make_int4(-1, -1, -1, 0), b = make_int4(0, 1, -1, 0);
    if (u / nkv < units_per_head) {
      int i = 0;                                             // the last token that begins at or before this unit
#pragma unroll
      for (int half = kA8PlanItems / 2; half; half >>= 1)
        if (s_first[i + half] <= u / nkv) i += half;
      const int n = s_first[i + 1] - s_first[i], at = u - s_first[i] * nkv;
      a = make_int4(s_t[i], s_r[i], s_p[i], at / n);
      b.x = at % n;
      b.y = n;
    }
    if (u < n_items * nkv && s_r[u / nkv] < 0) { b.z = s_t[u / nkv]; b.w = u % nkv; }
    units[2 * u] = a;
    units[2 * u + 1] = b;
  }
}

template <int D, typename T, int NT, int WARPS>
static int launch_single(const A8Params& p, unsigned blocks, cudaStream_t stream) {
  using Cfg = A8Single<D, NT, WARPS>;
  static SmemRaised raised = {};
  constexpr int kMost = Cfg::kSmem + Cfg::kPartBytes;
  if (int rc = raise_shared_memory("attention8_single", attention8_single_kernel<D, T, NT, WARPS>, kMost, raised)) return rc;
  const int share = (p.nq / p.nkv * D + p.splits - 1) / p.splits;
  return launch_kernel_cluster("attention8_single", attention8_single_kernel<D, T, NT, WARPS>, dim3(blocks), dim3(WARPS * 32),
                               Cfg::kSmem + (p.cluster ? share * p.splits * 12 : 0), stream, p.cluster ? p.splits : 1, p);
}

template <int D, typename T>
static int launch_attention8(const A8Params& p, int singles, int tiles, int per_head, int warps, cudaStream_t stream) {
  const int group = p.nq / p.nkv;
  if (singles) {
    const long long blocks = per_head ? (long long)p.nkv * per_head : (long long)singles * p.nkv * p.splits;
    PTL_REQUIRE(blocks <= 0x7fffffffLL, "attention8: too many blocks");
    if (group > 8) return launch_single<D, T, 2, 4>(p, (unsigned)blocks, stream);
    return warps == 8 ? launch_single<D, T, 1, 8>(p, (unsigned)blocks, stream) : launch_single<D, T, 1, 4>(p, (unsigned)blocks, stream);
  }
  using Cfg = A8Portion<D, T>;
  static SmemRaised raised = {};
  if (int rc = raise_shared_memory("attention8_portion", attention8_portion_kernel<D, T>, Cfg::kSmem, raised)) return rc;
  const int per_block = 8 * Cfg::kTiles / group * kA8Warps;
  if (int rc = launch_kernel("attention8_portion", attention8_portion_kernel<D, T>, dim3(p.nkv * ((128 + per_block - 1) / per_block), tiles, p.splits),
                             dim3(kA8Warps * 32), Cfg::kSmem, stream, p)) return rc;
  if (p.splits == 1) return 0;
  return launch_a8_join<D, T>(p, tiles, stream);
}

template <typename T>
static int attention8_mma(A8Params p, int singles, int tiles, int d, int page_size, int per_head, int warps, void* stream) {
  PTL_REQUIRE(p.nq > 0 && p.nkv > 0 && page_size > 0 && p.num_pages > 0 && p.bt_stride > 0 && singles >= 0 && tiles >= 0, "attention8: bad sizes");
  PTL_REQUIRE(p.nq % p.nkv == 0, "attention8: %d query heads are no multiple of %d kv heads", p.nq, p.nkv);
  PTL_REQUIRE(page_size % kKv8Block == 0, "attention8: pages of %d positions are not whole blocks of %d", page_size, kKv8Block);
  if ((d != 64 && d != 128) || p.nq / p.nkv > 16 || tiles > 65535 || p.q_stride % 8 || p.out_stride % 8) return -2;
  PTL_REQUIRE(aligned16(p.q) && aligned16(p.out) && aligned16(p.codes) && (reinterpret_cast<uintptr_t>(p.words) & 7u) == 0,
              "attention8: q, out and codes must be 16-byte and words 8-byte aligned");
  PTL_REQUIRE(p.splits >= 1 && (!p.cluster || p.splits <= 8) && p.splits <= 65535, "attention8: a cluster has up to 8 parts");
  PTL_REQUIRE(tiles == 0 || p.splits == 1 || (p.part_acc && p.part_ml), "attention8: splits > 1 need scratch buffers");
  PTL_REQUIRE(per_head == 0 || (p.units && aligned16(p.units) && p.counters && p.part_acc && p.part_ml), "attention8: units need their list and scratch");
  PTL_REQUIRE(p.status != nullptr, "attention8: needs a status word");
  p.blocks_per_page = page_size / kKv8Block;
  p.page_shift = -1;
  for (int b = 0; b < 20; ++b) if ((1 << b) == p.blocks_per_page) p.page_shift = b;
  if (singles == 0 && tiles == 0) return 0;
  return d == 64 ? launch_attention8<64, T>(p, singles, tiles, per_head, warps, as_stream(stream))
                 : launch_attention8<128, T>(p, singles, tiles, per_head, warps, as_stream(stream));
}

}  // namespace ptl

// The arguments of both entries, packed by the caller: the host converts 28 of a call's own in 2.9 us, and packs them in 0.4.
struct A8Args {
  void* out;
  float *part_acc, *part_ml;
  const void *q, *codes, *words;
  const int *block_table, *items, *tok_req, *positions, *units;
  int *counters, *status;
  void* stream;
  int n_items, q_stride, out_stride, bt_stride, nq, nkv, d, page_size, window, splits, warps, per_head, num_pages;
  float scale;
};
static_assert(sizeof(A8Args) == 14 * 8 + 14 * 4, "as it is packed");

template <typename T> static int attention8_entry(const void* args, bool single) {
  A8Args a;
  memcpy(&a, args, sizeof a);
  ptl::A8Params p{a.out, a.part_acc, a.part_ml, a.counters, a.q, (const unsigned char*)a.codes, (const uint32_t*)a.words, a.block_table, a.items,
                  a.tok_req, a.positions, (const int4*)a.units, a.status, a.q_stride, a.out_stride, a.bt_stride, a.nq, a.nkv, 0, 0, a.num_pages, a.window,
                  a.splits, single && a.per_head == 0 && a.splits > 1, a.scale * 1.4426950408889634f};
  return single ? ptl::attention8_mma<T>(p, a.n_items, 0, a.d, a.page_size, a.per_head, a.warps, a.stream)
                : ptl::attention8_mma<T>(p, 0, a.n_items, a.d, a.page_size, 0, 4, a.stream);
}

// Single tokens: `items` their rows (null: 0..n_items-1).  With per_head > 0 the keys are dealt out in units (`units` from
// ptl_attention8_units with the same sizes and with `counters`, one int per (row, kv head) of q), part_acc [nkv * per_head, nq / nkv, d] and part_ml
// [..., 2]; else every (token, kv head) has `splits` parts, up to 8, which join in a cluster.  `warps` of a block: 4 or 8.  -2: sizes this kernel does not take.
// *status: raised when a wait for a copy gave up.
// Portions: `items` their tiles; with splits > 1 part_acc [rows of q, nq, splits, d] and part_ml [rows of q, nq, splits, 2], float32.
PTL_EXPORT int ptl_attention8_single_f32(const void* args) { return attention8_entry<float>(args, true); }
PTL_EXPORT int ptl_attention8_single_bf16(const void* args) { return attention8_entry<__nv_bfloat16>(args, true); }
PTL_EXPORT int ptl_attention8_portion_f32(const void* args) { return attention8_entry<float>(args, false); }
PTL_EXPORT int ptl_attention8_portion_bf16(const void* args) { return attention8_entry<__nv_bfloat16>(args, false); }

// units: 8 ints for each of nkv * per_head blocks, per_head at least n_items; counters: n_counters ints, set to zero.  -2: more tokens than one block lays out.
PTL_EXPORT int ptl_attention8_units(int* units, int* counters, int n_counters, const int* items, const int* tok_req, const int* positions, int n_items,
                                    int nkv, int window, int per_head, void* stream) {
  using namespace ptl;
  if (n_items > kA8PlanItems) return -2;
  PTL_REQUIRE(n_items > 0 && nkv > 0 && per_head >= n_items && (long long)nkv * per_head <= (1 << 24) && units && aligned16(units) && counters && n_counters >= 0,
              "attention8_units: bad sizes");
  return launch_kernel("attention8_units", attention8_units_kernel, dim3(1), dim3(kA8PlanItems), 0, as_stream(stream), (int4*)units, items, tok_req,
                       positions, n_items, nkv, window, per_head, counters, n_counters);
}
