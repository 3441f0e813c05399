// Attention over an 8-bit cache (kv8.cuh) with mma.sync tensor products: head sizes 64 and 128, up to 16 query heads a kv head.
//
// A code u counts u - 128 = c steps and a half, and c is a half float exactly, so with a query row q = 2^e x, |x| < 2,
//   q . k = s_k 2^e (x . c + sum(x) / 2),        sum_j p_j v_j = sum over blocks of s_v (sum p_j c_j + sum p_j / 2):
// the two products run on half floats with float32 sums, a block's step is a float32 factor of its 16 keys' scores and of its 16
// keys' part of the output, and the halves cost one float32 sum a row.  x is a half float exactly for bfloat16 q (but for entries
// below 2^-14 of the row's largest, which lose bits below 2^-24 of it); weights p <= 1 are rounded to half floats, 2^-11 of each.
// float32 rows take two half floats each, x = x1 + x2 and p = p1 + p2, and twice the products.
//
// No shared memory on the way in.  For m16n8k16 the 16 dimensions of a step and the 8 columns of a value product may be any, as long
// as both operands agree, so they are chosen for the loads: lane (g, c) reads 16 bytes of key g's row at 16 c, which are its operand
// of four steps, and D / 8 bytes of value rows 2c, 2c + 1, 2c + 8, 2c + 9 at g D / 8, which are its operand of D / 8 products.  A
// byte becomes half float 1024 + u by one byte permutation, and 1024 + u - 1152 = c exactly.  A warp asks for the next keys as soon as
// it has multiplied this turn's, and for the next values likewise, so loads run under the other half of the turn.
//
// Rows of a tile: the heads of the group for one token, or for as many tokens of a portion as fit 16 rows.  Two ways of sharing:
// - single tokens (SINGLE): the four warps of a block take turns through the keys of one (token, kv head), or of a part of them, and
//   join through shared memory.  Parts of one (token, kv head) join in a cluster, or, where the contexts are cut into parts of equal
//   length (the list of decode_units_kernel), in the block that ends last.
// - portions: a warp has a tile of its own; the block's warps have neighbouring ones, which read the same keys out of L1.
#include "kv8.cuh"
#include "mma_utils.cuh"

namespace ptl {

constexpr int kA8Warps = 4;

struct A8Params {
  void* out;
  float* part_acc;            // [blocks][G][D]
  float* part_ml;             // [blocks][G][2], in units of log2
  int* counters;              // a zero per (item, kv head)
  const void* q;
  const unsigned char* codes;
  const uint32_t* words;
  const int* block_table;
  const int* items;           // singles: token rows, null for 0..; portions: tiles {request, first row, rows, first position}
  const int* tok_req;
  const int* positions;
  const int4* units;
  int q_stride, out_stride, bt_stride, nq, nkv, blocks_per_page, page_shift, num_pages, window, splits, cluster;
  float scale_log2;
};

__device__ __forceinline__ float a8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes `sel` picks, two of them, as half floats u - 128.
__device__ __forceinline__ uint32_t a8_pair(uint32_t bytes, uint32_t sel) {
  uint32_t x, y;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(x) : "r"(bytes), "r"(0x64646464u), "r"(sel));      // 1024 + u
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
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
template <int BYTES> __device__ __forceinline__ void a8_load(uint32_t (&r)[BYTES / 4], const unsigned char* p) {
  if constexpr (BYTES == 16) {
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
  } else {
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  }
}
__device__ __forceinline__ float ld_peer_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Rows per warp: 16 (WIDE) or 8, the upper half of the product's rows then being zeros.
template <int D, typename T, bool WIDE> struct A8Warp {
  static constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr int kHalves = WIDE ? 2 : 1;
  static constexpr int kChunks = D / 64;                     // 16-byte pieces of a key row a lane takes
  static constexpr int kTurn = D == 64 ? 2 : 1;              // blocks of 16 keys a turn
  static constexpr int kTiles = D / 8;                       // value products
  uint32_t qa[kParts][kChunks * 4][2 * kHalves];
  float half_sum[kHalves];                                   // sum(x) / 2
  float factor[kHalves];                                     // 2^e scale log2(e)
  int first[kHalves], last[kHalves];                         // positions a row sees
  float o[kTiles][2 * kHalves];
  float m[kHalves], l[kHalves], w[kHalves];

  // Row `row` of the tile is query head head0 + row % group of token t0 + row / group.
  __device__ __forceinline__ void load_rows(const A8Params& p, int t0, int tokens, int pos0, int kvh, int group) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const bool here = row < tokens * group;
      const int token = here ? row / group : 0;
      float x[kChunks][16];
      const T* src = static_cast<const T*>(p.q) + (size_t)(t0 + token) * p.q_stride + (size_t)(kvh * group + (here ? row % group : 0)) * D + 16 * c;
      float big = 0.f;
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int i = 0; i < 16; i += Vec16<T>::N) {
          Vec16<T> v;
          if (here) v = load16(src + 64 * k + i);
#pragma unroll
          for (int j = 0; j < Vec16<T>::N; ++j) {
            x[k][i + j] = here ? v.get(j) : 0.f;
            big = fmaxf(big, fabsf(x[k][i + j]));
          }
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // 2^e with |x| < 2; the powers of two that 1 / 2^e can be
      const uint32_t e = min(max(__float_as_uint(big) >> 23, 2u), 252u);
      const float scale = __uint_as_float(e << 23), inverse = __uint_as_float((254u - e) << 23);
      factor[h] = scale * p.scale_log2;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float a = x[k][4 * i + 2 * j] * inverse, b = x[k][4 * i + 2 * j + 1] * inverse;
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint32_t half = a8_pack(a, b);
              float fa, fb;
              a8_unpack(half, fa, fb);
              sum += fa + fb;
              qa[part][4 * k + i][j * kHalves + h] = half;
              a -= fa; b -= fb;
            }
          }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      half_sum[h] = 0.5f * sum;
      last[h] = here ? pos0 + token : -1;
      first[h] = p.window > 0 && last[h] + 1 > p.window ? last[h] + 1 - p.window : 0;
      m[h] = -INFINITY; l[h] = 0.f; w[h] = 0.f;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) { o[n][2 * h] = 0.f; o[n][2 * h + 1] = 0.f; }
    }
  }

  // Blocks begin, begin + stride, ... of kTurn blocks of 16 positions each, below `end`, of request r.  Rows with every position of
  // [all_first, all_last] in sight are not masked there.
  __device__ __forceinline__ void walk(const A8Params& p, int r, int kvh, int begin, int stride, int end, int all_first, int all_last) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int page_size = p.blocks_per_page * kKv8Block;
    const size_t plane = (size_t)p.nkv * page_size * D;
    const int* table = p.block_table + (size_t)r * p.bt_stride;
    const unsigned char* at[kTurn];
    uint2 word[kTurn], word_next[kTurn];
    bool have[kTurn], have_next[kTurn];
    uint32_t k[kTurn][2][kChunks][4], v[kTurn][4][D / 32];
    int page[kTurn];
    auto look_up = [&](int i) {
#pragma unroll
      for (int b = 0; b < kTurn; ++b) {
        const int blk = i + b, pg = p.page_shift >= 0 ? blk >> p.page_shift : blk / p.blocks_per_page;
        page[b] = blk < end && pg < p.bt_stride ? __ldg(table + pg) : -1;
      }
    };
    auto load_keys = [&](int i) {
#pragma unroll
      for (int b = 0; b < kTurn; ++b) {
        const int blk = i + b, sub = p.page_shift >= 0 ? blk & ((1 << p.page_shift) - 1) : blk % p.blocks_per_page;
        have_next[b] = page[b] >= 0 && page[b] < p.num_pages;
        if (!have_next[b]) { word_next[b] = make_uint2(0u, 0u); continue; }
        at[b] = p.codes + (size_t)page[b] * 2 * plane + ((size_t)kvh * page_size + sub * kKv8Block) * D;
        word_next[b] = __ldg(reinterpret_cast<const uint2*>(p.words + (((size_t)page[b] * p.nkv + kvh) * p.blocks_per_page + sub) * 2));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < kChunks; ++h) a8_load<16>(k[b][n][h], at[b] + (n * 8 + g) * D + h * 64 + 16 * c);
      }
    };
    auto load_values = [&]() {
#pragma unroll
      for (int b = 0; b < kTurn; ++b)
        if (have[b]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) a8_load<D / 8>(v[b][j], at[b] + plane + ((j >> 1) * 8 + 2 * c + (j & 1)) * D + g * (D / 8));
        }
    };
    look_up(begin);
    load_keys(begin);
#pragma unroll
    for (int b = 0; b < kTurn; ++b) { word[b] = word_next[b]; have[b] = have_next[b]; }
    load_values();
    look_up(begin + stride);
    for (int i = begin; i < end; i += stride) {
      float s[kTurn][2][2 * kHalves];
#pragma unroll
      for (int b = 0; b < kTurn; ++b) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float acc[4] = {half_sum[0], half_sum[0], half_sum[kHalves - 1], half_sum[kHalves - 1]};
          if (have[b]) {
#pragma unroll
            for (int h = 0; h < kChunks; ++h)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint32_t b0 = a8_pair(k[b][n][h][x], 0x4140u), b1 = a8_pair(k[b][n][h][x], 0x4342u);
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                  const uint32_t(&a)[2 * kHalves] = qa[part][4 * h + x];
                  mma_f16_16816(acc, a[0], WIDE ? a[kHalves - 1] : 0u, a[kHalves], WIDE ? a[2 * kHalves - 1] : 0u, b0, b1);
                }
              }
          }
          const float step = 2.0f * kv8_half_step(word[b].x & 255u);
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            s[b][n][2 * h] = acc[2 * h] * (factor[h] * step);
            s[b][n][2 * h + 1] = acc[2 * h + 1] * (factor[h] * step);
          }
        }
        const int key0 = (i + b) * kKv8Block;
        if (key0 < all_first || key0 + kKv8Block - 1 > all_last || !have[b] || ((word[b].x | word[b].y) >> 16)) {
          const uint32_t marks = (word[b].x | word[b].y) >> 16;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2 * kHalves; ++e) {
              const int off = n * 8 + 2 * c + (e & 1), key = key0 + off;
              if ((marks >> off) & 1u) s[b][n][e] = __uint_as_float(0x7fc00000u);
              if (key < first[e >> 1] || key > last[e >> 1] || !have[b]) s[b][n][e] = -INFINITY;
            }
        }
      }
      // this turn's keys are used: the next ones
      float vstep[kTurn];
      bool held[kTurn];
#pragma unroll
      for (int b = 0; b < kTurn; ++b) { vstep[b] = 2.0f * kv8_half_step(word[b].y & 255u); held[b] = have[b]; }
      if (i + stride < end) {
        load_keys(i + stride);
        look_up(i + 2 * stride);
      }
      uint32_t pa[kParts][kTurn][2][kHalves];
      bool moved = false;
      float alpha[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        float mx = m[h];
#pragma unroll
        for (int b = 0; b < kTurn; ++b)
          mx = fmaxf(mx, fmaxf(fmaxf(s[b][0][2 * h], s[b][0][2 * h + 1]), fmaxf(s[b][1][2 * h], s[b][1][2 * h + 1])));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float use = mx == -INFINITY ? 0.f : mx;
        alpha[h] = a8_exp2(m[h] - use);
        moved |= mx > m[h];
        m[h] = mx;
        float sum = 0.f, wsum = 0.f;
#pragma unroll
        for (int b = 0; b < kTurn; ++b) {
          float pr[2][2], part_sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            pr[n][0] = a8_exp2(s[b][n][2 * h] - use);
            pr[n][1] = a8_exp2(s[b][n][2 * h + 1] - use);
            part_sum += pr[n][0] + pr[n][1];
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint32_t half = a8_pack(pr[n][0], pr[n][1]);
              pa[part][b][n][h] = half;
              if (part + 1 < kParts) {
                float fa, fb;
                a8_unpack(half, fa, fb);
                pr[n][0] -= fa; pr[n][1] -= fb;
              }
            }
          }
          sum += part_sum;
          wsum = fmaf(part_sum, vstep[b], wsum);
        }
        l[h] = fmaf(l[h], alpha[h], sum);
        w[h] = fmaf(w[h], alpha[h], wsum);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 2 * kHalves; ++e) o[n][e] *= alpha[e >> 1];
      }
#pragma unroll
      for (int b = 0; b < kTurn; ++b) {
        if (!held[b]) continue;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          // four bytes of each of four value rows -> the operands of four products
          uint32_t lo[2], hi[2];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(lo[n]) : "r"(v[b][2 * n][x]), "r"(v[b][2 * n + 1][x]), "r"(0x5140u));
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(hi[n]) : "r"(v[b][2 * n][x]), "r"(v[b][2 * n + 1][x]), "r"(0x7362u));
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t sel = y & 1 ? 0x4342u : 0x4140u;
            const uint32_t b0 = a8_pair(y < 2 ? lo[0] : hi[0], sel), b1 = a8_pair(y < 2 ? lo[1] : hi[1], sel);
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              mma_f16_16816(acc, pa[part][b][0][0], WIDE ? pa[part][b][0][kHalves - 1] : 0u, pa[part][b][1][0],
                            WIDE ? pa[part][b][1][kHalves - 1] : 0u, b0, b1);
#pragma unroll
            for (int e = 0; e < 2 * kHalves; ++e) o[4 * x + y][e] = fmaf(acc[e], vstep[b], o[4 * x + y][e]);
          }
        }
      }
      if (i + stride < end) {
#pragma unroll
        for (int b = 0; b < kTurn; ++b) { word[b] = word_next[b]; have[b] = have_next[b]; }
        load_values();
      }
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
        w[h] += __shfl_xor_sync(0xffffffffu, w[h], x);
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) { o[n][2 * h] += 0.5f * w[h]; o[n][2 * h + 1] += 0.5f * w[h]; }
    }
  }
  // Lane (g, c) holds, of row g + 8 h, the dimensions c D / 4 + (0 .. D / 4 - 1): this is entry `i` of them.
  __device__ __forceinline__ float entry(int h, int i) const { return o[i % kTiles][2 * h + i / kTiles]; }
};

// What a row's weight sum l and a part's (m, l) give: parts without keys count nothing, a sum that is no number stays one.
__device__ __forceinline__ float a8_weight(float m, float l, float M) { return l == 0.f ? 0.f : a8_exp2(m - M); }
__device__ __forceinline__ float a8_inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }

template <int D, typename T, bool WIDE>
__global__ void __launch_bounds__(kA8Warps * 32, D == 64 && !WIDE ? 4 : 1)
attention8_single_kernel(const A8Params p) {
  using W = A8Warp<D, T, WIDE>;
  constexpr int kRows = WIDE ? 16 : 8;
  __shared__ float s_o[kA8Warps][kRows][D], s_m[kA8Warps][kRows], s_l[kA8Warps][kRows];
  __shared__ float s_part[kRows * D], s_pm[kRows], s_pl[kRows];
  __shared__ int s_last;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int group = p.nq / p.nkv;
  T* out = static_cast<T*>(p.out);
  int t, r, pos, kvh, split, splits, pair;
  if (p.units) {
    const int4 a = p.units[2 * blockIdx.x], b = p.units[2 * blockIdx.x + 1];
    t = a.x; r = a.y; pos = a.z; kvh = a.w; split = b.x; splits = b.y;
    if (b.z >= 0)                                            // a row without a request: zeros
      for (int e = tid; e < group * D; e += kA8Warps * 32) out[(size_t)b.z * p.out_stride + (size_t)b.w * group * D + e] = from_f32<T>(0.f);
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
        for (int e = tid; e < group * D; e += kA8Warps * 32) out[(size_t)t * p.out_stride + (size_t)kvh * group * D + e] = from_f32<T>(0.f);
      return;
    }
  }
  const int lo = p.window > 0 && pos + 1 > p.window ? pos + 1 - p.window : 0;
  const int b0 = lo / kKv8Block, blocks = pos < 0 ? 0 : pos / kKv8Block - b0 + 1;
  const int per = ((blocks + splits - 1) / splits + W::kTurn - 1) / W::kTurn * W::kTurn;
  const int begin = b0 + min(blocks, split * per), end = b0 + min(blocks, (split + 1) * per);
  W w;
  w.load_rows(p, t, 1, pos, kvh, group);
  w.walk(p, r, kvh, begin + warp * W::kTurn, kA8Warps * W::kTurn, end, lo, pos);
#pragma unroll
  for (int h = 0; h < W::kHalves; ++h) {
    const int row = g + 8 * h;
#pragma unroll
    for (int i = 0; i < D / 4; i += 4)
      *reinterpret_cast<float4*>(&s_o[warp][row][c * (D / 4) + i]) = make_float4(w.entry(h, i), w.entry(h, i + 1), w.entry(h, i + 2), w.entry(h, i + 3));
    if (c == 0) { s_m[warp][row] = w.m[h]; s_l[warp][row] = w.l[h]; }
  }
  __syncthreads();
  const bool whole = splits == 1;
  for (int e = tid; e < group * D; e += kA8Warps * 32) {
    const int row = e / D, col = e % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int i = 0; i < kA8Warps; ++i) M = fmaxf(M, s_m[i][row]);
#pragma unroll
    for (int i = 0; i < kA8Warps; ++i) {
      const float f = a8_weight(s_m[i][row], s_l[i][row], M);
      if (s_l[i][row] == 0.f) continue;
      L = fmaf(f, s_l[i][row], L);
      acc = fmaf(f, s_o[i][row][col], acc);
    }
    if (whole) {
      out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + col] = from_f32<T>(acc * a8_inverse(L));
    } else if (p.cluster) {
      s_part[e] = acc;
      if (col == 0) { s_pm[row] = M; s_pl[row] = L; }
    } else {
      const size_t at = (size_t)blockIdx.x * group + row;
      p.part_acc[at * D + col] = acc;
      if (col == 0) { p.part_ml[2 * at] = M; p.part_ml[2 * at + 1] = L; }
    }
  }
  if (whole) return;
  if (p.cluster) {
    // every block of the cluster finishes its share of the outputs from all of them
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const uint32_t at_o = smem_u32(s_part), at_m = smem_u32(s_pm), at_l = smem_u32(s_pl);
    const int share = (group * D + splits - 1) / splits;
    for (int e = split * share + tid; e < min(group * D, (split + 1) * share); e += kA8Warps * 32) {
      const int row = e / D;
      float M = -INFINITY, L = 0.f, acc = 0.f;
      float ms[8], ls[8], os[8];
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        if (z < splits) {
          ms[z] = ld_peer_f32(map_to_peer(at_m + 4 * row, z));
          ls[z] = ld_peer_f32(map_to_peer(at_l + 4 * row, z));
          os[z] = ld_peer_f32(map_to_peer(at_o + 4 * e, z));
          M = fmaxf(M, ms[z]);
        }
      }
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        if (z < splits && ls[z] != 0.f) {
          const float f = a8_weight(ms[z], ls[z], M);
          L = fmaf(f, ls[z], L);
          acc = fmaf(f, os[z], acc);
        }
      }
      out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + e % D] = from_f32<T>(acc * a8_inverse(L));
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();                                          // nobody leaves while a peer still reads
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
  for (int e = tid; e < group * D; e += kA8Warps * 32) {
    const int row = e / D, col = e % D;
    const float* ml = p.part_ml + 2 * (at0 + row);
    const float* acc_of = p.part_acc + (at0 + row) * D + col;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) M = fmaxf(M, __ldcg(ml + 2 * (size_t)z * group));
#pragma unroll 8
    for (int z = 0; z < splits; ++z) {
      const float mz = __ldcg(ml + 2 * (size_t)z * group), lz = __ldcg(ml + 2 * (size_t)z * group + 1), a = __ldcg(acc_of + (size_t)z * group * D);
      const float f = a8_weight(mz, lz, M);
      if (lz == 0.f) continue;
      L = fmaf(f, lz, L);
      acc = fmaf(f, a, acc);
    }
    out[(size_t)t * p.out_stride + (size_t)(kvh * group + row) * D + col] = from_f32<T>(acc * a8_inverse(L));
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kA8Warps * 32)
attention8_portion_kernel(const A8Params p) {
  using W = A8Warp<D, T, true>;
  pdl_wait();
  pdl_launch_dependents();
  const int group = p.nq / p.nkv, per_tile = 16 / group;      // tokens of a warp
  const int kvh = blockIdx.x % p.nkv;
  const int tile = gridDim.y - 1 - blockIdx.y;                // the last rows of a portion see the most keys: first
  const int* tl = p.items + 4 * tile;
  const int sub = (blockIdx.x / p.nkv) * kA8Warps + (threadIdx.x >> 5);
  const int begin = sub * per_tile, tokens = min(per_tile, tl[2] - begin);
  if (tokens <= 0) return;
  const int t0 = tl[1] + begin, pos0 = tl[3] + begin, last = pos0 + tokens - 1;
  const int lo = p.window > 0 && pos0 + 1 > p.window ? pos0 + 1 - p.window : 0;
  const int lo_last = p.window > 0 && last + 1 > p.window ? last + 1 - p.window : 0;
  W w;
  w.load_rows(p, t0, tokens, pos0, kvh, group);
  w.walk(p, tl[0], kvh, lo / kKv8Block, W::kTurn, last / kKv8Block + 1, lo_last, pos0);
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = g + 8 * h;
    if (row >= tokens * group) continue;
    const float inv = a8_inverse(w.l[h]);
    T* dst = static_cast<T*>(p.out) + (size_t)(t0 + row / group) * p.out_stride + (size_t)(kvh * group + row % group) * D + c * (D / 4);
#pragma unroll
    for (int i = 0; i < D / 4; i += Vec16<T>::N) {
      Vec16<T> v;
#pragma unroll
      for (int j = 0; j < Vec16<T>::N; ++j) v.set(j, w.entry(h, i + j) * inv);
      store16(dst + i, v);
    }
  }
}

template <int D, typename T>
static int launch_attention8(const A8Params& p, int singles, int tiles, int per_head, cudaStream_t stream) {
  const int group = p.nq / p.nkv;
  if (singles) {
    const long long blocks = per_head ? (long long)p.nkv * per_head : (long long)singles * p.nkv * p.splits;
    PTL_REQUIRE(blocks <= 0x7fffffffLL, "attention8: too many blocks");
    auto kernel = group <= 8 ? attention8_single_kernel<D, T, false> : attention8_single_kernel<D, T, true>;
    return launch_kernel_cluster("attention8_single", kernel, dim3((unsigned)blocks), dim3(kA8Warps * 32), 0, stream, p.cluster ? p.splits : 1, p);
  }
  const int per_tile = 16 / group, blocks_of_tile = ((128 + per_tile - 1) / per_tile + kA8Warps - 1) / kA8Warps;
  return launch_kernel("attention8_portion", attention8_portion_kernel<D, T>, dim3(p.nkv * blocks_of_tile, tiles), dim3(kA8Warps * 32), 0, stream, p);
}

template <typename T>
static int attention8_mma(A8Params p, int singles, int tiles, int d, int page_size, int per_head, void* stream) {
  PTL_REQUIRE(p.nq > 0 && p.nkv > 0 && page_size > 0 && p.num_pages > 0 && p.bt_stride > 0 && singles >= 0 && tiles >= 0, "attention8: bad sizes");
  PTL_REQUIRE(p.nq % p.nkv == 0, "attention8: %d query heads are no multiple of %d kv heads", p.nq, p.nkv);
  PTL_REQUIRE(page_size % kKv8Block == 0, "attention8: pages of %d positions are not whole blocks of %d", page_size, kKv8Block);
  if ((d != 64 && d != 128) || p.nq / p.nkv > 16 || tiles > 65535 || p.q_stride % 8 || p.out_stride % 8) return -2;
  PTL_REQUIRE(aligned16(p.q) && aligned16(p.out) && aligned16(p.codes) && (reinterpret_cast<uintptr_t>(p.words) & 7u) == 0,
              "attention8: q, out and codes must be 16-byte and words 8-byte aligned");
  PTL_REQUIRE(p.splits >= 1 && (!p.cluster || p.splits <= 8), "attention8: a cluster has up to 8 parts");
  PTL_REQUIRE(per_head == 0 || (p.units && aligned16(p.units) && p.counters && p.part_acc && p.part_ml), "attention8: units need their list and scratch");
  PTL_REQUIRE(per_head != 0 || p.splits == 1 || p.cluster, "attention8: parts of a token join in a cluster or are listed as units");
  p.blocks_per_page = page_size / kKv8Block;
  p.page_shift = -1;
  for (int b = 0; b < 20; ++b) if ((1 << b) == p.blocks_per_page) p.page_shift = b;
  if (singles == 0 && tiles == 0) return 0;
  return d == 64 ? launch_attention8<64, T>(p, singles, tiles, per_head, as_stream(stream)) : launch_attention8<128, T>(p, singles, tiles, per_head, as_stream(stream));
}

}  // namespace ptl

// Single tokens: `items` their rows (null: 0..n_items-1).  With per_head > 0 the keys are dealt out in units (`units` from
// ptl_decode_units_zeroed with the same sizes and with `counters`, one int per (row, kv head) of q), part_acc [nkv * per_head, nq / nkv, d] and part_ml
// [..., 2]; else every (token, kv head) has `splits` parts, up to 8, which join in a cluster.  -2: sizes this kernel does not take.
#define PTL_ATTENTION8_MMA(NAME, T)                                                                                                         \
  PTL_EXPORT int ptl_attention8_single_##NAME(void* out, float* part_acc, float* part_ml, const void* q, const void* codes,                 \
                                              const void* words, const int* block_table, const int* items, const int* tok_req,             \
                                              const int* positions, int n_items, int q_stride, int out_stride, int bt_stride, int nq,       \
                                              int nkv, int d, int page_size, float scale, int window, int splits, int per_head,             \
                                              const int* units, int* counters, int num_pages, void* stream) {                               \
    ptl::A8Params p{out, part_acc, part_ml, counters, q, (const unsigned char*)codes, (const uint32_t*)words, block_table, items, tok_req,  \
                    positions, (const int4*)units, q_stride, out_stride, bt_stride, nq, nkv, 0, 0, num_pages, window, splits,               \
                    per_head == 0 && splits > 1, scale * 1.4426950408889634f};                                                              \
    return ptl::attention8_mma<T>(p, n_items, 0, d, page_size, per_head, stream);                                                           \
  }                                                                                                                                         \
  PTL_EXPORT int ptl_attention8_portion_##NAME(void* out, const void* q, const void* codes, const void* words, const int* block_table,      \
                                               const int* tiles, int n_tiles, int q_stride, int out_stride, int bt_stride, int nq, int nkv, \
                                               int d, int page_size, float scale, int window, int num_pages, void* stream) {                \
    ptl::A8Params p{out, nullptr, nullptr, nullptr, q, (const unsigned char*)codes, (const uint32_t*)words, block_table, tiles, nullptr,    \
                    nullptr, nullptr, q_stride, out_stride, bt_stride, nq, nkv, 0, 0, num_pages, window, 1, 0,                              \
                    scale * 1.4426950408889634f};                                                                                           \
    return ptl::attention8_mma<T>(p, 0, n_tiles, d, page_size, 0, stream);                                                                  \
  }
PTL_ATTENTION8_MMA(f32, float)
PTL_ATTENTION8_MMA(bf16, __nv_bfloat16)
