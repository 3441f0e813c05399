// Attention over an 8-bit cache (kv8.cuh) on the CUDA cores: any head size in multiples of 16 up to 256, any group of query
// heads, float32 or bfloat16.  What the tensor-core kernels of the 8-bit cache do not take comes here.
//
// One block per (token, query head, split of its keys), 128 keys a turn: a thread scores one key, then the block's threads
// share the turn's values out as (key lane, four dimensions).  Scores, running maximum and sum, and the accumulator are
// float32.  Positions max(0, p - window + 1)..p are seen; one whose page is missing is not.  A marked token's score is NaN.
// A row without keys is zeros.
//
// What bounds it: shared-memory reads of the query and the scores, one multiply-add each; no head size that the tensor cores take comes
// here but with the groups of more than 16 that they leave.  64 tokens of 256 to 2,560 keys (32 heads of 64 over 8) take 206 us here and 27 there.
#include "kv8.cuh"

namespace ptl {

constexpr int kA8Threads = 128;
constexpr int kA8MaxDim = 256;

template <typename T>
__global__ void __launch_bounds__(kA8Threads)
attention8_simt_kernel(T* __restrict__ out, float* __restrict__ part_acc, float* __restrict__ part_ml, const T* __restrict__ q,
                       const unsigned char* __restrict__ codes, const uint32_t* __restrict__ words, const int* __restrict__ block_table,
                       const int* __restrict__ tok_req, const int* __restrict__ positions, int q_stride, int out_stride, int bt_stride,
                       int nq, int nkv, int d, int page_size, float scale_log2, int window, int num_pages) {
  __shared__ float s_q[kA8MaxDim], s_p[kA8Threads], s_vstep[kA8Threads], s_scratch[33];
  __shared__ const unsigned char* s_v[kA8Threads];
  __shared__ float4 s_acc[kA8Threads];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int t = blockIdx.x / nq, h = blockIdx.x % nq, split = blockIdx.y, splits = gridDim.y;
  const int kvh = h / (nq / nkv);
  const int r = tok_req[t], p = positions[t];
  const int lo = window > 0 && p + 1 > window ? p + 1 - window : 0;
  const int turns = r < 0 || p < 0 ? 0 : (p - lo + kA8Threads) / kA8Threads;
  const int per = (turns + splits - 1) / splits;
  const int first = min(turns, split * per), last = min(turns, first + per);
  for (int i = tid; i < d; i += kA8Threads) s_q[i] = to_f32(q[(size_t)t * q_stride + (size_t)h * d + i]) * scale_log2;
  __syncthreads();
  const int groups = d / 4;                        // threads a key's values take, and keys at once
  const int at_once = kA8Threads / groups;
  const int my_key = tid / groups, my_dim = tid % groups * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m_run = -INFINITY, l_run = 0.f;
  const size_t plane = (size_t)nkv * page_size * d;
  for (int turn = first; turn < last; ++turn) {
    const int key = lo + turn * kA8Threads + tid;
    float s = -INFINITY, vstep = 0.f;
    const unsigned char* vrow = nullptr;
    if (key <= p) {
      const int block = key / page_size, page = block < bt_stride ? block_table[(size_t)r * bt_stride + block] : -1, off = key % page_size;
      if (page >= 0 && page < num_pages) {
        const unsigned char* krow = codes + (size_t)page * 2 * plane + ((size_t)kvh * page_size + off) * d;
        vrow = krow + plane;
        const uint2 w = *reinterpret_cast<const uint2*>(words + (((size_t)page * nkv + kvh) * (page_size / kKv8Block) + off / kKv8Block) * 2);
        float a0 = 0.f, a1 = 0.f;
        for (int i = 0; i < d; i += 16) {
          const uint4 c = *reinterpret_cast<const uint4*>(krow + i);
          const uint32_t four[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            a0 = fmaf(s_q[i + j], (float)((four[j / 4] >> (8 * (j % 4))) & 255u) - 127.5f, a0);
            a1 = fmaf(s_q[i + j + 1], (float)((four[j / 4] >> (8 * (j % 4) + 8)) & 255u) - 127.5f, a1);
          }
        }
        s = 2.0f * kv8_half_step(w.x & 255u) * (a0 + a1);
        if (((w.x | w.y) >> (16 + off % kKv8Block)) & 1u) s = __uint_as_float(0x7fc00000u);
        vstep = 2.0f * kv8_half_step(w.y & 255u);
      }
    }
    const float m_new = fmaxf(m_run, block_max(s, s_scratch));
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m_run - m_use);
    const float w = exp2f(s - m_use);
    s_p[tid] = w;
    s_vstep[tid] = vstep;
    s_v[tid] = vrow;
    l_run = l_run * alpha + block_sum(w, s_scratch);          // (its barriers publish the three arrays)
    m_run = m_new;
    acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
    if (my_key < at_once) {
      for (int j = my_key; j < kA8Threads; j += at_once) {
        const unsigned char* v = s_v[j];
        if (!v) continue;
        const uint32_t c = *reinterpret_cast<const uint32_t*>(v + my_dim);
        const float f = s_p[j] * s_vstep[j];
        acc.x = fmaf(f, (float)(c & 255u) - 127.5f, acc.x);
        acc.y = fmaf(f, (float)((c >> 8) & 255u) - 127.5f, acc.y);
        acc.z = fmaf(f, (float)((c >> 16) & 255u) - 127.5f, acc.z);
        acc.w = fmaf(f, (float)(c >> 24) - 127.5f, acc.w);
      }
    }
    __syncthreads();
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < groups) {
    float4 a = s_acc[tid];
    for (int j = 1; j < at_once; ++j) {
      const float4 b = s_acc[j * groups + tid];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    if (splits == 1) {
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
      T* o = out + (size_t)t * out_stride + (size_t)h * d + my_dim;
      o[0] = from_f32<T>(a.x * inv); o[1] = from_f32<T>(a.y * inv);
      o[2] = from_f32<T>(a.z * inv); o[3] = from_f32<T>(a.w * inv);
    } else {
      const size_t at = ((size_t)t * nq + h) * splits + split;
      *reinterpret_cast<float4*>(part_acc + at * d + my_dim) = a;
      if (tid == 0) {
        // natural logarithms for the merge; a sum that is no number must not count as one without keys
        part_ml[at * 2] = l_run != l_run ? 0.f : m_run * 0.6931471805599453f;
        part_ml[at * 2 + 1] = l_run;
      }
    }
  }
}

// defined in attention_simt.cu
int attention_merge_bf16(void* out, const float* part_acc, const float* part_ml, int tokens, int out_stride, int nq, int d, int splits,
                         const int* items, void* stream);
int attention_merge_f32(void* out, const float* part_acc, const float* part_ml, int tokens, int out_stride, int nq, int d, int splits,
                        const int* items, void* stream);

template <typename T>
static int attention8_simt(T* out, float* part_acc, float* part_ml, const T* q, const void* codes, const void* words, const int* block_table,
                           const int* tok_req, const int* positions, int tokens, int q_stride, int out_stride, int bt_stride, int nq, int nkv,
                           int d, int page_size, float scale, int window, int splits, int num_pages, void* stream) {
  PTL_REQUIRE(tokens >= 0 && nq > 0 && nkv > 0 && page_size > 0 && num_pages > 0 && bt_stride > 0, "attention8: bad sizes");
  PTL_REQUIRE(nq % nkv == 0, "attention8: %d query heads are no multiple of %d kv heads", nq, nkv);
  PTL_REQUIRE(d > 0 && d % 16 == 0 && d <= kA8MaxDim, "attention8: head size %d is no multiple of 16 up to %d", d, kA8MaxDim);
  PTL_REQUIRE(page_size % kKv8Block == 0, "attention8: pages of %d positions are not whole blocks of %d", page_size, kKv8Block);
  PTL_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(words) & 7u) == 0, "attention8: codes must be 16-byte and words 8-byte aligned");
  PTL_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || (part_acc && part_ml)), "attention8: splits > 1 need scratch buffers");
  PTL_REQUIRE((long long)tokens * nq <= 0x7fffffffLL, "attention8: too many rows");
  if (tokens == 0) return 0;
  int rc = launch_kernel("attention8_simt", attention8_simt_kernel<T>, dim3((unsigned)(tokens * nq), splits), dim3(kA8Threads), 0,
                         as_stream(stream), out, part_acc, part_ml, q, (const unsigned char*)codes, (const uint32_t*)words, block_table, tok_req,
                         positions, q_stride, out_stride, bt_stride, nq, nkv, d, page_size, scale * 1.4426950408889634f, window, num_pages);
  if (rc || splits == 1) return rc;
  return (sizeof(T) == 2 ? attention_merge_bf16 : attention_merge_f32)(out, part_acc, part_ml, tokens, out_stride, nq, d, splits, nullptr, stream);
}

}  // namespace ptl

// part_acc [tokens, nq, splits, d] and part_ml [tokens, nq, splits, 2] float32 where splits > 1.
#define PTL_ATTENTION8_ENTRY(NAME, T)                                                                                                     \
  PTL_EXPORT int ptl_attention8_simt_##NAME(void* out, float* part_acc, float* part_ml, const void* q, const void* codes,                 \
                                            const void* words, const int* block_table, const int* tok_req, const int* positions,         \
                                            int tokens, int q_stride, int out_stride, int bt_stride, int nq, int nkv, int d,              \
                                            int page_size, float scale, int window, int splits, int num_pages, void* stream) {            \
    return ptl::attention8_simt<T>((T*)out, part_acc, part_ml, (const T*)q, codes, words, block_table, tok_req, positions, tokens,        \
                                   q_stride, out_stride, bt_stride, nq, nkv, d, page_size, scale, window, splits, num_pages, stream);     \
  }
PTL_ATTENTION8_ENTRY(f32, float)
PTL_ATTENTION8_ENTRY(bf16, __nv_bfloat16)
