// What a row of logits says about its next token: the log-probability of a given token, the entropy of the distribution,
// and the `top` most likely tokens with their log-probabilities, in one pass over the logits.
//
//   m = max x, S = sum e^(x - m), U = sum e^(x - m) (x - m)
//   log p(t) = x_t - m - log S          entropy = log S - U / S
//
// A row is cut into slices, one block of a cluster each.  A thread keeps (m, S, U) of what it has read; threads, then blocks are
// brought to one maximum.  The largest logits are found on the way: a 64-bit key holds the logit in an order of
// whole numbers and, below it, the index the other way round, so keys are unique and of equal logits the lowest index is
// the largest.  Every 4,096 logits, those above the threshold (the smallest of the `top` best so far) go to a list in shared
// memory.  Where more come than it has room for, the threshold is first raised to the `top`-th largest of the maxima of 64
// groups of 64 logits: at most `top` * 64 logits can lie above that, and the list holds as many.
//
// Logits of -inf have no probability.  A row with a NaN, with +inf, or with -inf only has no distribution: its
// log-probabilities and its entropy are NaN.  Its alternatives are the largest logits all the same, NaN behind all others.
#include "common.cuh"

namespace ptl {

constexpr int kTsThreads = 256;
constexpr int kTsPerThread = 16;                       // logits of a turn
constexpr int kTsTurn = kTsThreads * kTsPerThread;
constexpr int kTsMaxTop = 32;
constexpr int kTsGroups = 64;                          // of a turn, 4 threads each
constexpr int kTsRoom = kTsMaxTop * (kTsTurn / kTsGroups) + kTsMaxTop;      // of the list: the groups that may lie above a raised threshold, and what is there
constexpr int kTsMaxCluster = 8;

typedef unsigned long long TsKey;
// Larger logits have larger keys, equal ones larger keys at lower indices; NaN comes behind -inf.  No key is 0.
__device__ __forceinline__ TsKey ts_key(float x, int index) {
  uint32_t b = __float_as_uint(x);
  if (x == 0.f) b = 0u;                                // -0 equals 0
  const uint32_t order = x != x ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((TsKey)order << 32) | (uint32_t)~index;
}

__device__ __forceinline__ float ts_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The logit of a key (0 and NaN keys: NaN).
__device__ __forceinline__ float ts_logit(TsKey k) {
  const uint32_t order = (uint32_t)(k >> 32);
  return order == 0u ? __uint_as_float(0x7fc00000u) : __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

// A sum S of e^(x - m), and U of e^(x - m) (x - m), taken to the maximum `to` >= m.  Further apart than 200 nothing is left; logits
// of the type's lowest value are apart by what S times would not be a number.
__device__ __forceinline__ void ts_move(float m, float to, float& S, float& U) {
  if (m == -INFINITY) { S = S != S ? S : 0.f; U = 0.f; return; }      // (NaN in S: a logit was none)
  const float z = fmaxf(m - to, -200.f), f = ts_exp2(z * 1.4426950408889634f);
  U = f * (U + z * S);
  S *= f;
}

struct TsShared {
  TsKey list[kTsRoom];
  TsKey best[kTsMaxTop];                               // of this block, sorted
  TsKey group[kTsGroups];
  TsKey threshold;
  TsKey merged[kTsMaxCluster * kTsMaxTop];             // in the first block of a cluster: every block's best
  float sums[kTsMaxCluster][3];                        // ... and its m, S, U
  float red[33];
  int count;
};

// The `top` largest of n keys (unique, n >= top), sorted, to `best`: a key's place is the number of larger ones.
__device__ __forceinline__ void ts_select(const TsKey* keys, int n, int top, TsKey* best) {
  for (int i = threadIdx.x; i < n; i += kTsThreads) {
    const TsKey k = keys[i];
    int place = 0;
    for (int j = 0; j < n && place < top; ++j) place += keys[j] > k;
    if (place < top) best[place] = k;
  }
}

template <bool TOP>
__global__ void __launch_bounds__(kTsThreads, 3)
token_scores_kernel(float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_logprob, int* __restrict__ top_id,
                    const float* __restrict__ logits, const int* __restrict__ tokens, int vocab, int top, int slices) {
  extern __shared__ __align__(16) unsigned char smem[];
  TsShared& sh = *reinterpret_cast<TsShared*>(smem);
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int slice = blockIdx.x % slices;
  const long long row = blockIdx.x / slices;
  const float* x = logits + row * vocab;
  // slices begin at whole packets of four, counted from the packet that the row begins in
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15u) >> 2);
  const int packets = (vocab + skew + 3) / 4;
  const int per = (packets + slices - 1) / slices;
  const int p0 = slice * per, p1 = min(packets, p0 + per);
  if (TOP && tid == 0) { sh.count = 0; sh.threshold = 0; }
  float m = -INFINITY, S = 0.f, U = 0.f;
  const int want = TOP ? min(top, max(0, min(vocab, p1 * 4 - skew) - max(0, p0 * 4 - skew))) : 0;      // this block's share of the best
  if (TOP) __syncthreads();
  // a turn's logits are asked for while the turn before is worked on
  float ahead[kTsPerThread];
  auto ask = [&](int base) {
#pragma unroll
    for (int i = 0; i < kTsPerThread / 4; ++i) {
      const int p = base + i * kTsThreads + tid;
      const int e = p * 4 - skew;
      if (p < p1 && e >= 0 && e + 3 < vocab) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + e));
        ahead[4 * i] = f.x; ahead[4 * i + 1] = f.y; ahead[4 * i + 2] = f.z; ahead[4 * i + 3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) ahead[4 * i + j] = p < p1 && e + j >= 0 && e + j < vocab ? x[e + j] : -INFINITY;
      }
    }
  };
  ask(p0);
  for (int base = p0; base < p1; base += kTsTurn / 4) {
    float v[kTsPerThread];
#pragma unroll
    for (int i = 0; i < kTsPerThread; ++i) v[i] = ahead[i];
    if (base + kTsTurn / 4 < p1) ask(base + kTsTurn / 4);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < kTsPerThread; ++i) mx = fmaxf(mx, v[i]);
    if (mx > m) {                                      // (never at +inf twice)
      ts_move(m, mx, S, U);
      m = mx;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kTsPerThread; ++i) {
      const float z = v[i] - ref, e = ts_exp2(z * 1.4426950408889634f);
      S += e;                                          // (a NaN stays in it; +inf shows in the maximum)
      U = fmaf(e, fmaxf(z, -200.f), U);                // e^-200 is 0, and 0 * -200 is no NaN
    }
    if (TOP && want > 0) {
      // indices of this thread's logits: 4 * (base + i * kTsThreads + tid) - skew + j
      auto key_at = [&](int i) {
        const int e = 4 * (base + (i >> 2) * kTsThreads + tid) - skew + (i & 3);
        const bool here = base + (i >> 2) * kTsThreads + tid < p1 && e >= 0 && e < vocab;
        return here ? ts_key(v[i], e) : (TsKey)0;
      };
      TsKey threshold = sh.threshold;
      float least = ts_logit(threshold);               // (NaN, a threshold that is no number or none: everything comes in)
      const int threads_with = __syncthreads_count(!(mx < least));
      if (threads_with == 0) continue;                 // (the same in every thread)
      if (threads_with * kTsPerThread + sh.count > kTsRoom) {
        // raise the threshold: what the list holds down to the best, then the turn's group maxima
        if (sh.count > want) {
          const int n = sh.count;
          ts_select(sh.list, n, want, sh.best);
          __syncthreads();
          if (tid < want) sh.list[tid] = sh.best[tid];
          if (tid == 0) { sh.count = want; sh.threshold = max(sh.threshold, sh.best[want - 1]); }
        }
        TsKey mine = 0;
        if (mx > -INFINITY) {                          // the first of the thread's largest (what is behind the row is -inf)
#pragma unroll
          for (int i = kTsPerThread - 1; i >= 0; --i)
            if (v[i] == mx) mine = key_at(i);
        } else {
#pragma unroll
          for (int i = 0; i < kTsPerThread; ++i) mine = max(mine, key_at(i));
        }
#pragma unroll
        for (int o = 1; o < kTsThreads / kTsGroups; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (tid % (kTsThreads / kTsGroups) == 0) sh.group[tid / (kTsThreads / kTsGroups)] = mine;
        __syncthreads();
        if (tid < kTsGroups) {
          // the want-th largest group maximum (groups without logits have 0: no bound)
          const TsKey k = sh.group[tid];
          int place = 0;
          for (int j = 0; j < kTsGroups; ++j) place += sh.group[j] > k || (sh.group[j] == k && j < tid);
          // a logit equal to the threshold has to come in as well: the threshold is one less
          if (place == want - 1 && k > 0) atomicMax(&sh.threshold, k - 1);
        }
        __syncthreads();
        threshold = sh.threshold;
        least = ts_logit(threshold);
      }
      if (!(mx < least)) {
#pragma unroll
        for (int i = 0; i < kTsPerThread; ++i) {
          if (v[i] < least) continue;
          const TsKey k = key_at(i);
          if (k > threshold) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kTsRoom) sh.list[at] = k;
          }
        }
      }
      __syncthreads();
      if (sh.count >= 2 * want) {                      // an exact threshold keeps the list short
        const int n = min(sh.count, kTsRoom);
        ts_select(sh.list, n, want, sh.best);
        __syncthreads();
        if (tid < want) sh.list[tid] = sh.best[tid];
        if (tid == 0) { sh.count = want; sh.threshold = sh.best[want - 1]; }
      }
      __syncthreads();
    }
  }
  // ---- threads to one maximum
  const float bm = block_max(m, sh.red);
  ts_move(m, bm, S, U);
  const float bU = block_sum(U, sh.red);
  const float bS = block_sum(S, sh.red);
  if (TOP && want > 0) {
    ts_select(sh.list, sh.count, want, sh.best);
    __syncthreads();
  }
  // ---- blocks to the first of the cluster
  if (slices > 1) {
    cluster_arrive();                                  // every block of the cluster runs before a peer writes into it
    cluster_wait();
    if (tid < 3) st_peer_f32(map_to_peer((uint32_t)__cvta_generic_to_shared(&sh.sums[slice][tid]), 0), tid == 0 ? bm : tid == 1 ? bS : bU);
    if (TOP && tid < top) {
      const TsKey k = tid < want ? sh.best[tid] : 0;
      const uint32_t to = map_to_peer((uint32_t)__cvta_generic_to_shared(&sh.merged[slice * top + tid]), 0);
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to), "l"(k) : "memory");
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (slice != 0) return;
  }
  float M = bm, St = bS, Ut = bU;
  if (slices > 1) {
    M = -INFINITY;
    for (int s = 0; s < slices; ++s) M = fmaxf(M, sh.sums[s][0]);
    St = Ut = 0.f;
    for (int s = 0; s < slices; ++s) {
      float Ss = sh.sums[s][1], Us = sh.sums[s][2];
      ts_move(sh.sums[s][0], M, Ss, Us);
      St += Ss;
      Ut += Us;
    }
  }
  const float nan = __uint_as_float(0x7fc00000u);
  const bool bad = M == -INFINITY || M == INFINITY || St != St;
  const float log_sum = logf(St);
  if (tid == 0) {
    const int t = tokens[row];
    logprob[row] = bad ? nan : t >= 0 && t < vocab ? x[t] - M - log_sum : -INFINITY;
    entropy[row] = bad ? nan : log_sum - Ut / St;
  }
  if (TOP) {
    TsKey* all = sh.merged;
    const TsKey* best = sh.best;
    if (slices > 1) {
      // empty places (key 0) are the smallest: a place below `top` is a real key's, for top <= vocab
      for (int i = tid; i < slices * top; i += kTsThreads) {
        const TsKey k = all[i];
        if (k == 0) continue;
        int place = 0;
        for (int j = 0; j < slices * top; ++j) place += all[j] > k;
        if (place < top) sh.list[place] = k;
      }
      best = sh.list;
      __syncthreads();
    }
    if (tid < top) {
      const int id = (int)~(uint32_t)best[tid];
      top_id[row * top + tid] = id;
      top_logprob[row * top + tid] = bad ? nan : x[id] - M - log_sum;
    }
  }
}

}  // namespace ptl

// logits [rows, vocab] float32, tokens int32 [rows]; logprob and entropy float32 [rows], top_logprob float32 and top_id int32 [rows, top].
// top <= min(vocab, 32).  A token outside the vocabulary has log-probability -inf.
PTL_EXPORT int ptl_token_scores(float* logprob, float* entropy, float* top_logprob, int* top_id, const float* logits, const int* tokens,
                                int rows, int vocab, int top, void* stream) {
  using namespace ptl;
  PTL_REQUIRE(rows >= 0 && vocab > 0 && top >= 0, "token_scores: bad sizes");
  PTL_REQUIRE(top <= kTsMaxTop && top <= vocab, "token_scores: %d alternatives; at most %d, and no more than tokens", top, kTsMaxTop);
  PTL_REQUIRE(vocab <= 0x7fffff00 - kTsTurn, "token_scores: too many tokens");
  PTL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 3u) == 0, "token_scores: logits must be 4-byte aligned");
  if (rows == 0) return 0;
  int slices = 1;
  while (slices < kTsMaxCluster && (long long)rows * slices * 2 <= 1184 && vocab / (slices * 2) >= 4096) slices *= 2;
  PTL_REQUIRE((long long)rows * slices <= 0x7fffffffLL, "token_scores: too many rows");
  static SmemRaised raised[2] = {};
  constexpr int kSmem = (int)sizeof(TsShared);
  auto kernel = top ? token_scores_kernel<true> : token_scores_kernel<false>;
  if (int rc = raise_shared_memory("token_scores", kernel, kSmem, raised[top ? 1 : 0])) return rc;
  return launch_kernel_cluster("token_scores", kernel, dim3((unsigned)(rows * slices)), dim3(kTsThreads), kSmem, as_stream(stream), slices, logprob,
                               entropy, top_logprob, top_id, logits, tokens, vocab, top, slices);
}
