// What a row of logits says about its next token: the log-probability of a given token, the entropy of the distribution,
// and the `top` most likely tokens with their log-probabilities, in one pass over the logits.
//
//   m = max x, S = sum e^(x - m), U = sum e^(x - m) (x - m)
//   log p(t) = x_t - m - log S          entropy = log S - U / S
//
// A row is cut into slices, one block of a cluster each.  A thread keeps (m, S, U) of what it has read; threads, then blocks are
// brought to one maximum.  The largest logits are found on the way: a 64-bit key holds the logit in an order of
// whole numbers and, below it, the index the other way round, so keys are unique and of equal logits the lowest index is the
// largest.  Logits above the block's threshold go to a list of their warp's; where that grows to 32, they are ranked among the warp's best, which
// its lanes hold in order, by counting.  The threshold follows from what the threads know anyway: of 64 groups of four threads the
// `top`-th largest maximum so far is no larger than the `top`-th best logit, and little smaller; it is taken after 1, 4, 16, ... turns, and
// between those turns no barrier stands in the loop.  Where most lanes of a warp have a logit above it all the same (logits in ascending
// order, or equal ones), it is raised for them to the `top`-th largest of the lanes' own.  At the end what the warps have, then what
// the blocks have, is ranked the same way.
//
// What bounds it: the bytes where no alternatives are asked for (500 rows of 128,256: 42.8 us, 6.0 TB/s); with 20 of them 49.6, the turns that have
// logits above the threshold and the ranking at the end; 8 rows with five 9.3 us, a cluster of eight blocks a row, of which the bytes
// take 0.64: its start, four turns of loads with a threshold in the first and the fourth, the ranking and two cluster barriers.
//
// Logits of -inf have no probability.  A row with a NaN, with +inf, or with -inf only has no distribution: its
// log-probabilities and its entropy are NaN.  Its alternatives are the largest logits all the same, NaN behind all others.
#include "common.cuh"
#include <cstring>

namespace ptl {

constexpr int kTsWarps = 8;
constexpr int kTsThreads = kTsWarps * 32;
constexpr int kTsPerThread = 16;                       // logits of a turn
constexpr int kTsTurn = kTsThreads * kTsPerThread;
constexpr int kTsMaxTop = 32;
constexpr int kTsRoom = 32 * kTsPerThread + 31;        // of a warp's list: a turn's logits, and fewer than 32 that were left
constexpr int kTsMaxCluster = 8;
constexpr int kTsGroups = kTsThreads / 4;
static_assert(kTsGroups == 64, "six bits number the groups");
static_assert(kTsWarps <= kTsMaxCluster, "the warps' best and the blocks' have one place");

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
  TsKey list[kTsWarps][kTsRoom];
  TsKey all[kTsWarps * 64];                            // 32 for every warp to merge through; then what the warps have
  TsKey best[kTsMaxTop];                               // of the block
  TsKey threshold;
  TsKey merged[kTsMaxCluster * kTsMaxTop];             // in the first block of a cluster: every block's best
  float sums[kTsMaxCluster][3];                        // ... and its m, S, U
  __align__(16) uint32_t group[kTsGroups];
  float warp_sums[kTsWarps][3];
  int count[kTsWarps];
};

// Places the `top` largest of n keys (unique but for zeros, which are none) in order in best[0 .. top): a key's place is the number of larger ones.
__device__ __forceinline__ void ts_select(const TsKey* keys, int n, int top, TsKey* best) {
  if (n <= kTsThreads / 2) {                           // two or four threads a key
    const int parts = n <= kTsThreads / 4 ? 4 : 2, i = threadIdx.x / parts;
    const TsKey k = i < n ? keys[i] : 0;
    int place = 0;
#pragma unroll 8
    for (int j = threadIdx.x % parts; j < n; j += parts) place += keys[j] > k;
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    if (parts == 4) place += __shfl_xor_sync(0xffffffffu, place, 2);
    if (k != 0 && place < top && threadIdx.x % parts == 0) best[place] = k;
    return;
  }
  for (int i = threadIdx.x; i < n; i += kTsThreads) {
    const TsKey k = keys[i];
    if (k == 0) continue;
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += keys[j] > k;
    if (place < top) best[place] = k;
  }
}

// The 32 best of the warp, lane by lane in order, and 32 more keys (0: none), through 32 keys of shared memory.
__device__ __forceinline__ TsKey ts_merge(TsKey best, TsKey more, TsKey* through) {
  const int lane = threadIdx.x & 31;
  int place_best = lane, place_more = 0;
#pragma unroll 4
  for (int j = 0; j < 32; ++j) {
    const TsKey b = __shfl_sync(0xffffffffu, best, j), n = __shfl_sync(0xffffffffu, more, j);
    place_more += (b > more) + (n > more);
    place_best += n > best;
  }
  // (zeros share places behind all keys)
  through[lane] = 0;
  __syncwarp();
  if (best != 0 && place_best < 32) through[place_best] = best;
  if (more != 0 && place_more < 32) through[place_more] = more;
  __syncwarp();
  const TsKey r = through[lane];
  __syncwarp();
  return r;
}

template <bool TOP>
__global__ void __launch_bounds__(kTsThreads, 4)
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
  const int warp = tid >> 5, lane = tid & 31;
  if (slices > 1) cluster_arrive();                    // (waited for before a peer is written to: every block of the cluster runs by then)
  if (TOP) {
    if (tid == 0) sh.threshold = 0;
    if (tid < kTsMaxTop) sh.best[tid] = 0;
    __syncthreads();
  }
  float m = -INFINITY;
  float2 S2 = make_float2(0.f, 0.f), U2 = make_float2(0.f, 0.f);
  TsKey best = 0;                                      // the warp's lane-th best
  int have = 0;                                        // on the warp's list
  // packet i of the lane in the warp's turn from packet `base` on
  auto packet = [&](int base, int i) { return base + (warp * (kTsPerThread / 4) + i) * 32 + lane; };
  auto ask = [&](int base, float2 (&v)[kTsPerThread / 2]) {
#pragma unroll
    for (int i = 0; i < kTsPerThread / 4; ++i) {
      const int p = packet(base, i), e = p * 4 - skew;
      if (p < p1 && e >= 0 && e + 3 < vocab) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + e));
        v[2 * i] = make_float2(f.x, f.y);
        v[2 * i + 1] = make_float2(f.z, f.w);
      } else {
        float one[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) one[j] = p < p1 && e + j >= 0 && e + j < vocab ? x[e + j] : -INFINITY;
        v[2 * i] = make_float2(one[0], one[1]);
        v[2 * i + 1] = make_float2(one[2], one[3]);
      }
    }
  };
  auto flush = [&]() {                                 // the list into the best
    for (int i = 0; i < have; i += 32) best = ts_merge(best, i + lane < have ? sh.list[warp][i + lane] : 0, sh.all + warp * 32);
    have = 0;
    const TsKey last = __shfl_sync(0xffffffffu, best, top - 1);
    if (lane == 0 && last != 0) atomicMax(&sh.threshold, last);
    __syncwarp();
  };
  auto work = [&](int base, int turn, const float2 (&v)[kTsPerThread / 2]) {
    auto at = [&](int i) { return i % 2 ? v[i / 2].y : v[i / 2].x; };
    float mx = fmaxf(v[0].x, v[0].y);
#pragma unroll
    for (int i = 1; i < kTsPerThread / 2; ++i) mx = fmaxf(mx, fmaxf(v[i].x, v[i].y));
    if (mx > m) {                                      // (never at +inf twice)
      ts_move(m, mx, S2.x, U2.x);
      ts_move(m, mx, S2.y, U2.y);
      m = mx;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const float2 ref2 = make_float2(ref, ref), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
    for (int i = 0; i < kTsPerThread / 2; ++i) {
      const float2 z = sub2(v[i], ref2), y = mul2(z, log2e);
      const float2 e = make_float2(ts_exp2(y.x), ts_exp2(y.y));
      S2 = add2(S2, e);                                // (a NaN stays in it; +inf shows in the maximum)
      U2 = fma2(e, make_float2(fmaxf(z.x, -200.f), fmaxf(z.y, -200.f)), U2);      // e^-200 is 0, and 0 * -200 is no NaN
    }
    if (!TOP) return;
    if ((turn & 0x55555555) == turn && (turn & (turn - 1)) == 0) {      // 1, 4, 16, ...: the same in every thread
      float g = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
      // the maximum in the order of whole numbers, its last six bits the group's number: unique, and no larger
      const uint32_t mine = ((uint32_t)(ts_key(g, 0) >> 32) & ~63u) | (uint32_t)(tid / 4);
      if (tid % 4 == 0) sh.group[tid / 4] = mine;
      __syncthreads();
      int place = 0;                                   // each of a group's four threads looks at a quarter of the others
#pragma unroll
      for (int j = 0; j < kTsGroups / 16; ++j) {
        const uint4 o = reinterpret_cast<const uint4*>(sh.group)[tid % 4 * (kTsGroups / 16) + j];
        place += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      }
      place += __shfl_xor_sync(0xffffffffu, place, 1);
      place += __shfl_xor_sync(0xffffffffu, place, 2);
      // (-inf: a group without logits, or of no probability: no bound)
      if (tid % 4 == 0 && place == top - 1 && g > -INFINITY) {
        const TsKey bound = (TsKey)(mine & ~63u) << 32;          // below every key with that logit
        if (bound > sh.threshold) sh.threshold = bound;          // (the one thread that writes between the barriers)
      }
      __syncthreads();
    }
    TsKey threshold = *const_cast<volatile TsKey*>(&sh.threshold);
    float least = ts_logit(threshold);                 // (NaN, a threshold that is no number or none: everything comes in)
    const int lanes_with = __popc(__ballot_sync(0xffffffffu, !(mx < least)));
    if (lanes_with == 0) return;
    auto pick = [&](int i) {                           // at(i), i no constant
      float x8[8], x4[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) x8[j] = i & 1 ? v[j].y : v[j].x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x4[j] = i & 2 ? x8[2 * j + 1] : x8[2 * j];
      const float lo = i & 4 ? x4[1] : x4[0], hi = i & 4 ? x4[3] : x4[2];
      return i & 8 ? hi : lo;
    };
    static_assert(kTsPerThread == 16, "four choices between two");
    auto key_of = [&](int i, float x_i) {
      const int p = packet(base, i / 4), e = 4 * p - skew + i % 4;
      return p < p1 && e >= 0 && e < vocab ? ts_key(x_i, e) : (TsKey)0;
    };
    if (lanes_with > 16) {
      TsKey mine = 0;
      if (mx > -INFINITY) {                            // the first of the lane's largest (what is behind the row is -inf)
        int first = 0;
#pragma unroll
        for (int i = kTsPerThread - 1; i >= 0; --i)
          if (at(i) == mx) first = i;
        mine = key_of(first, mx);
      } else {
#pragma unroll 1
        for (int i = 0; i < kTsPerThread; ++i) mine = max(mine, key_of(i, pick(i)));
      }
      int place = 0;
      for (int j = 0; j < 32; ++j) place += __shfl_sync(0xffffffffu, mine, j) > mine;
      // (lanes without logits have 0 and come last; one less, so that the key itself comes in)
      const unsigned who = __ballot_sync(0xffffffffu, place == top - 1 && mine != 0);
      if (who) {
        const TsKey raised = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1) - 1;
        if (raised > threshold) { threshold = raised; least = ts_logit(raised); }
      }
    }
    // a bit for each logit that some lane may keep; few, and what they cost is theirs, not the sixteen's (2,300 cycles a turn that had one when
    // every logit of a thread was voted on, 100 rows with 20 alternatives 31 us)
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kTsPerThread; ++i)
      if (!(at(i) < least)) bits |= 1u << i;
#pragma unroll 1
    for (uint32_t left = __reduce_or_sync(0xffffffffu, bits); left; left &= left - 1) {
      const int i = __ffs(left) - 1;
      const TsKey k = key_of(i, pick(i));
      const unsigned who = __ballot_sync(0xffffffffu, k > threshold);
      if (k > threshold) sh.list[warp][have + __popc(who & ((1u << lane) - 1u))] = k;
      have += __popc(who);
    }
    __syncwarp();
    if (have >= 32) flush();
  };
  // a turn's logits are asked for while the turn before is worked on
  constexpr int kStep = kTsTurn / 4;
  float2 a[kTsPerThread / 2], b[kTsPerThread / 2];
  ask(p0, a);
  int turn = 1;
  for (int base = p0; base < p1; base += 2 * kStep, turn += 2) {
    if (base + kStep < p1) ask(base + kStep, b);
    work(base, turn, a);
    if (base + kStep >= p1) break;
    if (base + 2 * kStep < p1) ask(base + 2 * kStep, a);
    work(base + kStep, turn + 1, b);
  }
  // ---- threads, then warps to one maximum; what the warps have side by side
  float S = S2.x + S2.y, U = U2.x + U2.y;
  const float wm = warp_max(m);
  ts_move(m, wm, S, U);
  S = warp_sum(S);
  U = warp_sum(U);
  if (lane == 0) { sh.warp_sums[warp][0] = wm; sh.warp_sums[warp][1] = S; sh.warp_sums[warp][2] = U; }
  const int kept = TOP ? __popc(__ballot_sync(0xffffffffu, best != 0)) : 0;
  if (TOP && lane == 0) sh.count[warp] = kept + have;
  __syncthreads();
  float bm = -INFINITY, bS = 0.f, bU = 0.f;
  int before = 0, found_all = 0;
#pragma unroll
  for (int w = 0; w < kTsWarps; ++w) bm = fmaxf(bm, sh.warp_sums[w][0]);
#pragma unroll
  for (int w = 0; w < kTsWarps; ++w) {
    float s = sh.warp_sums[w][1], u = sh.warp_sums[w][2];
    ts_move(sh.warp_sums[w][0], bm, s, u);
    bS += s;
    bU += u;
    if (TOP) {
      if (w < warp) before += sh.count[w];
      found_all += sh.count[w];
    }
  }
  if (TOP) {
    if (lane < kept) sh.all[before + lane] = best;
    if (lane < have) sh.all[before + kept + lane] = sh.list[warp][lane];
    __syncthreads();
    ts_select(sh.all, found_all, top, sh.best);
    __syncthreads();
  }
  // ---- blocks to the first of the cluster
  if (slices > 1) {
    cluster_wait();
    if (tid < 3) st_peer_f32(map_to_peer((uint32_t)__cvta_generic_to_shared(&sh.sums[slice][tid]), 0), tid == 0 ? bm : tid == 1 ? bS : bU);
    if (TOP && tid < top) {
      const TsKey k = sh.best[tid];
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
    const TsKey* found = sh.best;
    if (slices > 1) {
      // (a place below `top` is a real key's: top <= vocab)
      ts_select(all, slices * top, top, sh.list[0]);
      found = sh.list[0];
      __syncthreads();
    }
    if (tid < top) {
      const int id = (int)~(uint32_t)found[tid];
      top_id[row * top + tid] = id;
      top_logprob[row * top + tid] = bad ? nan : x[id] - M - log_sum;
    }
  }
}

}  // namespace ptl

// logits [rows, vocab] float32, tokens int32 [rows]; logprob and entropy float32 [rows], top_logprob float32 and top_id int32 [rows, top].
// top <= min(vocab, 32).  A token outside the vocabulary has log-probability -inf.  The arguments are packed by the caller.
struct TokenScoresArgs {
  float *logprob, *entropy, *top_logprob;
  int* top_id;
  const float* logits;
  const int* tokens;
  void* stream;
  int rows, vocab, top, zero;
};
static_assert(sizeof(TokenScoresArgs) == 7 * 8 + 4 * 4, "as it is packed");
PTL_EXPORT int ptl_token_scores(const void* args) {
  TokenScoresArgs a;
  memcpy(&a, args, sizeof a);
  const int rows = a.rows, vocab = a.vocab, top = a.top;
  const float* logits = a.logits;
  using namespace ptl;
  PTL_REQUIRE(rows >= 0 && vocab > 0 && top >= 0, "token_scores: bad sizes");
  PTL_REQUIRE(top <= kTsMaxTop && top <= vocab, "token_scores: %d alternatives; at most %d, and no more than tokens", top, kTsMaxTop);
  PTL_REQUIRE(vocab <= 0x7fffff00 - kTsTurn, "token_scores: too many tokens");
  PTL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 3u) == 0, "token_scores: logits must be 4-byte aligned");
  if (rows == 0) return 0;
  // As many slices as are resident at once; with alternatives and more rows than SMs one, because a slice's first turns, before its threshold is
  // near, cost more than its last (128,256 logits, 20 alternatives: 100 rows in 1, 2 and 4 slices 30.7, 29.2 and 27.3 us, 200 rows in 1 and
  // 2 34.4 and 42.8, 290 36.3 and 43.9).
  int slices = 1;
  if (top == 0 || rows <= 148)
    while (slices < kTsMaxCluster && (long long)rows * slices * 2 <= 592 && vocab / (slices * 2) >= 4096) slices *= 2;
  PTL_REQUIRE((long long)rows * slices <= 0x7fffffffLL, "token_scores: too many rows");
  static SmemRaised raised[2] = {};
  constexpr int kSmem = (int)sizeof(TsShared);
  auto kernel = top ? token_scores_kernel<true> : token_scores_kernel<false>;
  if (int rc = raise_shared_memory("token_scores", kernel, kSmem, raised[top ? 1 : 0])) return rc;
  return launch_kernel_cluster("token_scores", kernel, dim3((unsigned)(rows * slices)), dim3(kTsThreads), kSmem, as_stream(a.stream), slices, a.logprob,
                               a.entropy, a.top_logprob, a.top_id, logits, a.tokens, vocab, top, slices);
}
