// Log-probability of a given token, entropy and the k largest entries of
// every row of logits (no counterpart in the reference, which has no model
// code).
//
//   m = max x, S = sum exp(x - m), lse = m + log S
//   logprob = x[token] - lse,  entropy = log S - sum (x - m) exp(x - m) / S
//   top k: by value, equal values by the lowest index
//
// One pass over the row with a running (m, S, sum) per thread, so each logit
// is read from HBM once. The top k cost no second pass over the row: along
// with its maximum each thread keeps the first piece (16 bytes) that held
// it. Order the threads by (maximum, piece): an element of the top k can only
// lie in the k first threads, because each thread before its own holds an
// element that precedes it. The k-th of these keys is found by bisection
// (block-wide counts), the pieces of k threads are read again (from L2),
// elements that can precede it are collected in shared memory and ranked by
// counting. If a contrived row overflows the collection, k rounds of a block
// maximum over the same pieces replace it.
//
// A row is shared by a thread-block cluster of 1 to 8 CTAs, joined by its
// first CTA over distributed shared memory: one launch, no workspace, and a
// fixed order of additions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <stdexcept>
#include <string>

#include "nab_device.cuh"
#include "nab_driver.h"
#include "nab_logprobs.h"
#include "nab_sm100.cuh"

namespace nab {

namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kCand = 1024;  // collected elements of a CTA
constexpr float kL2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

NAB_DINLINE float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that keeps NaN
NAB_DINLINE float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// Order-preserving image of a float in 32 bits (-0 as 0); NaN counts as -inf
// here, so every real element has a key above 0.
NAB_DINLINE uint32_t ordered(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
NAB_DINLINE float unordered(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// Larger = earlier in the top list: by value, then by the lowest index.
NAB_DINLINE uint64_t key_of(float x, uint32_t index) {
  return (static_cast<uint64_t>(ordered(x)) << 32) | (0xffffffffu - index);
}

// Running statistics: m >= every value so far (at least -FLT_MAX), S = sum
// exp(x - m), U = sum log2(e) (x - m) exp(x - m).
struct Stats {
  float m, s, u;
};
NAB_DINLINE void raise(Stats& a, float m) {
  // exponents below -1000 count as zero (exp2 of them is), which keeps 0 * inf out
  const float d = fmaxf((a.m - m) * kL2e, -1000.f);
  const float f = lp_ex2(d);
  a.u = f * (a.u + d * a.s);
  a.s *= f;
  a.m = m;
}
NAB_DINLINE Stats merge(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  raise(a, m);
  raise(b, m);
  return {m, a.s + b.s, a.u + b.u};
}

struct LpShared {
  Stats warp_stats[kLpWarps];
  Stats stats;                    // this CTA's, read by the cluster's first CTA
  uint64_t top[kMaxTopK];         // this CTA's largest keys, in order; 0 past its elements
  uint64_t cand[kCand];
  uint64_t best[kLpWarps];
  int who[kLpThreads];            // threads whose pieces are read again
  int n_who, n_cand;
};

// The largest t with at least k threads' keys >= t (0 if fewer than k keys
// are above 0): bisection from the top bit, which ends once exactly k are left.
NAB_DINLINE uint64_t kth_largest(uint64_t key, int k) {
  if (__syncthreads_count(key != 0) < k) return 0;
  uint64_t t = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t c = t | (uint64_t{1} << bit);
    const int n = __syncthreads_count(key >= c);
    if (n >= k) t = c;
    if (n == k) break;
  }
  return t;
}

template <typename T>
struct Row {
  static constexpr int kN = VecT<T>::kN;  // elements of a piece
  const T* x;       // the row
  int mis;          // elements between the 16-byte boundary before x and x
  int V;
  // piece p holds the elements [p * kN - mis, ...); those outside [0, V) read as `fill`
  NAB_DINLINE bool inner(int p) const { return p * kN >= mis && (p + 1) * kN - mis <= V; }
  NAB_DINLINE void load(int p, Acc<T>& a, float fill) const {
    const T* at = x + (static_cast<int64_t>(p) * kN - mis);
    if (inner(p)) {
      acc_set(a, ld_plain(at));
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const int i = p * kN - mis + e;
        a.v[e] = i >= 0 && i < V ? static_cast<float>(at[e]) : fill;
      }
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads) k_token_logprobs(const __grid_constant__ LogprobsArgs a, int cluster) {
  __shared__ LpShared sh;
  constexpr int N = Row<T>::kN;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / cluster;
  const int part = blockIdx.x % cluster;
  Row<T> r;
  r.x = static_cast<const T*>(a.logits) + row * a.stride;
  r.mis = static_cast<int>((reinterpret_cast<uintptr_t>(r.x) & 15u) / sizeof(T));
  r.V = a.V;
  const int pieces = (r.mis + a.V + N - 1) / N;
  const int per = (pieces + cluster - 1) / cluster;
  const int p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);
  const int k = a.top_k;

  // ------------------------------------------------------- one pass --
  Stats st = {-FLT_MAX, 0.f, 0.f};
  float kv = -INFINITY;  // largest value so far, first held by piece kp
  int kp = p0 + tid;
  auto take = [&](const Acc<T>& v, int p, int n_valid_mask) {
    float mx = v.v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, v.v[e]);
    if (mx > kv) {
      kv = mx;
      kp = p;
      if (mx > st.m) raise(st, mx);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = max_nan((v.v[e] - st.m) * kL2e, -1000.f);
      const float w = lp_ex2(d);
      if ((n_valid_mask >> e) & 1) {
        st.s += w;
        st.u += d * w;
      }
    }
  };
  constexpr int kUnroll = 4;
  int p = p0 + tid;
  for (; p + (kUnroll - 1) * kLpThreads < p1; p += kUnroll * kLpThreads) {
    if (r.inner(p) && r.inner(p + (kUnroll - 1) * kLpThreads)) {
      Acc<T> v[kUnroll];
      uint4 raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) raw[u] = ld_plain(r.x + (static_cast<int64_t>(p + u * kLpThreads) * N - r.mis));
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        acc_set(v[u], raw[u]);
        take(v[u], p + u * kLpThreads, (1 << N) - 1);
      }
    } else {
      for (int u = 0; u < kUnroll; ++u) {
        const int q = p + u * kLpThreads;
        Acc<T> v;
        r.load(q, v, -INFINITY);
        int mask = 0;
        for (int e = 0; e < N; ++e) mask |= (q * N - r.mis + e >= 0 && q * N - r.mis + e < a.V) << e;
        take(v, q, mask);
      }
    }
  }
  for (; p < p1; p += kLpThreads) {
    Acc<T> v;
    r.load(p, v, -INFINITY);
    int mask = (1 << N) - 1;
    if (!r.inner(p)) {
      mask = 0;
      for (int e = 0; e < N; ++e) mask |= (p * N - r.mis + e >= 0 && p * N - r.mis + e < a.V) << e;
    }
    take(v, p, mask);
  }

  // ------------------------------------------------ statistics of the CTA --
  Stats all = st;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats b = {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o),
                     __shfl_xor_sync(0xffffffffu, all.u, o)};
    all = merge(all, b);
  }
  if (lane == 0) sh.warp_stats[warp] = all;
  if (tid < kMaxTopK) sh.top[tid] = 0;
  if (tid == 0) sh.n_who = sh.n_cand = 0;
  __syncthreads();
  if (tid == 0) {
    Stats b = sh.warp_stats[0];
    for (int w = 1; w < kLpWarps; ++w) b = merge(b, sh.warp_stats[w]);
    sh.stats = b;
  }

  // ------------------------------------------------------ top k of the CTA --
  if (k > 0) {
    const bool has = p0 + tid < p1;
    const uint64_t key = has ? key_of(kv, static_cast<uint32_t>(kp)) : 0;
    const uint64_t cut = kth_largest(key, k);
    if (has && key >= cut) sh.who[atomicAdd(&sh.n_who, 1)] = tid;
    __syncthreads();
    const int n_who = sh.n_who;
    const int depth = (p1 - p0 + kLpThreads - 1) / kLpThreads;  // pieces of a thread, at most
    auto for_elements = [&](auto f) {
      for (int i = tid; i < n_who * depth; i += kLpThreads) {
        const int q = p0 + sh.who[i / depth] + (i % depth) * kLpThreads;
        if (q >= p1) continue;
        Acc<T> v;
        r.load(q, v, -INFINITY);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int index = q * N - r.mis + e;
          // as a thread's key would rank it, so that equal values of later pieces stay out
          if (index >= 0 && index < a.V && key_of(v.v[e], static_cast<uint32_t>(q)) >= cut)
            f(key_of(v.v[e], static_cast<uint32_t>(index)));
        }
      }
    };
    for_elements([&](uint64_t x) {
      const int at = atomicAdd(&sh.n_cand, 1);
      if (at < kCand) sh.cand[at] = x;
    });
    __syncthreads();
    const int n = sh.n_cand;
    if (n <= kCand) {
      for (int i = tid; i < n; i += kLpThreads) {
        const uint64_t mine = sh.cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.cand[j] > mine;
        if (rank < k) sh.top[rank] = mine;
      }
    } else {
      uint64_t last = ~uint64_t{0};
      for (int i = 0; i < k; ++i) {
        uint64_t best = 0;
        for_elements([&](uint64_t x) {
          if (x < last && x > best) best = x;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
          best = b > best ? b : best;
        }
        if (lane == 0) sh.best[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLpWarps; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        if (tid == 0) sh.top[i] = best;
        last = best;
        __syncthreads();
      }
    }
  }

  // ---------------------------------------------------- join of the cluster --
  if (cluster > 1) sm100::cluster_sync(); else __syncthreads();
  if (part == 0) {
    Stats b = sh.stats;
    uint64_t mine = 0;
    if (cluster > 1) {
      const uint32_t stats_at = sm100::smem_u32(&sh.stats);
      for (int c = 1; c < cluster; ++c) {
        const uint32_t at = sm100::dsmem_addr(stats_at, c);
        b = merge(b, {sm100::ld_dsmem_f32(at), sm100::ld_dsmem_f32(at + 4), sm100::ld_dsmem_f32(at + 8)});
      }
      // keys of every CTA, one per thread (8 x 32 at most); all are different
      if (tid < cluster * k) {
        const uint32_t at = sm100::dsmem_addr(sm100::smem_u32(&sh.top[tid % k]), tid / k);
        const uint32_t lo = __float_as_uint(sm100::ld_dsmem_f32(at)), hi = __float_as_uint(sm100::ld_dsmem_f32(at + 4));
        mine = (static_cast<uint64_t>(hi) << 32) | lo;
      }
      if (tid < kMaxCluster * kMaxTopK) sh.cand[tid] = mine;
      __syncthreads();
    } else if (tid < k) {
      mine = sh.top[tid];
    }
    const float log2_s = log2f(b.s);
    if (tid == 0) {
      const int64_t at = a.tokens[row] - a.vocab_start;
      float lp = -INFINITY;
      if (at >= 0 && at < a.V) lp = (static_cast<float>(r.x[at]) - b.m) - log2_s * kLn2;
      a.logprob[row] = lp;
      a.lse[row] = b.m + log2_s * kLn2;
      a.entropy[row] = (log2_s - b.u / b.s) * kLn2;
    }
    if (mine != 0) {
      int rank = tid;
      if (cluster > 1) {
        rank = 0;
        for (int j = 0; j < cluster * k; ++j) rank += sh.cand[j] > mine;
      }
      if (rank < k) {
        const float x = unordered(static_cast<uint32_t>(mine >> 32));
        a.top_logprobs[row * k + rank] = (x - b.m) - log2_s * kLn2;
        a.top_logits[row * k + rank] = x;
        a.top_tokens[row * k + rank] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(mine)) + a.vocab_start;
      }
    }
  }
  if (cluster > 1) sm100::cluster_sync();  // the first CTA has read the others
}

template <typename T>
void launch_lp(cudaStream_t s, const LogprobsArgs& a, int sms) {
  // CTAs per row: as many as keep two per SM busy, each with at least 2048 elements
  int cluster = 1;
  while (cluster < kMaxCluster && a.rows * cluster * 2 <= 2 * sms && a.V / (cluster * 2) >= 2048) cluster *= 2;
  cudaLaunchConfig_t cfg{};
  const int64_t grid = a.rows * cluster;
  if (grid > 0x7fffffff) throw std::invalid_argument("token_logprobs: too many rows for one launch");
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_token_logprobs<T>, a, cluster);
  if (e != cudaSuccess) throw std::runtime_error(std::string("token_logprobs launch failed: ") + cudaGetErrorString(e));
}

}  // namespace

void token_logprobs(cudaStream_t s, const LogprobsArgs& a, int dtype, int sms) {
  if (a.rows == 0) return;
  if (dtype == kF32) {
    launch_lp<float>(s, a, sms);
  } else if (dtype == kF16) {
    launch_lp<__half>(s, a, sms);
  } else {
    launch_lp<__nv_bfloat16>(s, a, sms);
  }
}

}  // namespace nab
