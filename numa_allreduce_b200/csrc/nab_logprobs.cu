// Log-probability of a given token, entropy and the k largest entries of
// every row of logits (no counterpart in the reference, which has no model
// code).
//
//   m = max x, S = sum exp(x - m), lse = m + log S
//   logprob = x[token] - lse,  entropy = log S - sum (x - m) exp(x - m) / S
//   top k: by value, equal values by the lowest index
//
// One pass over the row with a running (m, S, sum) per thread, so each logit
// is read from HBM once. The top k cost no second pass over the row: each
// thread notes, for each part of its share (an eighth, or a quarter), the
// maximum and the first 16-byte piece that held it. Take any partition of the
// row and order its parts by (maximum, piece): an element of the top k can
// only lie in a part whose key reaches the k-th of these keys, since each part
// before it holds an element that precedes it. The k-th of 64 coarse parts is
// a cut; the parts that reach it (about 1.2 k of them) are read again, from
// L2, and the elements that reach it are collected in shared memory and ranked
// by counting. If a contrived row overflows the collection, k rounds of a
// block maximum over the same pieces replace it.
//
// A row is shared by a thread-block cluster of 1 to 8 CTAs, which write their
// results into the first one's shared memory for it to join: one launch, no
// workspace, and a fixed order of additions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <string>

#include "nab_device.cuh"
#include "nab_driver.h"
#include "nab_logprobs.h"
#include "nab_sm100.cuh"

namespace nab {

namespace {

constexpr int kMaxCluster = 8;
constexpr int kCand = 1024;  // collected elements of a CTA
constexpr int kParts = 2048;  // parts of a CTA's share
constexpr int kPad = 24 * 1024;  // beside the static 37 KB of 256 threads: three CTAs per SM
constexpr int kCoarse = 64;  // parts that give the cut: the threads of one remainder mod 64
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

// Two floats in one 64-bit register: sm_100 adds and multiplies them in one instruction.
NAB_DINLINE uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
NAB_DINLINE float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
NAB_DINLINE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
NAB_DINLINE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
NAB_DINLINE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// How a piece of 16 bytes is read: its kN elements as pairs of floats, its
// largest element (NaN left out), a word of -inf, and how many of the lowest
// bits of `ordered` are the same for every value of the type and sign.
// kFloor: elements below it (masks of any kind, -inf) are raised to it
// (`raised`, in pairs for 16-bit types; NaN stays) and so count as
// probability 0 next to any maximum above kLow. Between kLow and kHigh the
// rounding of log2(e) max is below 2 in the exponent; a row whose maximum lies
// outside is summed again in another form.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr uint32_t kFill = 0xff800000u;
  static constexpr int kDrop = 0;
  static constexpr float kFloor = -0x1p24f, kLow = -0x1p23f, kHigh = 0x1p24f;
  NAB_DINLINE static uint4 raised(uint4 w) {
    return make_uint4(__float_as_uint(max_nan(__uint_as_float(w.x), kFloor)),
                      __float_as_uint(max_nan(__uint_as_float(w.y), kFloor)),
                      __float_as_uint(max_nan(__uint_as_float(w.z), kFloor)),
                      __float_as_uint(max_nan(__uint_as_float(w.w), kFloor)));
  }
  NAB_DINLINE static float largest(uint4 w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  NAB_DINLINE static void pairs(uint4 w, uint64_t (&v)[2]) {
    v[0] = pair(__uint_as_float(w.x), __uint_as_float(w.y));
    v[1] = pair(__uint_as_float(w.z), __uint_as_float(w.w));
  }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr uint32_t kFill = 0xff80ff80u;
  static constexpr int kDrop = 16;
  static constexpr float kFloor = -0x1p24f, kLow = -0x1p23f, kHigh = 0x1p24f;
  NAB_DINLINE static uint4 raised(uint4 w) {
    const __nv_bfloat162 f = __floats2bfloat162_rn(kFloor, kFloor);
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], f);
    return w;
  }
  NAB_DINLINE static float largest(uint4 w) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
    return fmaxf(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  NAB_DINLINE static void pairs(uint4 w, uint64_t (&v)[4]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pair(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  }
};
template <>
struct Piece<__half> {
  static constexpr uint32_t kFill = 0xfc00fc00u;
  static constexpr int kDrop = 13;
  static constexpr float kFloor = -60000.f, kLow = -50000.f, kHigh = 65504.f;
  NAB_DINLINE static uint4 raised(uint4 w) {
    const __half2 f = __floats2half2_rn(kFloor, kFloor);
    __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], f);
    return w;
  }
  NAB_DINLINE static float largest(uint4 w) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  NAB_DINLINE static void pairs(uint4 w, uint64_t (&v)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[i] = pair(f.x, f.y);
    }
  }
};

// m: the largest value so far. With e(x) = log2(e) x - l, l = scaled_max(m):
// s = sum 2^e(x), u = sum e(x) 2^e(x). One fused multiply-add gives e(x), and
// the rounding of l cancels, since lse = (l + log2 s) / log2(e) uses the same.
struct Stats {
  float m, s, u;
};
// (a rounded product of its own: fused into a difference, equal maxima would not cancel)
template <typename T>
NAB_DINLINE float scaled_max(float m) {
  return __fmul_rn(fmaxf(m, Piece<T>::kFloor), kL2e);
}
// exponents below -1000 count as -1000 (exp2 of them is zero), which keeps 0 * inf out
template <typename T>
NAB_DINLINE void raise(Stats& a, float m) {
  const float d = fmaxf(scaled_max<T>(a.m) - scaled_max<T>(m), -1000.f), f = lp_ex2(d);
  a.u = f * (a.u + d * a.s);
  a.s *= f;
  a.m = m;
}

template <int kThreads>
struct LpShared {
  float warp_m[kThreads / 32], warp_s[kThreads / 32], warp_u[kThreads / 32];
  // of each CTA of the cluster, written by that one into the first one's memory:
  Stats stats[kMaxCluster];
  uint64_t top[kMaxCluster * kMaxTopK]; // k largest keys, in order; 0 past its elements
  uint64_t cand[kCand];
  float2 part[kParts];       // of each part: its maximum, and as bits the first piece that holds it
  uint64_t best[kThreads];            // (value, piece) of each thread's largest, 0 without pieces
  uint64_t coarse[kCoarse];
  int coarse_rank[kCoarse];
  uint64_t cut;
  int who[kParts];           // parts that are read again
  int n_who, n_cand;
};

// Sum over the block, for every thread, in a fixed order; a and b are used again after the next barrier.
template <int kWarps>
NAB_DINLINE float2 block_sum(float2 v, float* a, float* b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (lane == 0) {
    a[warp] = v.x;
    b[warp] = v.y;
  }
  __syncthreads();
  v = lane < kWarps ? make_float2(a[lane], b[lane]) : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, v.x, 0), __shfl_sync(0xffffffffu, v.y, 0));
}

// A row as pieces of 16 aligned bytes: piece p holds the elements
// [p * kN - mis, (p + 1) * kN - mis), of which the first and the last piece
// may have some outside [0, V).
template <typename T>
struct Row {
  static constexpr int kN = VecT<T>::kN;
  const T* x;
  int mis;  // elements between the 16-byte boundary before x and x
  int V;
  NAB_DINLINE int first(int p) const { return p * kN - mis; }
  NAB_DINLINE bool inner(int p) const { return first(p) >= 0 && first(p) + kN <= V; }
  NAB_DINLINE uint4 whole(int p) const { return ld_plain(x + first(p)); }
};

// kCluster: rows are shared by clusters. Compiled apart: 1023 rows of one CTA each 52.5 -> 51.8 us.
template <typename T, bool kCluster, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    k_token_logprobs(const __grid_constant__ LogprobsArgs a, int cluster_size) {
  __shared__ LpShared<kThreads> sh;
  constexpr int kWarps = kThreads / 32;
  constexpr int kSub = kParts / kThreads;  // parts of a thread's share
  const int cluster = kCluster ? cluster_size : 1;
  constexpr int N = Row<T>::kN;
  constexpr int kBatch = 4;
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
  const int p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);  // this CTA's pieces
  const int i0 = max(p0, r.mis > 0), i1 = min(p1, (r.mis + a.V) / N);  // those within the row
  const int k = a.top_k;
  if (part == 0)
    for (int i = tid; i < cluster * k; i += kThreads) sh.top[i] = 0;
  if constexpr (kCluster) sm100::cluster_arrive();

  // ------------------------------------------------------- one pass --
  // Piece p is thread (p - p0) % kThreads's. Batches of kBatch pieces, the
  // next one's loads in flight during one's arithmetic; pieces past the end
  // read as -inf, i.e. as elements of probability 0.
  const int batches = ((p1 - p0 + kThreads - 1) / kThreads + kBatch - 1) / kBatch;
  const int sub_batches = max(1, (batches + kSub - 1) / kSub);
  // (value, piece within the CTA), larger = earlier, in as few bits as it takes
  const int piece_bits = 32 - __clz(p1 - p0);
  auto piece_key = [&](float x, int q) {
    return (static_cast<uint64_t>(ordered(x) >> Piece<T>::kDrop) << piece_bits) | static_cast<uint64_t>(p1 - 1 - q);
  };
  float big = -INFINITY;  // largest value so far, first held by piece big_at
  float kv = -INFINITY;   // the same within this part
  uint64_t s2 = 0, u2 = 0;
  float l = scaled_max<T>(big);
  const uint64_t l2e = pair(kL2e, kL2e);
  const uint4 fill = make_uint4(Piece<T>::kFill, Piece<T>::kFill, Piece<T>::kFill, Piece<T>::kFill);
  const uint4* at = reinterpret_cast<const uint4*>(r.x - r.mis) + p0 + tid;  // aligned; piece 0 may begin before x
  int p = p0 + tid, kp = p, big_at = p, sub = 0, left = sub_batches;
  uint4 cur[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const int q = p + b * kThreads;
    cur[b] = q >= i0 && q < i1 ? at[b * kThreads] : fill;
  }
  // (behind the first loads: a token's logit waits for its index)
  float picked = 0.f;  // the given token's logit, if it is in this part of the vocabulary
  bool here = false;
  if (tid == 0 && part == 0) {
    const int64_t token = a.tokens[row];  // any value
    here = token >= a.vocab_start && token - a.vocab_start < a.V;
    if (here) picked = static_cast<float>(r.x[token - a.vocab_start]);
  }
  for (int j = 0; j < batches; ++j) {
    uint4 next[kBatch];
    at += kBatch * kThreads;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      next[b] = fill;
      if (p + (kBatch + b) * kThreads < i1) next[b] = at[b * kThreads];
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const float mx = Piece<T>::largest(cur[b]);
      if (mx > kv) {
        kv = mx;
        kp = p + b * kThreads;
      }
    }
    {
      const float to = fmaxf(l, __fmul_rn(kv, kL2e));
      const float d = fmaxf(l - to, -1000.f), f = lp_ex2(d);
      const uint64_t f2 = pair(f, f);
      u2 = mul2(f2, fma2(pair(d, d), s2, u2));
      s2 = mul2(f2, s2);
      l = to;
    }
    const uint64_t neg = pair(-l, -l);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      uint64_t v[N / 2];
      Piece<T>::pairs(Piece<T>::raised(cur[b]), v);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const uint64_t x = fma2(v[e], l2e, neg);
        const float2 d = unpair(x);
        const uint64_t w = pair(lp_ex2(d.x), lp_ex2(d.y));
        s2 = add2(s2, w);
        u2 = fma2(x, w, u2);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) cur[b] = next[b];
    p += kBatch * kThreads;
    if (--left == 0 || j + 1 == batches) {  // the end of a part
      sh.part[sub * kThreads + tid] = make_float2(kv, __int_as_float(kp));
      if (kv > big) {
        big = kv;
        big_at = kp;
      }
      kv = -INFINITY;
      kp = p;
      ++sub;
      left = sub_batches;
    }
  }
  const int subs = sub;
  const float2 s_ = unpair(s2), u_ = unpair(u2);
  Stats st = {big, s_.x + s_.y, u_.x + u_.y};
  // the row's first and last piece, where they reach past it
  auto edge = [&](int q) {
    if (q < p0 || q >= p1 || r.inner(q) || (q - p0) % kThreads != tid) return;
    float2& part_max = sh.part[(q - p0) / kThreads / kBatch / sub_batches * kThreads + tid];
    for (int e = 0; e < N; ++e) {
      const int i = r.first(q) + e;
      if (i < 0 || i >= a.V) continue;
      const float x = static_cast<float>(r.x[i]);
      if (x > part_max.x || (x == part_max.x && q < __float_as_int(part_max.y)))
        part_max = make_float2(x, __int_as_float(q));
      if (x > st.m || (x == st.m && q < big_at)) big_at = q;
      if (x > st.m) raise<T>(st, x);
      const float d = fmaf(max_nan(x, Piece<T>::kFloor), kL2e, -scaled_max<T>(st.m)), w = lp_ex2(d);
      st.s += w;
      st.u += d * w;
    }
  };
  edge(0);
  if (pieces > 1) edge(pieces - 1);

  // ------------------------- statistics of the CTA, and the cut for its top k --
  float top = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sh.warp_m[warp] = top;
  sh.best[tid] = p0 + tid < p1 ? piece_key(st.m, big_at) : 0;
  if (tid < kCoarse) sh.coarse_rank[tid] = 0;
  if (tid == 0) {
    sh.n_who = sh.n_cand = 0;
    sh.cut = 0;
  }
  __syncthreads();
  if (tid < kCoarse) {
    uint64_t c = 0;
#pragma unroll
    for (int i = 0; i < kThreads / kCoarse; ++i) {
      const uint64_t b = sh.best[tid + i * kCoarse];
      c = b > c ? b : c;
    }
    sh.coarse[tid] = c;
  }
  top = sh.warp_m[lane % kWarps];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  raise<T>(st, top);
  const float2 sums = block_sum<kWarps>(make_float2(st.s, st.u), sh.warp_s, sh.warp_u);
  // where the first CTA takes this one's results from; it has started
  uint32_t stats_at = 0, top_at = 0;
  if constexpr (kCluster) {
    sm100::cluster_wait();
    stats_at = sm100::dsmem_addr(sm100::smem_u32(&sh.stats[part]), 0);
    top_at = sm100::dsmem_addr(sm100::smem_u32(&sh.top[part * k]), 0);
  }
  auto put = [&](int rank, uint64_t key) {
    if constexpr (kCluster) sm100::st_dsmem_u64(top_at + rank * 8, key); else sh.top[rank] = key;
  };
  if (tid == 0) {
    if constexpr (kCluster) {
      sm100::st_dsmem_f32(stats_at, top);
      sm100::st_dsmem_f32(stats_at + 4, sums.x);
      sm100::st_dsmem_f32(stats_at + 8, sums.y);
    } else {
      sh.stats[0] = {top, sums.x, sums.y};
    }
  }

  // ------------------------------------------------------ top k of the CTA --
  if (k > 0) {
    {
      constexpr int kEach = kCoarse * kCoarse / kThreads;  // comparisons of a thread
      const int i = tid % kCoarse, from = tid / kCoarse * kEach;
      const uint64_t mine = sh.coarse[i];
      int before = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) before += sh.coarse[from + j] > mine;
      if (before) atomicAdd(&sh.coarse_rank[i], before);
    }
    __syncthreads();
    // the k-th; if fewer than k coarse parts hold anything, the cut stays 0
    if (tid < kCoarse && sh.coarse_rank[tid] == k - 1 && sh.coarse[tid] != 0) sh.cut = sh.coarse[tid];
    __syncthreads();
    const uint64_t cut = sh.cut;
    for (int i = 0; i < subs; ++i) {
      const float2 part_max = sh.part[i * kThreads + tid];
      const int q = __float_as_int(part_max.y);
      if (q < p1 && piece_key(part_max.x, q) >= cut) sh.who[atomicAdd(&sh.n_who, 1)] = i * kThreads + tid;
    }
    __syncthreads();
    const int n_who = sh.n_who;
    const int depth = kBatch * sub_batches;  // pieces of a part, at most
    const uint32_t cut_value = static_cast<uint32_t>(cut >> piece_bits);
    auto for_elements = [&](auto f) {
      for (int i = tid; i < n_who * depth; i += kThreads) {
        const int part_at = sh.who[i / depth];
        const int q = p0 + part_at % kThreads + (part_at / kThreads * depth + i % depth) * kThreads;
        if (q >= p1) continue;
        if (r.inner(q)) {
          const uint4 w = r.whole(q);
          if ((ordered(Piece<T>::largest(w)) >> Piece<T>::kDrop) < cut_value) continue;
          Acc<T> v;
          acc_set(v, w);
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (piece_key(v.v[e], q) >= cut) f(key_of(v.v[e], static_cast<uint32_t>(r.first(q) + e)));
        } else {
          for (int j = max(0, r.first(q)); j < min(a.V, r.first(q) + N); ++j) {
            const float x = static_cast<float>(r.x[j]);
            if (piece_key(x, q) >= cut) f(key_of(x, static_cast<uint32_t>(j)));
          }
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
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t mine = sh.cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.cand[j] > mine;
        if (rank < k) put(rank, mine);
      }
    } else {
      uint64_t last = ~uint64_t{0};
      for (int i = 0; i < k; ++i) {
        uint64_t next = 0;
        for_elements([&](uint64_t x) {
          if (x < last && x > next) next = x;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t b = __shfl_xor_sync(0xffffffffu, next, o);
          next = b > next ? b : next;
        }
        if (lane == 0) sh.best[warp] = next;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) next = sh.best[w] > next ? sh.best[w] : next;
        if (tid == 0) put(i, next);
        last = next;
        __syncthreads();
      }
    }
  }

  // ---------------------------------------------------- join of the cluster --
  if constexpr (kCluster) sm100::cluster_sync(); else __syncthreads();
  if (part == 0) {
    Stats all = sh.stats[0];
    // keys of every CTA, one per thread; all are different
    static_assert(kMaxCluster * kMaxTopK <= kThreads, "one key per thread");
    const uint64_t mine = tid < cluster * k ? sh.top[tid] : 0;
    if constexpr (kCluster) {
      // every thread adds the CTAs up for itself, in their order
      for (int c = 1; c < cluster; ++c) all.m = fmaxf(all.m, sh.stats[c].m);
      all.s = all.u = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (c >= cluster) break;
        Stats one = sh.stats[c];
        raise<T>(one, all.m);
        all.s += one.s;
        all.u += one.u;
      }
    }
    const bool far = all.m > Piece<T>::kHigh || all.m < Piece<T>::kLow;
    if (all.m == -INFINITY && all.s == all.s) all.s = all.u = 0.f;  // nothing but -inf
    if (far && fabsf(all.m) != INFINITY) {  // this CTA sums the row again as it stands
      float2 sum = make_float2(0.f, 0.f);
      for (int i = tid; i < a.V; i += kThreads) {
        const float d = max_nan((static_cast<float>(r.x[i]) - all.m) * kL2e, -1000.f), w = lp_ex2(d);
        sum.x += w;
        sum.y += d * w;
      }
      __syncthreads();
      sum = block_sum<kWarps>(sum, sh.warp_s, sh.warp_u);
      all.s = sum.x;
      all.u = sum.y;
    }
    const float log2_s = log2f(all.s), scaled = scaled_max<T>(all.m);
    const float lse = far ? all.m + log2_s * kLn2 : (scaled + log2_s) * kLn2;
    auto logprob_of = [&](float x) {
      if (far) return (x - all.m) - log2_s * kLn2;
      return x < Piece<T>::kFloor ? x - lse : (fmaf(x, kL2e, -scaled) - log2_s) * kLn2;
    };
    if (tid == 0) {
      a.logprob[row] = here ? logprob_of(picked) : -INFINITY;
      a.lse[row] = lse;
      a.entropy[row] = (log2_s - all.u / all.s) * kLn2;
    }
    if (mine != 0) {
      int rank = tid;
      if constexpr (kCluster) {
        rank = 0;
        for (int j = 0; j < cluster * k; ++j) rank += sh.top[j] > mine;
      }
      if (rank < k) {
        const float x = unordered(static_cast<uint32_t>(mine >> 32));
        a.top_logprobs[row * k + rank] = logprob_of(x);
        a.top_logits[row * k + rank] = x;
        a.top_tokens[row * k + rank] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(mine)) + a.vocab_start;
      }
    }
  }
}

template <typename T>
void launch_lp(cudaStream_t s, const LogprobsArgs& a, int sms) {
  // While every CTA can have an SM to itself, it gets 512 threads, i.e. twice the loads in flight, and few long rows are
  // shared by clusters: at least 12000 elements per CTA while half of the SMs stay free, else 24000. Past that, 256
  // threads, four CTAs on an SM, and no clusters, which pay for two barriers and a slower launch. Measured (us, bf16,
  // k = 20): 256 threads with 1 / 2 / 4 / 8 CTAs per row; 512 threads: 1 x 128256 11.7 9.2 7.3 7.0; 10.2 8.6 7.4 7.2.
  // 16 rows 15.6 11.7 9.1 8.8; 11.0 9.4 8.1 9.6. 32 rows 15.7 12.0 9.6 9.9; 11.1 9.6 9.5 12.7. 64 rows 16.0 12.3 10.7
  // 13.7; 11.4 10.3 11.2 20.3. 148 rows 16.8 14.6 20.3 -; 12.7 14.3 24.8 -. 200 rows 18.7 20.4 - -; 17.9 22.1 - -. 1 x
  // 50000 7.8 7.1 6.2 6.5; 7.5 6.9 6.5 7.2. 32 rows 9.8 8.5 7.4 8.4; 8.1 7.6 7.6 12.0. 200 rows 11.7 13.9 - -; 12.4
  // 17.1 - -. 148 x 16032 6.5 7.1 12.8 -; 5.9 8.7 19.7 -. 400 rows 8.2; 11.2. k = 5, 1 x 1000 4.3; 4.8.
  const int64_t bytes = static_cast<int64_t>(a.V) * sizeof(T);
  const bool wide = a.rows <= sms && bytes >= 16 * 1024;
  int cluster = 1;
  for (int c = 2; wide && c <= kMaxCluster && a.rows * c <= sms; c *= 2) {
    if (a.V / c < (a.rows * c <= sms / 2 ? 12000 : 24000)) break;
    cluster = c;
  }
  cudaLaunchConfig_t cfg{};
  const int64_t grid = a.rows * cluster;
  if (grid > 0x7fffffff) throw std::invalid_argument("token_logprobs: too many rows for one launch");
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(wide ? 512 : 256);
  cfg.stream = s;
  // Four CTAs of 256 threads fit on an SM; of a grid that fills two to three per SM some SMs would get four and others
  // two. Shared memory that nobody uses makes it three: 300 x 128256 bf16 30.7 -> 25.2 us.
  if (grid > 2 * sms && grid <= 3 * sms) cfg.dynamicSmemBytes = kPad;
  const auto kernel = cluster > 1 ? k_token_logprobs<T, true, 512>
                                  : (wide ? k_token_logprobs<T, false, 512> : k_token_logprobs<T, false, 256>);
  static std::atomic<bool> ready[64];  // by device; setting it twice does no harm
  int dev = 0;
  NAB_CUDA_CHECK(cudaGetDevice(&dev));
  if (cfg.dynamicSmemBytes > 0 && !ready[dev & 63].load(std::memory_order_acquire)) {
    NAB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPad));
    ready[dev & 63].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, cluster);
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
