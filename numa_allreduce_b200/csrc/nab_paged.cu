// Block tables and slots of a paged KV cache, and the append of a step's k
// and v to it (no counterpart in the reference, which has no model code).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "nab_device.cuh"
#include "nab_driver.h"
#include "nab_kerr.h"
#include "nab_paged.h"

namespace nab {

namespace {

constexpr int kAssignThreads = 512;

NAB_DINLINE int64_t min64(int64_t x, int64_t y) { return x < y ? x : y; }

// With c cached and n new positions of a request, pages of P positions, table
// width M, F free pages of which u are taken:
//   old  = min(ceil(c / P), M)          pages it holds
//   need = min(ceil((c + n) / P), M) - old
//   off  = sum of `need` over the requests before it
//   new page i of all (request order): free_pages[u + i], none past F
//   token at position p: slot = page(p / P) * P + p % P, -1 without a page
// Latency is what counts: a decode step moves a few hundred bytes. Every CTA
// computes the scan over all requests by itself (B loads from L2) instead of
// a second launch or a grid barrier; the writes (tokens, new table entries,
// lengths) are spread over the grid. A token takes a new page's id from the
// free list, not from the table, so no CTA reads what another one writes.
__global__ void __launch_bounds__(kAssignThreads) k_assign_pages(const __grid_constant__ AssignPagesArgs a) {
  extern __shared__ int assign_smem[];
  int* off = assign_smem;         // [B]
  int* start = assign_smem + a.B;  // [B + 1], only with a.starts
  __shared__ int warp_sum[kAssignThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int taken = *a.taken;  // in flight during the scan
  auto new_tokens = [&](int b) { return a.starts ? max(0, a.starts[b + 1] - a.starts[b]) : 1; };
  auto pages_of = [&](uint32_t n) {  // n up to 2^31 + 2^30
    const uint32_t P = a.P;
    return static_cast<int>(min(n / P + (n % P != 0), static_cast<uint32_t>(a.M)));
  };
  int total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kAssignThreads) {
    const int b = b0 + tid;
    int need = 0;
    if (b < a.B) {
      const int c = max(0, a.cached[b]);
      need = pages_of(static_cast<uint32_t>(c) + new_tokens(b)) - pages_of(c);
      if (a.starts) start[b] = a.starts[b];
    }
    int x = need;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kAssignThreads / 32; ++w) {
      before += w < warp ? warp_sum[w] : 0;
      sum += warp_sum[w];
    }
    if (b < a.B) off[b] = total + before + x - need;
    total += sum;
    __syncthreads();
  }
  if (a.starts && tid == 0) start[a.B] = a.starts[a.B];
  __syncthreads();
  const int used = min(max(0, taken), a.F);
  const int avail = a.F - used;
  const int gtid = blockIdx.x * kAssignThreads + tid, gsize = gridDim.x * kAssignThreads;

  // new page i of all -> its request: the last b with off[b] <= i
  for (int i = gtid; i < total; i += gsize) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (off[mid] <= i) lo = mid; else hi = mid;
    }
    const int old = pages_of(max(0, a.cached[lo]));
    a.tables[lo * a.table_stride + old + (i - off[lo])] = i < avail ? a.free_pages[used + i] : -1;
  }
  for (int b = gtid; b < a.B; b += gsize) {
    const int c = max(0, a.cached[b]), old = pages_of(c);
    const uint32_t end = static_cast<uint32_t>(c) + new_tokens(b);
    const int have = old + min(max(0, avail - off[b]), pages_of(end) - old);
    a.lengths[b] = static_cast<int>(min64(min64(end, static_cast<int64_t>(have) * a.P), 0x7fffffff));
  }
  if (gtid == 0) *a.taken_out = used + min(total, avail);
  for (int t = gtid; t < a.T; t += gsize) {
    int b = t, row = 0;
    bool live = t < a.B;
    if (a.starts) {
      // the last request that starts at or before row t
      int lo = 0, hi = a.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
      }
      b = lo;
      live = t >= start[b] && t < start[b + 1];
      row = t - start[b];
    }
    uint32_t pos = 0;  // up to 2^31 + 2^30
    int64_t slot = -1;
    if (live) {
      const int c = max(0, a.cached[b]), old = pages_of(c);
      pos = static_cast<uint32_t>(c) + row;
      const int j = static_cast<int>(pos / static_cast<uint32_t>(a.P));
      int page = -1;
      if (j < old) {
        page = a.tables[b * a.table_stride + j];
      } else if (j < a.M) {
        const int i = off[b] + (j - old);
        if (i < avail) page = a.free_pages[used + i];
      }
      if (page >= 0) slot = static_cast<int64_t>(page) * a.P + (pos - static_cast<uint32_t>(j) * a.P);
    }
    a.positions[t] = static_cast<int>(min(pos, 0x7fffffffu));
    a.slots[t] = slot;
  }
}

struct RopeAppendDev {
  RopeAppendArgs a;
  ErrorState* err;
  uint32_t* err_host;
};

// y = x * rsqrt(mean(x^2) + eps) * w over a head (with norms), then for each
// pair (u, v) of its first R dims: (u c - v s, v c + u s); all in fp32 with
// one rounding at the end. k and v go to their page row, q to q_out.
//
// Bound by memory: each value is read and written once. One group of D / 16
// lanes per token and run of kHeads heads; a lane holds two 16-byte pieces
// of each head so that a rotary pair lies in one lane: half layout, dims
// [8c, 8c + 8) and [R/2 + 8c, ...); interleaved, dims [16c, 16c + 16); the
// lanes past R / 16 hold the rest of the head unrotated. The loads of all
// heads of a run are in flight together, and the token's cos and sin and the
// norm's weight stay in registers over them. A run is of q heads, of k heads
// or of v heads, the same for a whole block, and consecutive blocks take the
// runs of the same tokens (their cos and sin rows and cache lines of qkv).
// What limits it is how many bytes the resident threads keep in flight:
// 8191 tokens of 32 / 8 normed heads take 34.8 us (31.3 for a copy of the
// same bytes) with runs of 4 and 7 blocks of 128 threads per SM; 36.4 with 6,
// 38.2 with 5; blocks of 256, two per SM and runs of 8, 39.4.
constexpr int kAppendThreads = 128;
template <typename T, int D, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kAppendThreads, 7) k_rope_append_paged(const __grid_constant__ RopeAppendDev p) {
  constexpr int kLanes = D / 16, kTokens = kAppendThreads / kLanes;
  const RopeAppendArgs& a = p.a;
  pdl_wait();
  pdl_trigger();
  const int q_runs = (a.Hq + kHeads - 1) / kHeads, kv_runs = (a.Hkv + kHeads - 1) / kHeads;
  const unsigned runs = q_runs + 2 * kv_runs;
  const int run = static_cast<int>(blockIdx.x % runs);
  const int64_t token = static_cast<int64_t>(blockIdx.x / runs) * kTokens + threadIdx.x / kLanes;
  const bool live = token < a.T;
  // lanes past the end follow the last token without storing: the shuffles need the whole warp
  const int64_t t = live ? token : a.T - 1;
  const bool is_q = run < q_runs, is_v = run >= q_runs + kv_runs;
  const int h0 = (is_q ? run : is_v ? run - q_runs - kv_runs : run - q_runs) * kHeads;  // within its kind
  const int heads = min(kHeads, (is_q ? a.Hq : a.Hkv) - h0);
  const int c = threadIdx.x % kLanes;
  const bool rotated = c < a.R / 16;
  int d0, d1;  // the lane's two pieces of 8 dims
  if (kInterleaved || !rotated) {
    d0 = 16 * c;
    d1 = d0 + 8;
  } else {
    d0 = 8 * c;
    d1 = a.R / 2 + 8 * c;
  }
  const T* src = static_cast<const T*>(a.qkv) + t * a.qkv_stride +
                 static_cast<int64_t>((is_q ? 0 : is_v ? a.Hq + a.Hkv : a.Hq) + h0) * D;
  uint4 raw[kHeads][2];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = kHeads == 1 ? 0 : min(i, heads - 1);
    raw[i][0] = ld_plain(src + h * D + d0);
    raw[i][1] = ld_plain(src + h * D + d1);
  }

  // where the run's first head goes, and the distance between heads
  T* dst;
  int64_t step = D;
  bool store = live;
  if (is_q) {
    dst = static_cast<T*>(a.q_out) + (t * a.Hq + h0) * D;
  } else {
    const int64_t slot = a.slots[t];
    store = live && slot >= 0 && slot < a.num_slots;
    if (live && slot >= a.num_slots && h0 == 0 && !is_v && c == 0)
      record_local_failure(p.err, p.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(t));
    const uint32_t at = store ? static_cast<uint32_t>(slot) : 0u;  // below num_slots, which fits 32 bits
    const uint32_t page = at / static_cast<uint32_t>(a.P), row = at - page * a.P;
    dst = static_cast<T*>(is_v ? a.v_pages : a.k_pages) + ((static_cast<int64_t>(page) * a.Hkv + h0) * a.P + row) * D;
    step = static_cast<int64_t>(a.P) * D;
  }
  if (is_v) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (!store || i >= heads) break;
      st_plain(dst + i * step + d0, raw[i][0]);
      st_plain(dst + i * step + d1, raw[i][1]);
    }
    return;
  }

  // half layout: angle e belongs to dims (d0 + e, d1 + e); interleaved: to
  // (16c + 2e, 16c + 2e + 1)
  float cs[8], sn[8];
  if (rotated) {
    int pos = a.positions[t];
    if (pos < 0 || pos >= a.max_pos) {
      if (live && is_q && h0 == 0 && c == 0 && a.slots[t] >= 0)  // a token without a slot is dropped anyway
        record_local_failure(p.err, p.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(t));
      pos = min(max(pos, 0), a.max_pos - 1);
    }
    const float4* ct = reinterpret_cast<const float4*>(a.cos_t + static_cast<int64_t>(pos) * (a.R / 2) + 8 * c);
    const float4* st = reinterpret_cast<const float4*>(a.sin_t + static_cast<int64_t>(pos) * (a.R / 2) + 8 * c);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 x = __ldg(ct + k), y = __ldg(st + k);
      cs[4 * k] = x.x, cs[4 * k + 1] = x.y, cs[4 * k + 2] = x.z, cs[4 * k + 3] = x.w;
      sn[4 * k] = y.x, sn[4 * k + 1] = y.y, sn[4 * k + 2] = y.z, sn[4 * k + 3] = y.w;
    }
  }
  const T* w = static_cast<const T*>(is_q ? a.q_norm : a.k_norm);
  uint4 wr[2] = {};
  if (w != nullptr) {
    wr[0] = __ldg(reinterpret_cast<const uint4*>(w + d0));
    wr[1] = __ldg(reinterpret_cast<const uint4*>(w + d1));
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    Acc<T> x0, x1;
    acc_set(x0, raw[i][0]);
    acc_set(x1, raw[i][1]);
    if (w != nullptr) {  // the same for the whole block
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x0.v[e] * x0.v[e] + x1.v[e] * x1.v[e];
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      Acc<T> w0, w1;
      acc_set(w0, wr[0]);
      acc_set(w1, wr[1]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x0.v[e] *= inv * w0.v[e];
        x1.v[e] *= inv * w1.v[e];
      }
    }
    if (rotated) {
      if (kInterleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u0 = x0.v[2 * e], v0 = x0.v[2 * e + 1], u1 = x1.v[2 * e], v1 = x1.v[2 * e + 1];
          x0.v[2 * e] = u0 * cs[e] - v0 * sn[e];
          x0.v[2 * e + 1] = v0 * cs[e] + u0 * sn[e];
          x1.v[2 * e] = u1 * cs[4 + e] - v1 * sn[4 + e];
          x1.v[2 * e + 1] = v1 * cs[4 + e] + u1 * sn[4 + e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x0.v[e], v = x1.v[e];
          x0.v[e] = u * cs[e] - v * sn[e];
          x1.v[e] = v * cs[e] + u * sn[e];
        }
      }
    }
    if (store && i < heads) {
      st_plain(dst + i * step + d0, acc_pack(x0));
      st_plain(dst + i * step + d1, acc_pack(x1));
    }
  }
}

template <typename... KArgs, typename... Args>
void launch(void (*kernel)(KArgs...), int64_t grid, int block, size_t smem, cudaStream_t s, const char* what,
            Args... args) {
  if (grid > 0x7fffffff) throw std::invalid_argument(std::string(what) + ": too many rows for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + " launch failed: " + cudaGetErrorString(e));
}

template <typename T, int D, bool kInterleaved, int kHeads>
void launch_runs(cudaStream_t s, const RopeAppendDev& p) {
  constexpr int kTokens = kAppendThreads / (D / 16);
  const int64_t runs = (p.a.Hq + kHeads - 1) / kHeads + 2 * ((p.a.Hkv + kHeads - 1) / kHeads);
  launch(k_rope_append_paged<T, D, kInterleaved, kHeads>, (p.a.T + kTokens - 1) / kTokens * runs,
         kAppendThreads, 0, s, "rope_append_paged", p);
}

template <typename T, int D, bool kInterleaved>
void launch_append(cudaStream_t s, const RopeAppendDev& p, int sms) {
  // one head per group while that fills the GPU's threads less than twice, else runs of 4
  const int64_t threads = p.a.T * (p.a.Hq + 2 * p.a.Hkv) * (D / 16);
  if (threads <= int64_t{2} * sms * 2048) {
    launch_runs<T, D, kInterleaved, 1>(s, p);
  } else {
    launch_runs<T, D, kInterleaved, 4>(s, p);
  }
}

template <typename T>
void dispatch_append(cudaStream_t s, const RopeAppendDev& p, bool interleaved, int sms) {
  if (p.a.D == 64) {
    interleaved ? launch_append<T, 64, true>(s, p, sms) : launch_append<T, 64, false>(s, p, sms);
  } else {
    interleaved ? launch_append<T, 128, true>(s, p, sms) : launch_append<T, 128, false>(s, p, sms);
  }
}

}  // namespace

void assign_pages(cudaStream_t s, const AssignPagesArgs& a, int sms) {
  if (a.B < 1 || a.B > kMaxPagedRequests) throw std::invalid_argument("assign_pages: 1 to 8192 requests");
  const int64_t rows = std::max({a.T, a.B, 1});
  const int grid = static_cast<int>(std::min<int64_t>(sms, (rows + kAssignThreads - 1) / kAssignThreads));
  const size_t smem = (static_cast<size_t>(a.B) + (a.starts ? a.B + 1 : 0)) * sizeof(int);
  // The limit of 48 KB without opting in is for this and the kernel's static shared memory together. The attribute is
  // the device's and cheap: set on each such call.
  if (smem > 32 * 1024)
    NAB_CUDA_CHECK(cudaFuncSetAttribute(k_assign_pages, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (2 * kMaxPagedRequests + 1) * static_cast<int>(sizeof(int))));
  launch(k_assign_pages, grid, kAssignThreads, smem, s, "assign_pages", a);
}

void rope_append_paged(cudaStream_t s, const RopeAppendArgs& a, int dtype, bool interleaved, int sms) {
  if (a.T == 0) return;
  const KernelErrorRecord rec = kernel_error_record();
  const RopeAppendDev p{a, rec.dev, rec.host};
  if (dtype == kF16) {
    dispatch_append<__half>(s, p, interleaved, sms);
  } else {
    dispatch_append<__nv_bfloat16>(s, p, interleaved, sms);
  }
}

}  // namespace nab
