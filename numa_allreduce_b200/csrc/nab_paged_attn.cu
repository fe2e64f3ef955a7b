// GQA attention of one new token per request over a paged KV cache.
//
//   o[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j,  j < lengths[b]
//
// K and V are read once, so HBM bandwidth bounds it: 4 * G * D operations per
// position and kv head (G = Hq / Hkv query heads) against 4 * D bytes, i.e. G
// operations a byte. The contractions are warp-level 16-bit MMAs (m16n8k16,
// fp32 accumulators): rows are the query heads of one kv head, so one
// operand pass serves up to 16 heads, and the probabilities stay in registers
// between the two products. A tcgen05 version needs them in shared memory
// and two TMEM round trips with CTA barriers per chunk (the contiguous-cache
// kernel of nab_attn_sm100.cu), a serial chain that costs more than the
// bytes of a chunk; here four warps stream independently.
//
// Work: the (request, kv head, head tile) segments, cut into tiles of 64
// positions, laid end to end and dealt out in equal contiguous ranges to a
// grid of two CTAs per SM, so that ragged batches and single long requests
// load the GPU alike. Lengths are read on the device (a captured graph
// replays at any lengths); each CTA finds its range from a scan over them. A
// segment that lies in one CTA is written at once; of a segment that is cut,
// each CTA leaves (max, sum, unnormalised output) in fp32 and a second
// launch joins the parts in order.
//
// CTA: warp 4 produces, warps 0-3 consume. A tile arrives as TMA boxes of 16
// rows x 64 dims (128-byte swizzle), one per producer lane, looked up in the
// block table box by box (any page size that is a multiple of 16). Warp w takes rows [16w, 16w + 16) of
// each tile with its own running maximum and sum, so the warps meet only at
// the end of a segment.
//
// Every mbarrier wait is bounded. One that runs out records into the device's
// kernel error record; the CTA's warps then walk their ranges without
// waiting or computing (the same barriers), the producer waits (bounded) for
// its copies in flight, and the kernel returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <stdexcept>
#include <string>

#include "nab_device.cuh"
#include "nab_driver.h"
#include "nab_kerr.h"
#include "nab_paged.h"
#include "nab_sm100.cuh"

namespace nab {

namespace {

constexpr int kTile = 64;       // positions per stage
constexpr int kBoxRows = 16;    // rows of one TMA box: one consumer warp's share of a tile
constexpr int kConsumers = 4;   // consumer warps
constexpr int kPThreads = 32 * (kConsumers + 1);
constexpr int kRows = 16;       // query heads of one head tile (the MMA's M)
constexpr int kJoinThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct PagedCfg {
  static constexpr int kBoxBytes = kBoxRows * D * 2;
  static constexpr int kStageBytes = 2 * (kTile / kBoxRows) * kBoxBytes;  // K boxes, then V boxes
  static constexpr int kStages = 96 * 1024 / kStageBytes;                 // 3 (D = 128), 6 (D = 64)
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kMergeBytes = 2 * 8 * D * 4;  // two warps' partial of 8 rows
  static constexpr int kQ = kStages * kStageBytes;   // two buffers behind the ring
  static constexpr int kMerge = kQ + 2 * kQBytes;
  static constexpr int kMl = kMerge + kMergeBytes;   // [2][8][2] floats: (max, sum)
  static constexpr int kBars = kMl + 2 * 8 * 2 * 4;
  static constexpr int kMisc = kBars + (2 * kStages + 2) * 8;
  static constexpr int kSmem = kMisc + 64;
};

struct PagedDev {
  const int* tables;
  int64_t table_stride;
  const int* lengths;
  void* out;
  float* ws_o;    // [2 * grid][16][D]
  float2* ws_ml;  // [2 * grid][16]
  int4* desc;     // [grid]: the cut segment that begins in a CTA (row, heads, last CTA, 1), or w = 0
  int num_pages;
  int B, M, P, Hq, Hkv;
  int G;          // query heads per kv head
  int HT, GT;     // head tiles per kv head, heads per tile
  float scale_log2;
  ErrorState* err;
  uint32_t* err_host;
  uint64_t timeout_ns;
};

NAB_DINLINE void bar_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory"); }

NAB_DINLINE void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(sm100::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(sm100::smem_u32(bar))
      : "memory");
}
NAB_DINLINE void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
NAB_DINLINE void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
NAB_DINLINE void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
NAB_DINLINE void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
NAB_DINLINE void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
NAB_DINLINE uint32_t pack2(float lo, float hi);
template <>
NAB_DINLINE uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
NAB_DINLINE uint32_t pack2<__half>(float lo, float hi) {
  return pack_f16x2(lo, hi);
}
NAB_DINLINE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

NAB_DINLINE int64_t min64(int64_t x, int64_t y) { return x < y ? x : y; }

// A walk over the segments of one CTA's range [x, x1) of tiles.
struct Walk {
  int x, x1;     // next tile, end of the range (in tiles, all segments end to end)
  int b, h;      // request, kv head * HT + head tile
  int nt, len;   // tiles and positions of request b
  int t0;        // first tile of the current piece within the segment
};

// Length of request b, within what its table row can hold.
NAB_DINLINE int length_of(const PagedDev& a, int b) {
  return static_cast<int>(min64(max(a.lengths[b], 0), static_cast<int64_t>(a.M) * a.P));
}

template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kPThreads, 2)
    k_paged_attn(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                 const __grid_constant__ CUtensorMap tq, const __grid_constant__ PagedDev a) {
  using C = PagedCfg<D>;
  constexpr int S = C::kStages;
  constexpr int kHalves = D / 64;            // 128-byte column blocks of a row
  constexpr int kHalfBytes = kBoxRows * 128;  // of a K or V box, and of a Q buffer
  extern __shared__ __align__(1024) uint8_t paged_smem[];
  const uint32_t base = sm100::smem_u32(paged_smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(paged_smem + C::kBars);
  uint64_t* empty = full + S;
  uint64_t* q_empty = empty + S;
  int* misc = reinterpret_cast<int*>(paged_smem + C::kMisc);  // abort, b, first tile of b, total tiles, warp sums
  volatile int* abort_flag = misc;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int HH = a.Hkv * a.HT;

  if ((base & 1023u) != 0) {  // the swizzled tiles need it; the launch has no static shared memory before them
    if (tid == 0) record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, base);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], kConsumers);
    }
    sm100::mbar_init(&q_empty[0], kConsumers);
    sm100::mbar_init(&q_empty[1], kConsumers);
    sm100::fence_barrier_init();
    misc[0] = 0;
    misc[1] = a.B;
    sm100::prefetch_tensormap(&tk);
    sm100::prefetch_tensormap(&tv);
    sm100::prefetch_tensormap(&tq);
  }
  pdl_wait();
  pdl_trigger();

  // Scan of the requests' tile counts: thread i holds the requests
  // [i * per_thread, ...), then a block scan.
  const int per_thread = (a.B + kPThreads - 1) / kPThreads;
  const int rb0 = min(a.B, tid * per_thread), rb1 = min(a.B, rb0 + per_thread);
  int mine = 0;
  for (int b = rb0; b < rb1; ++b) {
    const int raw = a.lengths[b];
    if (blockIdx.x == 0 && (raw < 0 || raw > static_cast<int64_t>(a.M) * a.P))
      record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(b));
    mine += (length_of(a, b) + kTile - 1) / kTile;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) misc[4 + warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kPThreads / 32; ++w) {
    before += w < warp ? misc[4 + w] : 0;
    total += misc[4 + w];
  }
  const int W = total * HH;
  const int per = max(1, (W + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  const int64_t lo64 = static_cast<int64_t>(blockIdx.x) * per;
  const int lo = static_cast<int>(min64(lo64, W)), hi = static_cast<int>(min64(lo64 + per, W));
  // the request that holds tile `lo`
  if (lo < hi && before * HH <= lo && lo < (before + mine) * HH) {
    int cum = before;
    for (int b = rb0; b < rb1; ++b) {
      const int nt = (length_of(a, b) + kTile - 1) / kTile;
      if (lo < (cum + nt) * HH) {
        misc[1] = b;
        misc[2] = cum;
        break;
      }
      cum += nt;
    }
  }
  __syncthreads();
  Walk w;
  w.x = lo;
  w.x1 = hi;
  w.b = misc[1];
  w.h = 0;
  w.nt = 0;
  w.len = 0;
  w.t0 = 0;
  if (lo < hi) {
    w.len = length_of(a, w.b);
    w.nt = (w.len + kTile - 1) / kTile;
    const int y = lo - misc[2] * HH;
    w.h = y / w.nt;
    w.t0 = y - w.h * w.nt;
  }
  auto next_segment = [&]() {
    w.t0 = 0;
    if (++w.h < HH) return;
    w.h = 0;
    do {
      ++w.b;
      w.len = w.b < a.B ? length_of(a, w.b) : 1;
    } while (w.len == 0);
    w.nt = (w.len + kTile - 1) / kTile;
  };
  auto fail = [&](uint32_t observed) {
    if (!*abort_flag) record_local_failure(a.err, a.err_host, kErrTimeout, kStageAttn, observed);
    *abort_flag = 1;
  };

  if (warp == kConsumers) {
    // --------------------------------------------------------- producer --
    // lane -> (K or V, warp share of the tile, 64-dim column block): one TMA box each
    constexpr int kBoxes = 2 * (kTile / kBoxRows) * kHalves;
    int tile = 0, seg = 0;
    const CUtensorMap* map = lane < kBoxes / 2 ? &tk : &tv;
    const int half = lane % kHalves, box = (lane / kHalves) % (kTile / kBoxRows);
    const int64_t bad_row = static_cast<int64_t>(a.num_pages) * a.Hkv * a.P;  // past the pages: TMA fills zeros
    auto row_of = [&](int t) -> int64_t {  // first cache row of this lane's box of tile t
      const int pos = t * kTile + box * kBoxRows;
      if (lane >= kBoxes || pos >= w.len) return -1;
      const int page = __ldg(a.tables + w.b * a.table_stride + pos / a.P);
      if (page < 0 || page >= a.num_pages) {
        if (lane < kBoxes / 2 && half == 0 && w.h == 0)
          record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(page));
        return bad_row;
      }
      return (static_cast<int64_t>(page) * a.Hkv + w.h / a.HT) * a.P + pos % a.P;
    };
    while (w.x < w.x1) {
      const int n = min(w.nt - w.t0, w.x1 - w.x);
      int64_t row = row_of(w.t0);
      for (int i = 0; i < n; ++i, ++tile) {
        const int s = tile % S;
        const int64_t row_next = i + 1 < n ? row_of(w.t0 + i + 1) : -1;
        if (!*abort_flag && tile >= S && !sm100::mbar_wait(&empty[s], (tile / S - 1) & 1, a.timeout_ns, abort_flag))
          fail(tile);
        if (i == 0 && !*abort_flag && seg >= 2 &&
            !sm100::mbar_wait(&q_empty[seg & 1], (seg / 2 - 1) & 1, a.timeout_ns, abort_flag))
          fail(tile);
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        const int boxes = __popc(__ballot_sync(0xffffffffu, row >= 0));
        if (lane == 0)
          sm100::mbar_arrive_expect_tx(&full[s], boxes * kHalfBytes + (i == 0 ? C::kQBytes : 0));
        __syncwarp();
        if (i == 0 && lane < kHalves)
          tma_load_3d(paged_smem + C::kQ + (seg & 1) * C::kQBytes + half * kHalfBytes, &tq, half * 64,
                      (w.h / a.HT) * a.G + (w.h % a.HT) * a.GT, w.b, &full[s]);
        if (row >= 0)
          sm100::tma_load_2d(paged_smem + s * C::kStageBytes + lane * kHalfBytes, map, half * 64,
                             static_cast<int>(row), &full[s]);
        row = row_next;
      }
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
      w.x += n;
      ++seg;
      if (w.x < w.x1) next_segment();
    }
    // the copies in flight land before the CTA's memory goes away, whatever the consumers do
    volatile int never = 0;
    for (int i = max(0, tile - S); i < tile; ++i)
      sm100::mbar_wait(&full[i % S], (i / S) & 1, a.timeout_ns, &never);
    return;
  }

  // ------------------------------------------------------------ consumers --
  // requests without positions: their rows are zero
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (length_of(a, b) > 0) continue;
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.Hq * D);
    for (int i = tid; i < a.Hq * D / 8; i += 32 * kConsumers) o[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);

  constexpr int kNt = D / 8;           // output column tiles
  constexpr int kR = kWide ? 2 : 1;    // row halves in use
  const int g = lane >> 2, t4 = lane & 3;
  const int lr = lane & 7, lm = lane >> 3;  // ldmatrix: row within a matrix, matrix
  uint32_t qf[D / 16][4];
  int tile = 0, seg = 0;
  while (w.x < w.x1) {
    const int n = min(w.nt - w.t0, w.x1 - w.x);
    float acc[kNt][4], m[kR], l[kR];
#pragma unroll
    for (int j = 0; j < kNt; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    for (int i = 0; i < n; ++i, ++tile) {
      const int s = tile % S;
      if (!*abort_flag && !sm100::mbar_wait(&full[s], (tile / S) & 1, a.timeout_ns, abort_flag)) fail(tile);
      // the warp goes on together: a lane that gave up takes the others along
      const bool dead = __any_sync(0xffffffffu, *abort_flag != 0);
      if (!dead && i == 0) {
        // Q fragments: A rows are heads; matrices (rows 0-7 | 8-15) x (dims 0-7 | 8-15) of each 16-dim step
        const uint32_t qb = base + C::kQ + (seg & 1) * C::kQBytes;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int row = lr + (lm & 1) * 8, chunk = (k & 3) * 2 + (lm >> 1);
          ldsm4(qb + (k >> 2) * kHalfBytes + row * 128 + ((chunk ^ (row & 7)) << 4), qf[k]);
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&q_empty[seg & 1]);
      }
      const int nv = w.len - (w.t0 + i) * kTile - warp * kBoxRows;  // valid rows of this warp's box
      if (!dead && nv > 0) {
        const uint32_t kb = base + s * C::kStageBytes + warp * C::kBoxBytes;
        const uint32_t vb = kb + (kTile / kBoxRows) * C::kBoxBytes;
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          // matrices: (positions 0-7 | 8-15 by lm >> 1) x (dims 0-7 | 8-15 by lm & 1)
          const int row = lr + (lm >> 1) * 8, chunk = (k & 3) * 2 + (lm & 1);
          uint32_t kf[4];
          ldsm4(kb + (k >> 2) * kHalfBytes + row * 128 + ((chunk ^ (row & 7)) << 4), kf);
          mma16816<T>(sc[0], qf[k], kf[0], kf[1]);
          mma16816<T>(sc[1], qf[k], kf[2], kf[3]);
        }
        uint32_t pf[4];
        bool grown = false;
        float alpha[kR];
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          float v[4] = {sc[0][2 * r] * a.scale_log2, sc[0][2 * r + 1] * a.scale_log2, sc[1][2 * r] * a.scale_log2,
                        sc[1][2 * r + 1] * a.scale_log2};
          if (nv < kBoxRows) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((e >> 1) * 8 + 2 * t4 + (e & 1) >= nv) v[e] = -INFINITY;
          }
          float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[r], mx);
          grown |= mn != m[r];
          // every score -inf so far: subtract 0, so that exp(-inf) = 0 and no NaN comes from inf - inf
          const float ms = mn == -INFINITY ? 0.f : mn;
          alpha[r] = ex2(m[r] - ms);
          m[r] = mn;
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = ex2(v[e] - ms);
            sum += v[e];
          }
          l[r] = l[r] * alpha[r] + sum;
          // rounded to 16 bits for the product with V, as V itself is; the sum keeps 32
          pf[r] = pack2<T>(v[0], v[1]);
          pf[2 + r] = pack2<T>(v[2], v[3]);
        }
        if (!kWide) pf[1] = pf[3] = 0u;
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int j = 0; j < kNt; ++j) {
#pragma unroll
            for (int r = 0; r < kR; ++r) {
              acc[j][2 * r] *= alpha[r];
              acc[j][2 * r + 1] *= alpha[r];
            }
          }
        }
        // rows past the length may hold anything (NaN too): zero them in the fragments
        uint32_t mask0 = 0xffffffffu, mask1 = 0xffffffffu;
        if (nv < kBoxRows) {
          const int p0 = 2 * t4, p1 = p0 + 8;
          mask0 = (p0 < nv ? 0xffffu : 0u) | (p0 + 1 < nv ? 0xffff0000u : 0u);
          mask1 = (p1 < nv ? 0xffffu : 0u) | (p1 + 1 < nv ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          // matrices: (positions 0-7 | 8-15 by lm & 1) x (dims 0-7 | 8-15 by lm >> 1), transposed
          const int row = lr + (lm & 1) * 8, chunk = (j & 3) * 2 + (lm >> 1);
          uint32_t vf[4];
          ldsm4_t(vb + (j >> 2) * kHalfBytes + row * 128 + ((chunk ^ (row & 7)) << 4), vf);
          mma16816<T>(acc[2 * j], pf, vf[0] & mask0, vf[1] & mask1);
          mma16816<T>(acc[2 * j + 1], pf, vf[2] & mask0, vf[3] & mask1);
        }
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[s]);
    }
    // ---------------------------------------------- end of the piece --
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    // warps 2, 3 hand their part to warps 0, 1, then 1 to 0; 8 rows at a time
#pragma unroll
    for (int r = 0; r < kR; ++r) {
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        float* mo = reinterpret_cast<float*>(paged_smem + C::kMerge) + (warp & 1) * 8 * D;
        float* ml = reinterpret_cast<float*>(paged_smem + C::kMl) + (warp & 1) * 16;
        const bool gives = step == 0 ? warp >= 2 : warp == 1;
        const bool takes = step == 0 ? warp < 2 : warp == 0;
        if (step == 1 && warp == 0) {
          mo += 8 * D;
          ml += 16;
        }
        if (gives) {
#pragma unroll
          for (int j = 0; j < kNt; ++j)
            *reinterpret_cast<float2*>(mo + (j * 8 + g) * 8 + 2 * t4) = make_float2(acc[j][2 * r], acc[j][2 * r + 1]);
          if (t4 == 0) {
            ml[2 * g] = m[r];
            ml[2 * g + 1] = l[r];
          }
        }
        bar_consumers();
        if (takes) {
          const float mo_ = ml[2 * g], lo_ = ml[2 * g + 1];
          const float mn = fmaxf(m[r], mo_);
          const float ms = mn == -INFINITY ? 0.f : mn;
          const float w0 = ex2(m[r] - ms), w1 = ex2(mo_ - ms);
          m[r] = mn;
          l[r] = l[r] * w0 + lo_ * w1;
#pragma unroll
          for (int j = 0; j < kNt; ++j) {
            const float2 o = *reinterpret_cast<const float2*>(mo + (j * 8 + g) * 8 + 2 * t4);
            acc[j][2 * r] = acc[j][2 * r] * w0 + o.x * w1;
            acc[j][2 * r + 1] = acc[j][2 * r + 1] * w0 + o.y * w1;
          }
        }
        if (step == 1) bar_consumers();  // the buffers are free again
      }
    }
    if (warp == 0) {
      const bool whole = w.t0 == 0 && n == w.nt;
      const int h0 = (w.h % a.HT) * a.GT;          // first head of the tile within the group
      const int heads = min(a.GT, a.G - h0);
      const int64_t row0 = static_cast<int64_t>(w.b) * a.Hq + (w.h / a.HT) * a.G + h0;
      if (whole) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const int row = g + 8 * r;
          if (row < heads) {
            const float inv = 1.f / l[r];
            T* o = static_cast<T*>(a.out) + (row0 + row) * D + 2 * t4;
#pragma unroll
            for (int j = 0; j < kNt; ++j)
              *reinterpret_cast<uint32_t*>(o + 8 * j) = pack2<T>(acc[j][2 * r] * inv, acc[j][2 * r + 1] * inv);
          }
        }
      } else {
        // slot 2c: the piece that begins with CTA c's range; 2c + 1: one that begins inside it
        const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (w.x != lo);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const int row = g + 8 * r;
          if (row < heads) {
            float* o = a.ws_o + (part * kRows + row) * D + 2 * t4;
#pragma unroll
            for (int j = 0; j < kNt; ++j)
              *reinterpret_cast<float2*>(o + 8 * j) = make_float2(acc[j][2 * r], acc[j][2 * r + 1]);
            if (t4 == 0) a.ws_ml[part * kRows + row] = make_float2(m[r], l[r]);
          }
        }
        if (w.t0 == 0 && lane == 0) {
          const int last = static_cast<int>((static_cast<int64_t>(w.x) + w.nt - 1) / per);  // CTA of the last tile
          a.desc[blockIdx.x] = make_int4(static_cast<int>(row0), heads, last, 1 + (w.x != lo));
        }
      }
    }
    w.x += n;
    ++seg;
    if (w.x < w.x1) next_segment();
  }
}

// Joins the pieces of the segment that begins in main CTA blockIdx.x (if one
// that is cut does): o = sum_i exp(m_i - M) o_i / sum_i exp(m_i - M) l_i, in
// the order of the pieces. blockIdx.y: which of the segment's heads. The
// lanes of a group of D / 4 threads hold 4 dims each; the groups take every
// kGroups-th piece.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const __grid_constant__ PagedDev a) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 s_o[kGroups][kLanes];
  __shared__ float s_m[kGroups], s_l[kGroups];
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x;
  const int4 d = a.desc[c];
  if (d.w == 0) return;
  const int grp = threadIdx.x / kLanes, ln = threadIdx.x % kLanes;
  const int pieces = d.z - c + 1;
  for (int row = blockIdx.y; row < d.y; row += gridDim.y) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
#pragma unroll 4
    for (int i = grp; i < pieces; i += kGroups) {
      const int64_t part = 2 * static_cast<int64_t>(c + i) + (i == 0 ? d.w - 1 : 0);
      const float2 ml = a.ws_ml[part * kRows + row];
      const float4 x = *reinterpret_cast<const float4*>(a.ws_o + (part * kRows + row) * D + 4 * ln);
      const float mn = fmaxf(m, ml.x);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float w0 = ex2(m - ms), w1 = ex2(ml.x - ms);
      m = mn;
      l = l * w0 + ml.y * w1;
      o.x = o.x * w0 + x.x * w1;
      o.y = o.y * w0 + x.y * w1;
      o.z = o.z * w0 + x.z * w1;
      o.w = o.w * w0 + x.w * w1;
    }
    s_o[grp][ln] = o;
    if (ln == 0) {
      s_m[grp] = m;
      s_l[grp] = l;
    }
    __syncthreads();
    if (grp == 0) {
      float M = s_m[0];
#pragma unroll
      for (int i = 1; i < kGroups; ++i) M = fmaxf(M, s_m[i]);
      const float ms = M == -INFINITY ? 0.f : M;
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const float wgt = ex2(s_m[i] - ms);
        const float4 x = s_o[i][ln];
        den += wgt * s_l[i];
        r.x += wgt * x.x;
        r.y += wgt * x.y;
        r.z += wgt * x.z;
        r.w += wgt * x.w;
      }
      const float inv = 1.f / den;
      uint2 packed;
      packed.x = pack2<T>(r.x * inv, r.y * inv);
      packed.y = pack2<T>(r.z * inv, r.w * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (static_cast<int64_t>(d.x) + row) * D + 4 * ln) = packed;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------ host side --
using PFN_Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

CUtensorMap encode(const void* ptr, int dtype, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box) {
  static const PFN_Encode fn = driver_fn<PFN_Encode>("cuTensorMapEncodeTiled");
  CUtensorMap m;
  std::memset(&m, 0, sizeof(m));
  const cuuint32_t estr[3] = {1, 1, 1};
  NAB_CU_CHECK(fn(&m, dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                  const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
  return m;
}

// Pages as a matrix [rows, D]; a box is 16 rows of one 64-dim column block.
CUtensorMap page_map(const void* ptr, int dtype, int64_t rows, int D) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(D) * 2};
  const cuuint32_t box[2] = {64, kBoxRows};
  return encode(ptr, dtype, 2, dims, strides, box);
}

// [B][Hq][D]; a box is 16 heads of one 64-dim column block (heads past Hq read as zero).
CUtensorMap q_map(const PagedAttnArgs& a, int dtype) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.Hq),
                              static_cast<cuuint64_t>(a.B)};
  const int64_t stride = a.B == 1 ? static_cast<int64_t>(a.Hq) * a.D : a.q_stride;
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.D) * 2, static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[3] = {64, kRows, 1};
  return encode(a.q, dtype, 3, dims, strides, box);
}

struct PagedPlan {
  int HT, GT, grid;
  bool join;
};

PagedPlan plan_of(int B, int M, int P, int Hq, int Hkv, int sms) {
  PagedPlan p;
  const int G = Hq / Hkv;
  p.HT = (G + kRows - 1) / kRows;
  p.GT = (G + p.HT - 1) / p.HT;
  const int64_t tiles = (static_cast<int64_t>(M) * P + kTile - 1) / kTile;  // of the longest request
  const int64_t most = tiles * B * Hkv * p.HT;
  if (most > 0x3fffffff) throw std::invalid_argument("paged_attention: too many positions for one call");
  p.grid = static_cast<int>(std::min<int64_t>(2 * sms, std::max<int64_t>(1, most)));
  p.join = tiles > 1;  // a request of one tile is never cut
  return p;
}

// ws: [2 * grid][16][D] outputs, [2 * grid][16] (max, sum), [grid] descriptors
int64_t ws_floats(int grid, int D) { return static_cast<int64_t>(grid) * (2 * kRows * (D + 2) + 4); }

void launch(const void* kernel, dim3 grid, int block, size_t smem, cudaStream_t s, void** args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("paged_attention launch failed: ") + cudaGetErrorString(e));
}

template <typename T, int D>
void run(cudaStream_t s, const PagedAttnArgs& in, int dtype, int sms) {
  const PagedPlan p = plan_of(in.B, in.M, in.P, in.Hq, in.Hkv, sms);
  const int64_t rows = in.num_pages * in.Hkv * in.P;
  const CUtensorMap tk = page_map(in.k_pages, dtype, rows, D), tv = page_map(in.v_pages, dtype, rows, D);
  const CUtensorMap tq = q_map(in, dtype);
  const KernelErrorRecord rec = kernel_error_record();
  PagedDev a{};
  a.tables = in.tables;
  a.table_stride = in.table_stride;
  a.lengths = in.lengths;
  a.out = in.out;
  a.ws_o = in.ws;
  a.ws_ml = reinterpret_cast<float2*>(in.ws + static_cast<int64_t>(p.grid) * 2 * kRows * D);
  a.desc = reinterpret_cast<int4*>(a.ws_ml + static_cast<int64_t>(p.grid) * 2 * kRows);
  a.num_pages = static_cast<int>(in.num_pages);
  a.B = in.B;
  a.M = in.M;
  a.P = in.P;
  a.Hq = in.Hq;
  a.Hkv = in.Hkv;
  a.G = in.Hq / in.Hkv;
  a.HT = p.HT;
  a.GT = p.GT;
  a.scale_log2 = in.scale * kLog2e;
  a.err = rec.dev;
  a.err_host = rec.host;
  a.timeout_ns = kernel_timeout_ns();
  const void* kernel = p.GT > 8 ? reinterpret_cast<const void*>(&k_paged_attn<T, D, true>)
                                : reinterpret_cast<const void*>(&k_paged_attn<T, D, false>);
  static std::atomic<bool> ready[64][2];  // by device and variant; setting it twice does no harm
  int dev = 0;
  NAB_CUDA_CHECK(cudaGetDevice(&dev));
  std::atomic<bool>& set = ready[dev & 63][p.GT > 8];
  if (!set.load(std::memory_order_acquire)) {
    NAB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedCfg<D>::kSmem));
    set.store(true, std::memory_order_release);
  }
  void* args[4] = {const_cast<CUtensorMap*>(&tk), const_cast<CUtensorMap*>(&tv), const_cast<CUtensorMap*>(&tq), &a};
  launch(kernel, dim3(p.grid), kPThreads, PagedCfg<D>::kSmem, s, args);
  if (p.join) {
    void* jargs[1] = {&a};
    launch(reinterpret_cast<const void*>(&k_paged_join<T, D>), dim3(p.grid, p.GT), kJoinThreads, 0, s, jargs);
  }
}

}  // namespace

int64_t paged_attention_ws_floats(int B, int M, int P, int Hq, int Hkv, int D, int sms) {
  return ws_floats(plan_of(B, M, P, Hq, Hkv, sms).grid, D);
}

void paged_attention(cudaStream_t s, const PagedAttnArgs& a, int dtype, int sms) {
  if (dtype == kF16) {
    a.D == 64 ? run<__half, 64>(s, a, dtype, sms) : run<__half, 128>(s, a, dtype, sms);
  } else {
    a.D == 64 ? run<__nv_bfloat16, 64>(s, a, dtype, sms) : run<__nv_bfloat16, 128>(s, a, dtype, sms);
  }
}

}  // namespace nab
