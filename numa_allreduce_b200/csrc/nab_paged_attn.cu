// GQA attention of one new token per request over a paged KV cache.
//
//   o[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j,  j < lengths[b]
//
// K and V are read once, so HBM bandwidth bounds it: 4 * G * D operations per
// position and kv head (G = Hq / Hkv query heads) against 4 * D bytes, i.e. G
// operations a byte. The contractions are warp-level 16-bit MMAs (m16n8k16,
// fp32 accumulators): rows are the query heads of one kv head, so one
// operand pass serves up to 16 heads, and the probabilities stay in registers
// between the two products, as two 16-bit values each. A tcgen05 version needs them in shared memory
// and two TMEM round trips with CTA barriers per chunk (the contiguous-cache
// kernel of nab_attn_sm100.cu), a serial chain that costs more than the
// bytes of a chunk; here four warps stream independently.
//
// Work: the (request, kv head, head tile) segments, cut into tiles of 32 KB
// of K and V (64 positions of 128 dims, 128 of 64). Lengths are read on the
// device: a captured graph replays at any lengths. Three ways to deal the
// tiles out, chosen on the host from the table's width (plan_of):
//   even     all tiles laid end to end, equal contiguous ranges for a grid of
//            two CTAs per SM, so that ragged batches and single long requests
//            load the GPU alike. Each CTA finds its range by a scan over the
//            lengths. A segment within one CTA is written at once; of a cut
//            one, each CTA leaves (max, sum, unnormalised output) in fp32 and
//            a second launch joins the parts in order. (Joining in the CTA
//            that finds all parts written needs no second launch but takes
//            longer: two fences, a read of the flags and the join, 3 to 5 us
//            that hold up the CTA's next segment, against 2.7 to 4 us.)
//   whole    the same with ranges of whole segments, for short requests: no
//            part, no second launch.
//   cluster  calls bound by latency: a thread-block cluster of 1 to 8 CTAs
//            per segment, joined over distributed shared memory, without
//            scan, workspace or second launch.
//
// CTA: warp 4 fetches, warps 0-3 compute. A tile arrives as TMA boxes of 64
// dims x as many rows as the page size allows (16 to a whole tile, 128-byte
// swizzle): issuing one takes its warp about 60 cycles whatever its size (16
// boxes of 2 KB are 900 cycles, 4 of 8 KB 260). The tile that holds a
// request's end is fetched in boxes of 16 rows, no further than it goes.
// Warp w computes a quarter of each tile with its own running maximum and
// sum, so the warps meet only at the end of a segment.
//
// Every mbarrier wait is bounded. One that runs out records into the device's
// kernel error record; the warps then walk their ranges without waiting,
// fetching or computing (the same barriers), the fetching warp waits
// (bounded) for its copies in flight, and the kernel returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "nab_device.cuh"
#include "nab_driver.h"
#include "nab_kerr.h"
#include "nab_paged.h"
#include "nab_sm100.cuh"

namespace nab {

namespace {

constexpr int kBoxRows = 16;    // rows of the smallest TMA box, and of one step of a warp
constexpr int kWarps = 4;       // computing warps
constexpr int kPThreads = 32 * (kWarps + 1);
constexpr int kRows = 16;       // query heads of one head tile (the MMA's M)
constexpr int kJoinThreads = 512, kFewThreads = 128;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct PagedCfg {
  static constexpr int kTile = 8192 / D;                       // positions of a tile
  static constexpr int kSteps = kTile / kWarps / kBoxRows;     // 16-row steps of a warp's share: 1 (D = 128), 2 (D = 64)
  static constexpr int kHalves = D / 64;                       // 128-byte column blocks of a row
  static constexpr int kBlock = kTile * 128;                   // bytes of one column block of a tile
  static constexpr int kStageBytes = 2 * kHalves * kBlock;     // K blocks, then V blocks: 32 KB
  static constexpr int kStages = 3;
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
  float* ws_o;    // [2 * grid][16][D]: parts
  float2* ws_ml;  // [2 * grid][16]: their (max, sum)
  // (output row, heads, first CTA, last CTA * 2 + inside) of a cut segment, or heads = 0: of the one that begins in
  // a CTA, or with by_segment of each segment (fewer than CTAs)
  int4* desc;
  int by_segment;
  int num_pages;
  int B, M, P, Hq, Hkv;
  int G;          // query heads per kv head
  int HT, GT;     // head tiles per kv head, heads per tile
  int cluster;    // CTAs per segment (cluster form)
  int whole;      // ranges of whole segments
  int box_rows;   // rows of the large boxes
  float scale_log2;
  ErrorState* err;
  uint32_t* err_host;
  uint64_t timeout_ns;
};

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
template <typename T>
NAB_DINLINE float2 unpack2(uint32_t v);
template <>
NAB_DINLINE float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
NAB_DINLINE float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// Infinities and NaN as the largest finite value.
template <typename T>
NAB_DINLINE uint32_t finite2(uint32_t v);
template <>
NAB_DINLINE uint32_t finite2<__nv_bfloat16>(uint32_t v) {
  uint32_t r;
  asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x7f7f7f7fu));
  return r;
}
template <>
NAB_DINLINE uint32_t finite2<__half>(uint32_t v) {
  uint32_t r;
  asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x7bff7bffu));
  return r;
}
NAB_DINLINE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The probabilities relative to the maximum are held times 2^kBits, in sums and outputs alike, so it cancels. In fp16
// one below 2^-25 would be zero and one below 2^-14 lose bits, which in a long cache are many: with 2^15 (its largest
// is 65504) these become 2^-40 and 2^-29. bf16 has fp32's exponents.
template <typename T>
struct ProbShift {
  static constexpr float kBits = 0.f;
};
template <>
struct ProbShift<__half> {
  static constexpr float kBits = 15.f;
};

NAB_DINLINE int64_t min64(int64_t x, int64_t y) { return x < y ? x : y; }

NAB_DINLINE void bar_compute() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

// A walk over the segments of one CTA's range [x, x1): tiles, all segments
// end to end (even, cluster), or segments (whole).
struct Walk {
  int x, x1;
  int b, h;      // request, kv head * HT + head tile
  int nt, len;   // tiles and positions of request b
  int t;         // next tile within the segment
};

// Length of request b, within what its table row can hold.
NAB_DINLINE int length_of(const PagedDev& a, int b) {
  return static_cast<int>(min64(max(a.lengths[b], 0), static_cast<int64_t>(a.M) * a.P));
}

// kWide: more than 8 heads in a head tile. kCluster: the cluster form.
template <typename T, int D, bool kWide, bool kCluster>
__global__ void __launch_bounds__(kPThreads, 2)
    k_paged_attn(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                 const __grid_constant__ CUtensorMap tk16, const __grid_constant__ CUtensorMap tv16,
                 const __grid_constant__ CUtensorMap tq, const __grid_constant__ PagedDev a) {
  using C = PagedCfg<D>;
  constexpr int S = C::kStages;
  constexpr int kTile = C::kTile, kSteps = C::kSteps, kHalves = C::kHalves;
  constexpr int kQHalf = kRows * 128;  // one column block of a Q buffer
  extern __shared__ __align__(1024) uint8_t paged_smem[];
  const uint32_t base = sm100::smem_u32(paged_smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(paged_smem + C::kBars);
  uint64_t* empty = full + S;
  uint64_t* q_empty = empty + S;
  int* misc = reinterpret_cast<int*>(paged_smem + C::kMisc);  // abort, b, first unit of b, -, warp sums, warp maxima
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
      sm100::mbar_init(&empty[s], kWarps);
    }
    sm100::mbar_init(&q_empty[0], kWarps);
    sm100::mbar_init(&q_empty[1], kWarps);
    sm100::fence_barrier_init();
    misc[0] = 0;
    misc[1] = a.B;
    sm100::prefetch_tensormap(&tk);
    sm100::prefetch_tensormap(&tv);
    sm100::prefetch_tensormap(&tk16);
    sm100::prefetch_tensormap(&tv16);
    sm100::prefetch_tensormap(&tq);
  }
  pdl_wait();
  pdl_trigger();

  Walk w;
  int per = 1, lo = 0;  // units per CTA, first unit of this one's range
  int early = 0;        // cluster form, fetching warp: lane i's is page i of the request
  if constexpr (kCluster) {
    const int segment = static_cast<int>(blockIdx.x) / a.cluster, rank = static_cast<int>(blockIdx.x) % a.cluster;
    w.b = segment / HH;
    w.h = segment % HH;
    // loaded beside the length, which says only then which of them count (plain loads of the table: the launch before
    // may have written it while this CTA was already resident)
    if (warp == kWarps && lane < a.M) early = a.tables[w.b * a.table_stride + lane];
    const int raw = a.lengths[w.b];
    if (tid == 0 && rank == 0 && w.h == 0 && (raw < 0 || raw > static_cast<int64_t>(a.M) * a.P))
      record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(w.b));
    w.len = length_of(a, w.b);
    w.nt = (w.len + kTile - 1) / kTile;
    const int share = (w.nt + a.cluster - 1) / a.cluster;
    w.t = min(w.nt, rank * share);
    w.x = 0;
    w.x1 = min(w.nt, w.t + share) - w.t;
    __syncthreads();  // barriers initialised
  } else {
    // Scan of the requests' units (tiles, or 1 if there is any): thread i
    // holds the requests [i * per_thread, ...), then a block scan.
    const int per_thread = (a.B + kPThreads - 1) / kPThreads;
    const int rb0 = min(a.B, tid * per_thread), rb1 = min(a.B, rb0 + per_thread);
    auto units = [&](int b) {
      const int len = length_of(a, b);
      return a.whole ? (len > 0) : (len + kTile - 1) / kTile;
    };
    int mine = 0, most = 0;
    for (int b = rb0; b < rb1; ++b) {
      const int raw = a.lengths[b];
      if (blockIdx.x == 0 && (raw < 0 || raw > static_cast<int64_t>(a.M) * a.P))
        record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(b));
      const int n = units(b);
      mine += n;
      most = max(most, n);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) {
      misc[4 + warp] = incl;
      misc[4 + kPThreads / 32 + warp] = most;
    }
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kPThreads / 32; ++i) {
      before += i < warp ? misc[4 + i] : 0;
      total += misc[4 + i];
      most = max(most, misc[4 + kPThreads / 32 + i]);
    }
    const int W = total * HH;
    per = max(1, (W + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
    // A tile takes its CTA 0.55 us, a part the join 0.014 us: with p tiles per CTA the longest segment of `most`
    // tiles costs 0.55 p + 0.014 most / p, least at p = sqrt(most / 39).
    if (!a.whole) per = max(per, static_cast<int>(ceilf(sqrtf(static_cast<float>(most) * (1.f / 39.f)))));
    const int64_t lo64 = static_cast<int64_t>(blockIdx.x) * per;
    lo = static_cast<int>(min64(lo64, W));
    const int hi = static_cast<int>(min64(lo64 + per, W));
    // the request that holds unit `lo`
    if (lo < hi && before * HH <= lo && lo < (before + mine) * HH) {
      int cum = before;
      for (int b = rb0; b < rb1; ++b) {
        const int n = units(b);
        if (lo < (cum + n) * HH) {
          misc[1] = b;
          misc[2] = cum;
          break;
        }
        cum += n;
      }
    }
    __syncthreads();
    w.x = lo;
    w.x1 = hi;
    w.b = misc[1];
    w.h = 0;
    w.nt = 0;
    w.len = 0;
    w.t = 0;
    if (lo < hi) {
      w.len = length_of(a, w.b);
      w.nt = (w.len + kTile - 1) / kTile;
      const int y = lo - misc[2] * HH, n = a.whole ? 1 : w.nt;
      w.h = y / n;
      w.t = y - w.h * n;
    }
  }
  // tiles of the current segment in this range, and the step to the next one
  auto tiles_here = [&]() { return !kCluster && a.whole ? w.nt : min(w.nt - w.t, w.x1 - w.x); };
  auto advance = [&](int n) -> bool {
    w.x += !kCluster && a.whole ? 1 : n;
    if (w.x >= w.x1) return false;
    w.t = 0;
    if (++w.h < HH) return true;
    w.h = 0;
    do {
      ++w.b;
      w.len = w.b < a.B ? length_of(a, w.b) : 1;
    } while (w.len == 0);
    w.nt = (w.len + kTile - 1) / kTile;
    return true;
  };
  auto fail = [&](uint32_t observed) {
    if (!*abort_flag) record_local_failure(a.err, a.err_host, kErrTimeout, kStageAttn, observed);
    *abort_flag = 1;
  };

  if (warp == kWarps) {
    // -------------------------------------------------------- fetching --
    // Lane -> one box of a tile: (K or V, column block, run of rows).
    int tile = 0, seg = 0;
    // lane i holds the id of page window + i of request w.b, and of page i of request w.b + 1, loaded when the walk
    // comes to w.b so that the next request starts without a wait
    int window = 0, ids = 0, ahead = 0;
    auto load_ids = [&](int b, int first) {
      return b < a.B && first + lane < a.M ? a.tables[b * a.table_stride + first + lane] : 0;
    };
    bool more = w.x < w.x1, given_up = false;
    if (more) {
      if constexpr (kCluster) {
        ids = early;
      } else {
        window = static_cast<int>(static_cast<int64_t>(w.t) * kTile / a.P);
        ids = load_ids(w.b, window);
        ahead = load_ids(w.b + 1, 0);
      }
    }
    while (more) {
      const int n = tiles_here();
      const int kvh = w.h / a.HT;
      for (int i = 0; i < n; ++i, ++tile) {
        const int s = tile % S;
        const int left = w.len - (w.t + i) * kTile;  // positions from this tile on
        const bool small = left < kTile;
        const int rows = small ? kBoxRows : a.box_rows;
        const int per_block = kTile / rows;          // boxes of a column block
        const int v = lane / (kHalves * per_block), half = lane / per_block % kHalves, from = lane % per_block * rows;
        const bool mine = v < 2 && from < left;
        const int pos = (w.t + i) * kTile + (mine ? from : 0);
        const int page_at = pos / a.P, first = (w.t + i) * kTile / a.P;
        if (first < window || first + kTile / kBoxRows > window + 32) {  // a tile has at most kTile / 16 pages
          window = first;
          ids = load_ids(w.b, window);
        }
        const int page = __shfl_sync(0xffffffffu, ids, page_at - window);
        int64_t row = (static_cast<int64_t>(page) * a.Hkv + kvh) * a.P + (pos - page_at * a.P);
        if (page < 0 || page >= a.num_pages) {
          if (mine && v == 0 && half == 0 && w.h == 0)
            record_local_failure(a.err, a.err_host, kErrBadLaunch, kStageBounds, static_cast<uint32_t>(page));
          row = static_cast<int64_t>(a.num_pages) * a.Hkv * a.P;  // past the pages: TMA fills zeros
        }
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
        bool ok = tile < S || sm100::mbar_wait(&empty[s], (tile / S - 1) & 1, a.timeout_ns, abort_flag);
        if (ok && i == 0 && seg >= 2) ok = sm100::mbar_wait(&q_empty[seg & 1], (seg / 2 - 1) & 1, a.timeout_ns, abort_flag);
        if (!ok) fail(tile);
        if (__any_sync(0xffffffffu, !ok)) {
          given_up = true;
          break;
        }
        if (lane == 0) sm100::mbar_arrive_expect_tx(&full[s], boxes * rows * 128 + (i == 0 ? C::kQBytes : 0));
        __syncwarp();
        if (i == 0 && lane < kHalves)
          tma_load_3d(paged_smem + C::kQ + (seg & 1) * C::kQBytes + lane * kQHalf, &tq, lane * 64,
                      kvh * a.G + (w.h % a.HT) * a.GT, w.b, &full[s]);
        if (mine)
          sm100::tma_load_2d(paged_smem + s * C::kStageBytes + (v * kHalves + half) * C::kBlock + from * 128,
                             small ? (v ? &tv16 : &tk16) : (v ? &tv : &tk), half * 64, static_cast<int>(row), &full[s]);
      }
      if (given_up) break;
      ++seg;
      const int b = w.b;
      more = advance(n);
      if (more && w.b != b) {
        ids = w.b == b + 1 ? ahead : load_ids(w.b, 0);
        window = 0;
        ahead = load_ids(w.b + 1, 0);
      }
    }
    // the copies in flight land before the CTA's memory goes away, whatever the other warps do
    volatile int never = 0;
    for (int i = max(0, tile - S); i < tile; ++i)
      sm100::mbar_wait(&full[i % S], (i / S) & 1, a.timeout_ns, &never);
    if constexpr (kCluster) {
      if (a.cluster > 1) {
        sm100::cluster_sync();  // the parts are in shared memory
        sm100::cluster_sync();  // and have been read
      }
    }
    return;
  }

  // ----------------------------------------------------------- computing --
  if constexpr (!kCluster) {
    // requests without positions: their rows are zero
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      if (length_of(a, b) > 0) continue;
      uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.Hq * D);
      for (int i = tid; i < a.Hq * D / 8; i += 32 * kWarps) o[i] = make_uint4(0u, 0u, 0u, 0u);
      if (a.by_segment)
        for (int i = tid; i < HH; i += 32 * kWarps) a.desc[b * HH + i] = make_int4(0, 0, 0, 0);
    }
    if (tid == 0 && !a.whole && !a.by_segment) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
  }

  constexpr int kNt = D / 8;           // output column tiles
  constexpr int kR = kWide ? 2 : 1;    // row halves in use
  const int g = lane >> 2, t4 = lane & 3;
  const int lr = lane & 7, lm = lane >> 3;  // ldmatrix: row within a matrix, matrix
  // Byte offsets of this lane's ldmatrix rows within a 16-row step, for column chunk 0 (16-byte chunks permuted by
  // row % 8); column step j is 32 bytes on, i.e. XOR j << 5.
  const uint32_t k_off = (warp * kSteps * kBoxRows + lr + (lm >> 1) * 8) * 128 + (((lm & 1) ^ lr) << 4);
  const uint32_t v_off = (warp * kSteps * kBoxRows + lr + (lm & 1) * 8) * 128 + (((lm >> 1) ^ lr) << 4);
  // Q fragments: per 16-dim step rows 0-7 and 8-15, or (up to 8 heads) of two steps rows 0-7
  uint32_t qf[kWide ? D / 16 : D / 32][4];
  int tile = 0, seg = 0;
  bool dead = false;
  // a segment's running maximum, sum and output of this warp's positions
  float acc[kNt][4], m[kR], l[kR];

  // One tile's share: nv valid rows, all of them unless kTail.
  auto compute = [&](uint32_t stage, int nv, auto tail) {
    constexpr bool kTail = decltype(tail)::value;
    const uint32_t kb = stage + k_off, vb = stage + C::kStageBytes / 2 + v_off;
    // scores: two chains of products per 8 positions (even and odd 16-dim steps) while there is one step of rows
    constexpr int kChains = kSteps == 1 ? 2 : 1;
    float sc[2 * kSteps][4], odd[2][4];
#pragma unroll
    for (int j = 0; j < 2 * kSteps; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) odd[j][0] = odd[j][1] = odd[j][2] = odd[j][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t q4[4] = {kWide ? qf[k][0] : qf[k >> 1][2 * (k & 1)], kWide ? qf[k][1] : 0u,
                              kWide ? qf[k][2] : qf[k >> 1][2 * (k & 1) + 1], kWide ? qf[k][3] : 0u};
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
        // matrices: (positions 0-7 | 8-15 by lm >> 1) x (dims 0-7 | 8-15 by lm & 1)
        uint32_t kf[4];
        ldsm4((kb ^ ((k & 3) << 5)) + (k >> 2) * C::kBlock + x * kBoxRows * 128, kf);
        if (kChains == 2 && (k & 1)) {
          mma16816<T>(odd[0], q4, kf[0], kf[1]);
          mma16816<T>(odd[1], q4, kf[2], kf[3]);
        } else {
          mma16816<T>(sc[2 * x], q4, kf[0], kf[1]);
          mma16816<T>(sc[2 * x + 1], q4, kf[2], kf[3]);
        }
      }
    }
    if (kChains == 2) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] += odd[j][e];
      }
    }
    uint32_t pf[kSteps][4], pl[kSteps][4];
    bool grown = false;
    float alpha[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      float v[4 * kSteps];
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4 * kSteps; ++e) {
        v[e] = sc[e >> 1][2 * r + (e & 1)] * a.scale_log2;
        if (kTail && (e >> 1) * 8 + 2 * t4 + (e & 1) >= nv) v[e] = -INFINITY;
        mx = fmaxf(mx, v[e]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[r], mx);
      grown |= mn != m[r] && m[r] != -INFINITY;  // (nothing to scale before the first score)
      // every score -inf so far: subtract 0, so that exp(-inf) = 0 and no NaN comes from inf - inf
      const float ms = mn == -INFINITY ? 0.f : mn;
      alpha[r] = ex2(m[r] - ms);
      m[r] = mn;
      const float base_exp = ms - ProbShift<T>::kBits;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4 * kSteps; ++e) {
        v[e] = ex2(v[e] - base_exp);
        sum += v[e];
      }
      l[r] = l[r] * alpha[r] + sum;
      // For the product with V a probability is the sum of two 16-bit values, its rounding and what that left out: off
      // by 2^-16 of it in bf16 and 2^-22 in fp16, where the rounding alone is 2^-8 and 2^-11. (The second value's sign
      // may differ: a product of it with an infinity must not join the first's.) One value against two (us):
      // up to 8 heads 64 requests of up to 8192 171.4 / 172.2, 640 of up to 256 19.4 / 19.9, 1 of 1025 5.95 / 6.0; 16
      // heads 175.8 / 177.2, 32 of up to 2500 36.8 / 38.5, 1 of 1025 6.9 / 7.5.
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float lo = v[4 * x + 2 * i], hi = v[4 * x + 2 * i + 1];
          const uint32_t p = pack2<T>(lo, hi);
          const float2 back = unpack2<T>(p);
          pf[x][2 * i + r] = p;
          pl[x][2 * i + r] = pack2<T>(lo - back.x, hi - back.y);
        }
      }
    }
    if (!kWide) {
      // up to 8 heads: the second values take the rows of the product that are free
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
        pf[x][1] = pl[x][0];
        pf[x][3] = pl[x][2];
      }
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int j = 0; j < kNt; ++j) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          acc[j][2 * r] *= alpha[kWide ? r : 0];
          acc[j][2 * r + 1] *= alpha[kWide ? r : 0];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      // rows past the length may hold anything (NaN too): zero them in the fragments
      const int p0 = x * kBoxRows + 2 * t4, p1 = p0 + 8;
      const uint32_t mask0 = (p0 < nv ? 0xffffu : 0u) | (p0 + 1 < nv ? 0xffff0000u : 0u);
      const uint32_t mask1 = (p1 < nv ? 0xffffu : 0u) | (p1 + 1 < nv ? 0xffff0000u : 0u);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        // matrices: (positions 0-7 | 8-15 by lm & 1) x (dims 0-7 | 8-15 by lm >> 1), transposed
        uint32_t vf[4];
        ldsm4_t((vb ^ ((j & 3) << 5)) + (j >> 2) * C::kBlock + x * kBoxRows * 128, vf);
        if (kTail) {
          vf[0] &= mask0;
          vf[1] &= mask1;
          vf[2] &= mask0;
          vf[3] &= mask1;
        }
        mma16816<T>(acc[2 * j], pf[x], vf[0], vf[1]);
        mma16816<T>(acc[2 * j + 1], pf[x], vf[2], vf[3]);
        if (kWide) {
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[i] = finite2<T>(vf[i]);
          mma16816<T>(acc[2 * j], pl[x], vf[0], vf[1]);
          mma16816<T>(acc[2 * j + 1], pl[x], vf[2], vf[3]);
        }
      }
    }
  };

  for (bool more = w.x < w.x1; more;) {
    const int n = tiles_here(), t0 = w.t;
#pragma unroll
    for (int j = 0; j < kNt; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    for (int i = 0; i < n; ++i, ++tile) {
      const int s = tile % S;
      // a lane that gave up takes the others along; once dead, the warp only keeps the barriers
      if (!dead) {
        const bool ok = sm100::mbar_wait(&full[s], (tile / S) & 1, a.timeout_ns, abort_flag);
        if (!ok) fail(tile);
        dead = __any_sync(0xffffffffu, !ok);
      }
      if (!dead) {
        if (i == 0) {
          // A rows are heads; matrices, by lm: (rows 0-7 | 8-15) x (dims 0-7 | 8-15) of a step, or (rows 0-7) x
          // (dims 0-7 | 8-15) of two steps
          const uint32_t qb = base + C::kQ + (seg & 1) * C::kQBytes;
#pragma unroll
          for (int k = 0; k < (kWide ? D / 16 : D / 32); ++k) {
            const int step = kWide ? k : 2 * k + (lm >> 1);
            const int row = kWide ? lr + (lm & 1) * 8 : lr, chunk = (step & 3) * 2 + (kWide ? lm >> 1 : lm & 1);
            ldsm4(qb + (step >> 2) * kQHalf + row * 128 + ((chunk ^ lr) << 4), qf[k]);
          }
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&q_empty[seg & 1]);
        }
        const int nv = w.len - (t0 + i) * kTile - warp * kSteps * kBoxRows;  // valid rows of this warp's share
        if (nv >= kSteps * kBoxRows) {
          compute(base + s * C::kStageBytes, nv, std::false_type{});
        } else if (nv > 0) {
          compute(base + s * C::kStageBytes, nv, std::true_type{});
        }
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[s]);
    }
    // ---------------------------------------------- end of the piece --
    if (!kWide) {  // the probabilities' second values; an infinity of V stays what the first ones made of it
#pragma unroll
      for (int j = 0; j < kNt; ++j) {
        if (fabsf(acc[j][0]) < INFINITY) acc[j][0] += acc[j][2];
        if (fabsf(acc[j][1]) < INFINITY) acc[j][1] += acc[j][3];
      }
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    // Warps 2, 3 hand their part to warps 0, 1, then 1 to 0; 8 rows at a time. A short piece has not given all of
    // them rows.
    const int active = n > 1 ? kWarps : min(kWarps, (w.len - t0 * kTile + kSteps * kBoxRows - 1) / (kSteps * kBoxRows));
    auto give = [&](int r, int buffer) {
      float* mo = reinterpret_cast<float*>(paged_smem + C::kMerge) + buffer * 8 * D;
      float* ml = reinterpret_cast<float*>(paged_smem + C::kMl) + buffer * 16;
#pragma unroll
      for (int j = 0; j < kNt; ++j)
        *reinterpret_cast<float2*>(mo + (j * 8 + g) * 8 + 2 * t4) = make_float2(acc[j][2 * r], acc[j][2 * r + 1]);
      if (t4 == 0) {
        ml[2 * g] = m[r];
        ml[2 * g + 1] = l[r];
      }
    };
    auto take = [&](int r, int buffer) {
      const float* mo = reinterpret_cast<const float*>(paged_smem + C::kMerge) + buffer * 8 * D;
      const float* ml = reinterpret_cast<const float*>(paged_smem + C::kMl) + buffer * 16;
      const float m1 = ml[2 * g], l1 = ml[2 * g + 1];
      const float mn = fmaxf(m[r], m1);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float w0 = ex2(m[r] - ms), w1 = ex2(m1 - ms);
      m[r] = mn;
      l[r] = l[r] * w0 + l1 * w1;
#pragma unroll
      for (int j = 0; j < kNt; ++j) {
        const float2 o = *reinterpret_cast<const float2*>(mo + (j * 8 + g) * 8 + 2 * t4);
        acc[j][2 * r] = acc[j][2 * r] * w0 + o.x * w1;
        acc[j][2 * r + 1] = acc[j][2 * r + 1] * w0 + o.y * w1;
      }
    };
    if (active > 1) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        bar_compute();  // the buffers have been read
        if (active > 2) {
          if (warp >= 2) give(r, warp & 1);
          bar_compute();
          if (warp < 2) take(r, warp);
        }
        __syncwarp();  // warp 1 overwrites the (max, sum) that its lanes have just read
        if (warp == 1) give(r, 1);
        bar_compute();
        if (warp == 0) take(r, 1);
      }
    }
    const int h0 = (w.h % a.HT) * a.GT;  // first head of the tile within the group
    const int heads = min(a.GT, a.G - h0);
    const int64_t row0 = static_cast<int64_t>(w.b) * a.Hq + (w.h / a.HT) * a.G + h0;
    if (kCluster && a.cluster > 1) {
      // this CTA's part, for the cluster: [16][D] floats, then 16 x (max, sum), where the ring was
      if (warp == 0) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const int row = g + 8 * r;
          float* o = reinterpret_cast<float*>(paged_smem) + row * D + 2 * t4;
#pragma unroll
          for (int j = 0; j < kNt; ++j)
            *reinterpret_cast<float2*>(o + 8 * j) = make_float2(acc[j][2 * r], acc[j][2 * r + 1]);
          if (t4 == 0) reinterpret_cast<float2*>(paged_smem + kRows * D * 4)[row] = make_float2(m[r], l[r]);
        }
      }
    } else if (warp == 0) {
      if (t0 == 0 && n == w.nt) {
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
      }
      if (lane == 0 && t0 == 0 && !a.whole && (n < w.nt || a.by_segment)) {
        const int last = (w.x + w.nt - 1) / per;  // CTA of the last tile
        a.desc[a.by_segment ? w.b * HH + w.h : blockIdx.x] =
            make_int4(static_cast<int>(row0), n < w.nt ? heads : 0, blockIdx.x, 2 * last + (w.x != lo));
      }
    }
    ++seg;
    more = advance(n);
  }
  if constexpr (kCluster) {
    if (a.cluster == 1) {
      if (seg == 0) {  // a request without positions: zeros
        const int h0 = (w.h % a.HT) * a.GT, heads = min(a.GT, a.G - h0);
        uint2* o = reinterpret_cast<uint2*>(static_cast<T*>(a.out) +
                                            (static_cast<int64_t>(w.b) * a.Hq + (w.h / a.HT) * a.G + h0) * D);
        for (int i = tid; i < heads * (D / 4); i += 32 * kWarps) o[i] = make_uint2(0u, 0u);
      }
      return;
    }
    if (seg == 0 && tid < kRows)  // no tile for this CTA: a part of weight 0
      reinterpret_cast<float2*>(paged_smem + kRows * D * 4)[tid] = make_float2(-INFINITY, 0.f);
    sm100::cluster_sync();
    const int h0 = (w.h % a.HT) * a.GT, heads = min(a.GT, a.G - h0);
    const int rank = static_cast<int>(blockIdx.x) % a.cluster;
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(w.b) * a.Hq + (w.h / a.HT) * a.G + h0) * D;
    // the cluster's CTAs share the output in runs of 4 dims; parts in rank order
    for (int i = rank * 32 * kWarps + tid; i < heads * (D / 4); i += a.cluster * 32 * kWarps) {
      const uint32_t ml_at = base + kRows * D * 4 + i / (D / 4) * 8, o_at = base + i * 16;
      float2 ml[kMaxCluster];
      float4 x[kMaxCluster];
      float M = -INFINITY;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        const int from = min(c, a.cluster - 1);
        const uint32_t at = sm100::dsmem_addr(ml_at, from);
        ml[c] = make_float2(sm100::ld_dsmem_f32(at), sm100::ld_dsmem_f32(at + 4));
        x[c] = sm100::ld_dsmem_f4(sm100::dsmem_addr(o_at, from));
        M = fmaxf(M, ml[c].x);
      }
      const float ms = M == -INFINITY ? 0.f : M;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        // a part without tiles has nothing stored but its (max, sum)
        if (c >= a.cluster || (ml[c].x == -INFINITY && ml[c].y == 0.f)) continue;
        const float wgt = ex2(ml[c].x - ms);
        den += wgt * ml[c].y;
        o.x += wgt * x[c].x;
        o.y += wgt * x[c].y;
        o.z += wgt * x[c].z;
        o.w += wgt * x[c].w;
      }
      const float inv = w.len == 0 ? 0.f : 1.f / den;  // a request without positions: zeros
      uint2 packed;
      packed.x = pack2<T>(o.x * inv, o.y * inv);
      packed.y = pack2<T>(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(out + static_cast<int64_t>(i) * 4) = packed;
    }
    sm100::cluster_sync();  // the others' shared memory has been read
  }
}

// Joins the parts of cut segment desc[blockIdx.x], in order: o = sum_i exp(m_i - M) o_i / sum_i exp(m_i - M) l_i. Two
// forms:
//   few   a thread per 4 dims of a head, the parts one after the other with 8
//         loads in flight, for many heads and few parts;
//   many  blockIdx.y takes a head, groups of D / 4 threads every n-th part.
// Time that the join adds to the main kernel (us, few / many): 64 requests of
// up to 8192, 8 heads of 128 dims 4.0 / 15.6; 32 of up to 2500, 16 heads 2.7 /
// 16, 4 heads 2.9 / 5.6; 37 parts of 4 heads of 64 dims 7.5 / 3.2; 86 parts of
// 8 heads of 128 dims 10.4 / 2.9.
template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads) k_paged_join_few(const __grid_constant__ PagedDev a) {
  constexpr int kAhead = 8;
  pdl_wait();
  pdl_trigger();
  const int at = blockIdx.y * kFewThreads + threadIdx.x;
  const int4 d = a.desc[blockIdx.x];
  const int row = at / (D / 4), col = at % (D / 4) * 4;
  if (row >= d.y) return;
  const int c = d.z, count = (d.w >> 1) - c + 1;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  for (int i0 = 0; i0 < count; i0 += kAhead) {
    float2 ml[kAhead];
    float4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i < count) {
        const int64_t part = 2 * static_cast<int64_t>(c + i0 + i) + (i0 + i == 0 ? d.w & 1 : 0);
        ml[i] = a.ws_ml[part * kRows + row];
        x[i] = *reinterpret_cast<const float4*>(a.ws_o + (part * kRows + row) * D + col);
      }
    }
    float mn = M;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) mn = fmaxf(mn, ml[i].x);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float keep = ex2(M - ms);
    M = mn;
    L *= keep;
    o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float wgt = ex2(ml[i].x - ms);
      L += ml[i].y * wgt;
      o.x += x[i].x * wgt;
      o.y += x[i].y * wgt;
      o.z += x[i].z * wgt;
      o.w += x[i].w * wgt;
    }
  }
  const float inv = 1.f / L;
  uint2 packed;
  packed.x = pack2<T>(o.x * inv, o.y * inv);
  packed.y = pack2<T>(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (static_cast<int64_t>(d.x) + row) * D + col) = packed;
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const __grid_constant__ PagedDev a) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 s_o[kGroups][kLanes];
  __shared__ float s_m[kGroups], s_l[kGroups];
  pdl_wait();
  pdl_trigger();
  const int4 d = a.desc[blockIdx.x];
  const int grp = threadIdx.x / kLanes, ln = threadIdx.x % kLanes;
  const int c = d.z, pieces = (d.w >> 1) - c + 1;
  for (int row = blockIdx.y; row < d.y; row += gridDim.y) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
#pragma unroll 4
    for (int i = grp; i < pieces; i += kGroups) {
      const int64_t part = 2 * static_cast<int64_t>(c + i) + (i == 0 ? d.w & 1 : 0);
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

// Pages as a matrix [rows, D]; a box is some rows of one 64-dim column block.
CUtensorMap page_map(const void* ptr, int dtype, int64_t rows, int D, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(D) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
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
  int cluster;   // CTAs per segment in the cluster form, 0 for the others
  bool whole;    // ranges of whole segments
  bool few;      // which form of the join
  int descs;     // segments that it may have to join
  int box_rows;
};

PagedPlan plan_of(int B, int M, int P, int Hq, int Hkv, int D, int sms) {
  PagedPlan p;
  const int G = Hq / Hkv;
  p.HT = (G + kRows - 1) / kRows;
  p.GT = (G + p.HT - 1) / p.HT;
  const int tile = 8192 / D;
  const int64_t tiles = std::max<int64_t>(1, (static_cast<int64_t>(M) * P + tile - 1) / tile);  // of the longest request
  const int64_t segments = static_cast<int64_t>(B) * Hkv * p.HT, slots = 2 * sms;
  if (tiles * segments > 0x3fffffff)
    throw std::invalid_argument("paged_attention: too many positions for one call");
  // The cluster form takes ceil(tiles / c) tiles one after the other, the even one ceil(tiles * segments / slots) and
  // about three more for its second launch. Measured (us, cluster / even; 8 heads per kv head, D = 128): 1 request of
  // 1025 6.0 / 7.1, of 4096 9.9 / 7.6; 32 of 2500 12.1 / 14.0, of 1 to 2500 9.7 / 12.2; 128 of 1025 16.8 / 19.1. The
  // bound of 10 tiles keeps ragged batches, where the longest request decides, from losing more than that.
  int c = 1;
  while (c < kMaxCluster && 2 * c <= tiles && segments * c * 2 <= slots) c *= 2;
  const int64_t share = (tiles + c - 1) / c, even = (tiles * segments + slots - 1) / slots;
  p.cluster = segments * c <= slots && share <= std::min<int64_t>(10, even + 3) ? c : 0;
  // Short requests are not worth a cut: up to 4 tiles of imbalance against the second launch (whole / even: 640 of up
  // to 256 positions in pages of 64 16.7 / 17.2 us, in pages of 16, whose boxes take longer to issue, 19.3 / 17.1; 160
  // of up to 5 with 4 kv heads 7.3 / 8.5).
  p.whole = !p.cluster && tiles <= 4;
  p.grid = static_cast<int>(p.cluster ? segments * c : std::min<int64_t>(slots, p.whole ? segments : tiles * segments));
  // parts of a segment when all requests are of one length: grid / segments and two ends
  p.descs = static_cast<int>(std::min<int64_t>(segments, p.grid));
  p.few = p.grid / segments + 2 <= 8 && p.GT * D >= 4 * kFewThreads;
  p.box_rows = tile;
  while (P % p.box_rows != 0) p.box_rows /= 2;  // P is a multiple of 16
  return p;
}

// ws: [2 * grid][16][D] outputs, [2 * grid][16] (max, sum), [grid] descriptors: for the even form alone
int64_t ws_floats(const PagedPlan& p, int D) {
  return p.cluster || p.whole ? 0 : static_cast<int64_t>(p.grid) * (2 * kRows * (D + 2) + 4);
}

void launch(const void* kernel, dim3 grid, int block, size_t smem, int cluster, cudaStream_t s, void** args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("paged_attention launch failed: ") + cudaGetErrorString(e));
}

template <typename T, int D>
void run(cudaStream_t s, const PagedAttnArgs& in, int dtype, int sms) {
  const PagedPlan p = plan_of(in.B, in.M, in.P, in.Hq, in.Hkv, D, sms);
  const int64_t rows = in.num_pages * in.Hkv * in.P;
  const CUtensorMap tk16 = page_map(in.k_pages, dtype, rows, D, kBoxRows);
  const CUtensorMap tv16 = page_map(in.v_pages, dtype, rows, D, kBoxRows);
  const CUtensorMap tk = p.box_rows == kBoxRows ? tk16 : page_map(in.k_pages, dtype, rows, D, p.box_rows);
  const CUtensorMap tv = p.box_rows == kBoxRows ? tv16 : page_map(in.v_pages, dtype, rows, D, p.box_rows);
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
  a.cluster = p.cluster;
  a.whole = p.whole;
  a.by_segment = !p.cluster && !p.whole && p.descs < p.grid;
  a.box_rows = p.box_rows;
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
  const bool wide = p.GT > 8;
  const void* kernel = p.cluster ? (wide ? reinterpret_cast<const void*>(&k_paged_attn<T, D, true, true>)
                                         : reinterpret_cast<const void*>(&k_paged_attn<T, D, false, true>))
                                 : (wide ? reinterpret_cast<const void*>(&k_paged_attn<T, D, true, false>)
                                         : reinterpret_cast<const void*>(&k_paged_attn<T, D, false, false>));
  static std::atomic<bool> ready[64][4];  // by device and variant; setting it twice does no harm
  int dev = 0;
  NAB_CUDA_CHECK(cudaGetDevice(&dev));
  std::atomic<bool>& set = ready[dev & 63][2 * (p.cluster > 0) + wide];
  if (!set.load(std::memory_order_acquire)) {
    NAB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedCfg<D>::kSmem));
    set.store(true, std::memory_order_release);
  }
  void* args[6] = {const_cast<CUtensorMap*>(&tk),   const_cast<CUtensorMap*>(&tv), const_cast<CUtensorMap*>(&tk16),
                   const_cast<CUtensorMap*>(&tv16), const_cast<CUtensorMap*>(&tq), &a};
  launch(kernel, dim3(p.grid), kPThreads, PagedCfg<D>::kSmem, p.cluster, s, args);
  if (!p.cluster && !p.whole) {
    void* join_args[1] = {&a};
    if (p.few) {
      launch(reinterpret_cast<const void*>(&k_paged_join_few<T, D>),
             dim3(p.descs, (p.GT * (D / 4) + kFewThreads - 1) / kFewThreads), kFewThreads, 0, 0, s, join_args);
    } else {
      launch(reinterpret_cast<const void*>(&k_paged_join<T, D>), dim3(p.descs, p.GT), kJoinThreads, 0, 0, s, join_args);
    }
  }
}

}  // namespace

int64_t paged_attention_ws_floats(int B, int M, int P, int Hq, int Hkv, int D, int sms) {
  return ws_floats(plan_of(B, M, P, Hq, Hkv, D, sms), D);
}

void paged_attention(cudaStream_t s, const PagedAttnArgs& a, int dtype, int sms) {
  if (dtype == kF16) {
    a.D == 64 ? run<__half, 64>(s, a, dtype, sms) : run<__half, 128>(s, a, dtype, sms);
  } else {
    a.D == 64 ? run<__nv_bfloat16, 64>(s, a, dtype, sms) : run<__nv_bfloat16, 128>(s, a, dtype, sms);
  }
}

}  // namespace nab
