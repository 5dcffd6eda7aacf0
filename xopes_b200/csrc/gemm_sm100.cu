// The matrix products of linear_fn and gated_linear_fn on tcgen05: 16-bit operands, fp32 accumulation in tensor
// memory, and the epilogue of linear.cuh on the way out.
//
//   C[m][n] = sum over segments s, k of A_s(m, k) B_s(n, k)
//
// A pair of CTAs works on a tile of 256 rows x BN columns (cta_group::2: each CTA stages its 128 rows of A and half
// the columns of B, so an SM moves 24 or 32 KB through shared memory for every 64 steps of the contraction where one CTA
// alone would move 48 for the same products).  The operands arrive by TMA, as they lie in memory: the contraction next
// to each other (x, W, dz in a row) or the rows next to each other (W in dx = dz W, dz and x in dW = dz^T x), which the
// shared-memory descriptors and the instruction take either way; nothing is transposed.  The gated pair is one
// product: the first CTA of the pair stages rows of Wg, the second the same rows of Wu, so that a tile's columns are
// BN/2 of g and the same BN/2 of u, and both meet in the epilogue's registers.  dx of a pair is one accumulation over two
// segments, dg Wg and du Wu.
//
// Warps: 0 loads, 1 multiplies (one elected lane of the first CTA for both), 2 owns tensor memory, 4..11 write.  Two
// accumulators: while one tile is written the next is multiplied.  Persistent: one pair of CTAs per two SMs, tiles in
// groups of 8 rows of tiles, so that the operands of the tiles in flight stay in L2.  Where there are fewer tiles than
// SMs the contraction is split over several units, whose fp32 sums another kernel adds in a fixed order (gemm_plan).
//
// Every wait is bounded (mbar_wait); one that runs out ends the kernel with the device's status word set.
#include "linear.cuh"
#include "sm100_ptx.cuh"
#include "tile_common.cuh"

namespace la {
namespace lin {
namespace {

using namespace la::ptx;

constexpr int kRows = 256;                 // rows of a tile, 128 of each CTA
constexpr int kStepK = 64;                 // contraction steps of a stage: 128 bytes
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr uint32_t kABytes = 128 * 128;    // 128 rows of 128 bytes
constexpr int kGroup = 8;                  // rows of tiles walked together
constexpr uint32_t kGroupBytes = 64 * 128; // 64 rows of an operand whose rows lie next to each other, 64 steps

template <int BN> struct Cfg {
  static constexpr uint32_t kBBytes = BN / 2 * 128;
  static constexpr uint32_t kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr uint32_t kSmem = 1024 + kStages * kStage + 512;
  static constexpr uint32_t kCols = 2 * BN;  // tensor memory: two accumulators
};

struct GemmArgs {
  CUtensorMap a[2], b[2];
  Epilogue e;
  float *partial;
  int *status;
  int M, N;
  int kb[2];                 // stages of each segment
  int m_tiles, n_tiles, splits;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same barrier in the first CTA of the pair
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, 0;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n\t}" ::"r"(bar) : "memory");
}
// a box into this CTA's shared memory; the bytes count on the first CTA's barrier (bit 24 of a shared-memory address is
// the CTA's place in the pair)
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & 0xFEFFFFFFu), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void mma_two(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// the barrier at this address in both CTAs arrives once all products issued so far are done
__device__ __forceinline__ void commit_two(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"((uint16_t)3)
      : "memory");
}

// mbar_wait with one answer for the whole warp (a lane may find that its own time has run out)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}

struct Unit {
  int m0, n0, k0, k1, split;
};
template <int BN, bool PAIR>
__device__ __forceinline__ Unit unit_of(const GemmArgs &g, int u) {
  const int tile = u / g.splits, split = u - tile * g.splits;
  const int per = kGroup * g.n_tiles, group = tile / per, first = group * kGroup;
  const int rows = min(g.m_tiles - first, kGroup), r = tile - group * per;
  Unit x;
  x.m0 = (first + r % rows) * kRows;
  x.n0 = r / rows * (PAIR ? BN / 2 : BN);
  const long long all = g.kb[0] + g.kb[1];
  x.k0 = (int)(all * split / g.splits);
  x.k1 = (int)(all * (split + 1) / g.splits);
  x.split = split;
  return x;
}

template <typename T, bool A_MN, bool B_MN, int BN, bool PAIR>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs g) {
  typedef Cfg<BN> C;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t bars = base + C::kStages * C::kStage;
  const uint32_t full = bars, empty = full + 8 * C::kStages, tfull = empty + 8 * C::kStages, tempty = tfull + 16;
  const uint32_t tmem_at = tempty + 16;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(raw + (tmem_at + 4 - smem_u32(raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int units = g.m_tiles * g.n_tiles * g.splits;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull + 8 * s, 1);
      mbar_init(tempty + 8 * s, 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_at), "r"(C::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(raw + (tmem_at - smem_u32(raw)));

  if (warp == 0) {
    // ------------------------------------------------------------ loads, in both CTAs
    if (lane == 0) {
      prefetch_tmap(&g.a[0]);
      prefetch_tmap(&g.b[PAIR ? rank : 0]);
    }
    int it = 0;
    bool ok = true;
    for (int u = first; u < units && ok; u += stride) {
      const Unit x = unit_of<BN, PAIR>(g, u);
      const int am = x.m0 + (int)rank * 128, bn = PAIR ? x.n0 : x.n0 + (int)rank * (BN / 2);
      for (int kb = x.k0; kb < x.k1; ++kb, ++it) {
        const int s = it % C::kStages;
        if (!warp_wait(empty + 8 * s, ((it / C::kStages) & 1) ^ 1, abort_flag, g.status, 301)) {
          ok = false;
          break;
        }
        const int seg = kb >= g.kb[0];
        const int k = (seg ? kb - g.kb[0] : kb) * kStepK;
        const CUtensorMap *ma = &g.a[seg], *mb = &g.b[PAIR ? rank : seg];
        const uint32_t as = base + s * C::kStage, bs = as + kABytes, bar = full + 8 * s;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(bar, 2 * C::kStage);
          if (!A_MN) {
            load_box(as, ma, bar, k, am);
          } else {
            load_box(as, ma, bar, am, k);
            load_box(as + kGroupBytes, ma, bar, am + 64, k);
          }
          if (!B_MN) {
            load_box(bs, mb, bar, k, bn);
          } else {
#pragma unroll
            for (int i = 0; i < BN / 128; ++i) load_box(bs + i * kGroupBytes, mb, bar, bn + 64 * i, k);
          }
        }
        __syncwarp();
      }
    }
    // the other CTA's last arrivals on this CTA's barriers have to land before it ends
    for (int i = 0; i < C::kStages && i < it && ok; ++i) {
      const int j = it - 1 - i, s = j % C::kStages;
      ok = warp_wait(empty + 8 * s, (j / C::kStages) & 1, abort_flag, g.status, 302);
    }
    if (!ok) {  // a wait gave up: let the copies in flight land
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ products, one lane of the first CTA
    constexpr uint32_t idesc = instr_desc(tile::Fmt<T>::kAB, A_MN, B_MN, kRows, BN);
    int it = 0, n = 0;
    bool ok = true;
    for (int u = first; u < units && ok; u += stride, ++n) {
      const Unit x = unit_of<BN, PAIR>(g, u);
      const int buf = n & 1;
      if (!warp_wait(tempty + 8 * buf, ((n >> 1) & 1) ^ 1, abort_flag, g.status, 303)) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * BN;
      for (int kb = x.k0; kb < x.k1; ++kb, ++it) {
        const int s = it % C::kStages;
        if (!warp_wait(full + 8 * s, (it / C::kStages) & 1, abort_flag, g.status, 304)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t as = base + s * C::kStage, bs = as + kABytes;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kStepK / 16; ++i) {
            const uint64_t da = A_MN ? desc_mnmajor(as + i * 2048, kGroupBytes) : desc_kmajor(as + i * 32);
            const uint64_t db = B_MN ? desc_mnmajor(bs + i * 2048, kGroupBytes) : desc_kmajor(bs + i * 32);
            mma_two(d, da, db, idesc, kb > x.k0 || i > 0);
          }
          commit_two(empty + 8 * s);
          if (kb + 1 == x.k1) commit_two(tfull + 8 * buf);
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue, in both CTAs
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    constexpr int kOut = PAIR ? BN / 2 : BN;  // result columns of a tile, half of them this warp's
    int n = 0;
    for (int u = first; u < units; u += stride, ++n) {
      const Unit x = unit_of<BN, PAIR>(g, u);
      const int buf = n & 1;
      if (!warp_wait(tfull + 8 * buf, (n >> 1) & 1, abort_flag, g.status, 305)) break;
      tc_fence_after();
      const long long m = (long long)x.m0 + rank * 128 + quarter * 32 + lane;
      const bool in = m < g.M;
      const uint32_t t0 = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = half * (kOut / 2); c < (half + 1) * (kOut / 2); c += 16) {
        __syncwarp();  // lanes past the last row skipped the stores
        uint32_t r[16], r2[16];
        tmem_ld16(t0 + c, r);
        if (PAIR) tmem_ld16(t0 + kOut + c, r2);
        tmem_wait_ld();
        const int col = x.n0 + c;
        if (!in || col >= g.N) continue;
        float p[16], q[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          p[j] = __uint_as_float(r[j]);
          q[j] = PAIR ? __uint_as_float(r2[j]) : 0.f;
        }
        if (g.partial != nullptr) {
          float *o = g.partial + ((long long)x.split * (PAIR ? 2 : 1) * g.M + m) * g.N + col;
          store_row<float, 16>(o, g.N % 4 == 0, g.N - col, p);
          if (PAIR) store_row<float, 16>(o + (long long)g.M * g.N, g.N % 4 == 0, g.N - col, q);
        } else if (PAIR) {
          finish_pair<T, 16>(g.e, m, col, g.N, p, q);
        } else {
          finish_one<T, 16>(g.e, m, col, g.N, p);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_first(tempty + 8 * buf);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
}

// (outer, inner) matrix of 16-bit elements, inner next to each other, rows `ld` elements apart; boxes of 64 inner
// elements (128 bytes, swizzled) by `rows` outer ones, zeros outside.
int make_map_2d(CUtensorMap *m, const void *p, int dtype, int64_t inner, int64_t outer, int64_t ld, int rows) {
  tile::EncodeTiledFn enc = tile::encode_fn();
  if (enc == nullptr) return LA_ERR_CUDA;
  static thread_local bool bound = false;  // the encoder needs the device's context current on this thread
  if (!bound) {
    cudaFree(nullptr);
    bound = true;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, dtype == LA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void *>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    snprintf(last_cuda_error_buf(), 256, "cuTensorMapEncodeTiled: CUresult %d (%lld x %lld, stride %lld)", (int)r,
             (long long)outer, (long long)inner, (long long)ld);
  return r == CUDA_SUCCESS ? LA_OK : LA_ERR_CUDA;
}
int operand_map(CUtensorMap *m, const Operand &o, int dtype, int64_t R, int64_t K, int rows) {
  return o.mn_major ? make_map_2d(m, o.p, dtype, R, K, o.ld, kStepK) : make_map_2d(m, o.p, dtype, K, R, o.ld, rows);
}

template <typename T, bool A_MN, bool B_MN, int BN, bool PAIR>
int launch_cfg(const GemmArgs &g, int units, cudaStream_t st) {
  typedef Cfg<BN> C;
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LA_ERR_CUDA;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_kernel<T, A_MN, B_MN, BN, PAIR>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) {
      note_cuda_error(e, "gemm shared memory");
      return LA_ERR_CUDA;
    }
    set[dev] = true;
  }
  const int pairs = sm_count() / 2;
  const int grid = 2 * (units < pairs ? units : pairs);
  gemm_kernel<T, A_MN, B_MN, BN, PAIR><<<grid, kThreads, C::kSmem, st>>>(g);
  return launch_status();
}

template <typename T, int BN>
int launch_t(const Product &p, const GemmArgs &g, int units, cudaStream_t st) {
  const bool am = p.a[0].mn_major, bm = p.b[0].mn_major;
  if (p.pair) return am || bm ? LA_ERR_UNSUPPORTED : launch_cfg<T, false, false, BN, true>(g, units, st);
  if (!am && !bm) return launch_cfg<T, false, false, BN, false>(g, units, st);
  if (!am && bm) return launch_cfg<T, false, true, BN, false>(g, units, st);
  if (am && bm) return launch_cfg<T, true, true, BN, false>(g, units, st);
  return LA_ERR_UNSUPPORTED;
}

}  // namespace

GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K0, int64_t K1, bool pair) {
  const int64_t pairs = sm_count() / 2;
  const int64_t mt = (M + kRows - 1) / kRows;
  const int64_t kb = (K0 + kStepK - 1) / kStepK + (K1 + kStepK - 1) / kStepK;
  GemmPlan best = {256, 1};
  double best_us = 1e30;
  for (int bn = 256; bn >= 128; bn /= 2) {
    const int64_t cols = pair ? bn / 2 : bn;
    const int64_t tiles = mt * ((N + cols - 1) / cols);
    const double step = bn == 256 ? 0.28 : 0.20;  // us a stage
    for (int64_t s = 1; s <= 16 && s * 4 <= kb + 3; ++s) {
      if (s > 1 && tiles * (s - 1) >= pairs * 4) break;
      const int64_t waves = (tiles * s + pairs - 1) / pairs;
      double us = waves * ((kb + s - 1) / s * step + 0.5) + 2.0;
      if (s > 1) us += 2.5 + (double)s * M * N * (pair ? 2 : 1) * 8 / 4e6;
      if (us < best_us) {
        best_us = us;
        best = GemmPlan{bn, (int)s};
      }
    }
  }
  return best;
}

int gemm_launch(const Product &p, const GemmPlan &plan, float *partial, int dtype, cudaStream_t st) {
  GemmArgs g = {};
  const int half = plan.bn / 2;
  int rc = LA_OK;
  for (int s = 0; s < 2 && rc == LA_OK; ++s) {
    if (s < p.segments) rc = operand_map(&g.a[s], p.a[s], dtype, p.M, p.K[s], 128);
    if (rc == LA_OK && (s < p.segments || p.pair)) rc = operand_map(&g.b[s], p.b[s], dtype, p.N, p.K[p.pair ? 0 : s], half);
    g.kb[s] = s < p.segments ? (int)((p.K[s] + kStepK - 1) / kStepK) : 0;
  }
  if (rc != LA_OK) return rc;
  g.e = p.e;
  g.partial = partial;
  g.status = status_word_ptr();
  g.M = (int)p.M; g.N = (int)p.N;
  const int cols = p.pair ? half : plan.bn;
  const int64_t mt = (p.M + kRows - 1) / kRows, nt = (p.N + cols - 1) / cols;
  if (mt * nt * plan.splits > INT32_MAX / 2) return LA_ERR_TOO_LARGE;
  g.m_tiles = (int)mt; g.n_tiles = (int)nt; g.splits = plan.splits;
  const int units = (int)(mt * nt * plan.splits);
  if (dtype == LA_BF16)
    return plan.bn == 256 ? launch_t<__nv_bfloat16, 256>(p, g, units, st) : launch_t<__nv_bfloat16, 128>(p, g, units, st);
  return plan.bn == 256 ? launch_t<__half, 256>(p, g, units, st) : launch_t<__half, 128>(p, g, units, st);
}

}  // namespace lin
}  // namespace la
