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
// groups of 8 rows of tiles, so that the operands of the tiles in flight stay in L2.  Tiles that do not fill a round of the
// pairs (all of them where there are few, else the last round's) have their contraction split over several units, whose
// fp32 sums tile_sum_kernel adds in a fixed order (gemm_plan).
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
constexpr uint32_t kStrip = 32 * 256;      // an epilogue warp's 32 rows of 64 fp32 values
constexpr int kGroup = 8;                  // rows of tiles walked together
constexpr uint32_t kGroupBytes = 64 * 128; // 64 rows of an operand whose rows lie next to each other, 64 steps

template <int BN> struct Cfg {
  static constexpr uint32_t kBBytes = BN / 2 * 128;
  static constexpr uint32_t kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 5 : 6;
  static constexpr uint32_t kSmem = 1024 + kStages * kStage + kEpiWarps * kStrip + 512;
  static constexpr uint32_t kCols = 2 * BN;  // tensor memory: two accumulators
};

struct GemmArgs {
  CUtensorMap a[2], b[2];
  Epilogue e;
  float *partial;            // sums of split tiles: [tile - whole][split][row][BN]
  int *status;
  int M, N;
  int kb[2];                 // stages of each segment
  int m_tiles, n_tiles;
  int whole, splits;         // tiles [0, whole) are done whole, the others in `splits` units each
  int rows;                  // rows of a split tile
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same place in the first CTA of the pair
__device__ __forceinline__ uint32_t in_first(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(bar)) : "memory");
}
// a box into this CTA's shared memory; the bytes count on the first CTA's barrier (`bar`: out of in_first)
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
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
  int m0, n0, k0, k1;
  int slot;  // place of its sums, or -1 for a whole tile
};
template <int BN, bool PAIR> __device__ __forceinline__ void place_of(const GemmArgs &g, int tile, int &m0, int &n0) {
  const int per = kGroup * g.n_tiles, group = tile / per, first = group * kGroup;
  const int rows = min(g.m_tiles - first, kGroup), r = tile - group * per;
  m0 = (first + r % rows) * kRows;
  n0 = r / rows * (PAIR ? BN / 2 : BN);
}
template <int BN, bool PAIR>
__device__ __forceinline__ Unit unit_of(const GemmArgs &g, int u) {
  const int v = u - g.whole;
  const bool cut = v >= 0;
  const int part = cut ? v / g.splits : 0, split = v - part * g.splits;
  Unit x;
  place_of<BN, PAIR>(g, cut ? g.whole + part : u, x.m0, x.n0);
  const int all = g.kb[0] + g.kb[1];
  x.k0 = cut ? (int)((long long)all * split / g.splits) : 0;
  x.k1 = cut ? (int)((long long)all * (split + 1) / g.splits) : all;
  x.slot = cut ? v : -1;
  return x;
}

// An epilogue warp's strip: 32 rows of 64 fp32 values, 64 result columns or 32 of g and 32 of u.  Pieces of 16 bytes lie
// where neither the writing lanes (8 rows, one piece) nor the reading lanes (kLanes lanes a row, 8 columns each) meet
// in a bank.
template <bool PAIR> struct Strip {
  static constexpr int kCols = PAIR ? 32 : 64;
  static constexpr int kLanes = kCols / 8;
  static constexpr int kRowsAt = 32 / kLanes;  // rows the warp reads at a time
  static __device__ __forceinline__ float4 *piece(float *strip, int row, int i) {
    const int f = PAIR ? i : (i >> 1) | (i & 1) << 3;
    return reinterpret_cast<float4 *>(strip) + row * 16 + (f ^ (row & 7));
  }
  // columns 8 cl .. 8 cl + 7 of a row; u: of the second product of a pair
  static __device__ __forceinline__ void take(float *strip, int row, int cl, int u, float *v) {
    const float4 x = *piece(strip, row, 8 * u + 2 * cl), y = *piece(strip, row, 8 * u + 2 * cl + 1);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  }
};

template <typename T> __device__ __forceinline__ void unpack8(const uint4 &r, float *v) {
  const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = Cvt<T>::to_f(h[j]);
}

// where rows m0 .. m0 + 31 of the result go if they lie together, else null
template <typename T> __device__ __forceinline__ T *out_rows(const Epilogue &e, long long m0) {
  if (m0 + 32 <= e.split) return m0 + 32 <= e.live ? static_cast<T *>(e.out) + m0 * e.ldo : nullptr;
  if (m0 < e.split) return nullptr;
  return m0 - e.split + 32 <= e.live ? static_cast<T *>(e.out2) + (m0 - e.split) * e.ldo : nullptr;
}

// a strip that lies inside the matrix, everything on 16 bytes
template <typename T, bool PAIR>
__device__ __forceinline__ void inner_strip(const Epilogue &e, float *strip, T *out, long long m0, int n0, int lane) {
  typedef Strip<PAIR> S;
  constexpr int G = 4;
  const int cl = lane % S::kLanes, rl = lane / S::kLanes, col = n0 + 8 * cl;
  out += rl * e.ldo + col;
  const long long ostep = S::kRowsAt * e.ldo;
  float b0[8], b1[8];
  if (e.bias[0] != nullptr) unpack8<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(e.bias[0]) + col), b0);
  if (PAIR && e.bias[1] != nullptr)
    unpack8<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(e.bias[1]) + col), b1);
  const T *res = e.residual == nullptr ? nullptr : static_cast<const T *>(e.residual) + (m0 + rl) * e.ldr + col;
  const long long rstep = S::kRowsAt * e.ldr;
  long long kept = (m0 + rl) * e.lds + col;
  const long long kstep = S::kRowsAt * e.lds;
#pragma unroll 1
  for (int i = 0; i < S::kLanes; i += G) {
    uint4 r[G];
    if (!PAIR && res != nullptr) {
#pragma unroll
      for (int k = 0; k < G; ++k) r[k] = *reinterpret_cast<const uint4 *>(res + k * rstep);
      res += G * rstep;
    }
    float p[8 * G], q[8 * G];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      S::take(strip, (i + k) * S::kRowsAt + rl, cl, 0, p + 8 * k);
      if (PAIR) S::take(strip, (i + k) * S::kRowsAt + rl, cl, 1, q + 8 * k);
    }
    if (e.bias[0] != nullptr) {
#pragma unroll
      for (int k = 0; k < 8 * G; ++k) p[k] += b0[k & 7];
    }
    if (PAIR && e.bias[1] != nullptr) {
#pragma unroll
      for (int k = 0; k < 8 * G; ++k) q[k] += b1[k & 7];
    }
    if (e.save.p != nullptr) {
#pragma unroll
      for (int k = 0; k < G; ++k) {
        store_saved<T, 8>(e.save, kept + k * kstep, true, 8, reinterpret_cast<const float (&)[8]>(p[8 * k]));
        if (PAIR)
          store_saved<T, 8>(e.save, kept + k * kstep + e.save_up, true, 8, reinterpret_cast<const float (&)[8]>(q[8 * k]));
      }
      kept += G * kstep;
    }
    activate<T, 8 * G>(p, e.act);
    if (PAIR) {
#pragma unroll
      for (int k = 0; k < 8 * G; ++k) p[k] *= q[k];
    } else if (e.residual != nullptr) {
      float v[8];
#pragma unroll
      for (int k = 0; k < G; ++k) {
        unpack8<T>(r[k], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[8 * k + j] += v[j];
      }
    }
#pragma unroll
    for (int k = 0; k < G; ++k)
      store_row<T, 8>(out + k * ostep, true, 8, reinterpret_cast<const float (&)[8]>(p[8 * k]));
    out += G * ostep;
  }
}

// a strip at the edge, or tensors that are not on 16 bytes
template <typename T, bool PAIR>
__device__ __noinline__ void edge_strip(const Epilogue &e, float *strip, long long m0, int n0, int M, int N, int lane) {
  typedef Strip<PAIR> S;
  const int cl = lane % S::kLanes, rl = lane / S::kLanes, col = n0 + 8 * cl;
#pragma unroll 1
  for (int i = 0; i < S::kLanes; ++i) {
    const int row = i * S::kRowsAt + rl;
    float p[8], q[8];
    S::take(strip, row, cl, 0, p);
    if (PAIR) S::take(strip, row, cl, 1, q);
    if (m0 + row >= M) continue;
    if (PAIR) finish_pair<T, 8>(e, m0 + row, col, N, p, q);
    else finish_one<T, 8>(e, m0 + row, col, N, p);
  }
}

// a strip of a split tile's sums: rows r0 .. r0 + 31 of the tile, accumulator columns from c (and for u from c2) on
template <bool PAIR, int BN>
__device__ __noinline__ void sums_strip(const GemmArgs &g, float *strip, int slot, int r0, int c, int c2, int lane) {
  typedef Strip<PAIR> S;
  const int cl = lane % S::kLanes, rl = lane / S::kLanes;
  float *o = g.partial + ((long long)slot * g.rows + r0 + rl) * BN + 8 * cl;
#pragma unroll 4
  for (int i = 0; i < S::kLanes; ++i, o += S::kRowsAt * BN) {
    const int row = i * S::kRowsAt + rl;
    if (r0 + row >= g.rows) break;
    float p[8];
    S::take(strip, row, cl, 0, p);
    store_row<float, 8>(o + c, true, 8, p);
    if (PAIR) {
      S::take(strip, row, cl, 1, p);
      store_row<float, 8>(o + c2, true, 8, p);
    }
  }
}

template <typename T, bool A_MN, bool B_MN, int BN, bool PAIR>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs g) {
  typedef Cfg<BN> C;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t strips = base + C::kStages * C::kStage;
  const uint32_t bars = strips + kEpiWarps * kStrip;
  const uint32_t full = bars, empty = full + 8 * C::kStages, tfull = empty + 8 * C::kStages, tempty = tfull + 16;
  const uint32_t tmem_at = tempty + 16;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(raw + (tmem_at + 4 - smem_u32(raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int units = g.whole + (g.m_tiles * g.n_tiles - g.whole) * g.splits;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  lets_next_start();
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
  after_previous();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(raw + (tmem_at - smem_u32(raw)));

  if (warp == 0) {
    // ------------------------------------------------------------ loads, in both CTAs
    if (lane == 0) {
      prefetch_tmap(&g.a[0]);
      prefetch_tmap(&g.b[PAIR ? rank : 0]);
    }
    const uint32_t full0 = in_first(full);
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
        const uint32_t as = base + s * C::kStage, bs = as + kABytes, bar = full0 + 8 * s;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * C::kStage);
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
    // A lane of tensor memory is a row, so a thread holds 64 columns of one row (32 of g and the same 32 of u).  Written
    // from there, every store would touch 32 rows with 16 bytes each (the epilogue took 32,000 cycles a tile that way, 17 us);
    // through a strip of shared memory of the warp's own 8 or 4 lanes share a row and a store touches 4 or 8 rows with
    // 128 or 64 bytes.  With two warps per scheduler the latency of every instruction counts: four rows at a time, one
    // branch per option for all four, pointers that only advance; strips at the matrix's edge go another way.
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    constexpr int kOut = PAIR ? BN / 2 : BN;  // result columns of a tile, half of them this warp's
    float *strip = reinterpret_cast<float *>(raw + (strips - smem_u32(raw)) + (warp - 4) * kStrip);
    int n = 0;
    for (int u = first; u < units; u += stride, ++n) {
      const Unit x = unit_of<BN, PAIR>(g, u);
      const int buf = n & 1;
      const long long m0 = (long long)x.m0 + rank * 128 + quarter * 32;
      if (!warp_wait(tfull + 8 * buf, (n >> 1) & 1, abort_flag, g.status, 305)) break;
      tc_fence_after();
      const uint32_t t0 = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = half * (kOut / 2); c < (half + 1) * (kOut / 2); c += Strip<PAIR>::kCols) {
        const int n0 = x.n0 + c;
        if (m0 >= g.M || n0 >= g.N) break;
        {
          uint32_t r[32], r2[32];
          tmem_ld32(t0 + c, r);
          tmem_ld32(t0 + c + (PAIR ? kOut : 32), r2);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            *Strip<PAIR>::piece(strip, lane, i) = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                              __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
            *Strip<PAIR>::piece(strip, lane, i + 8) =
                make_float4(__uint_as_float(r2[4 * i]), __uint_as_float(r2[4 * i + 1]), __uint_as_float(r2[4 * i + 2]),
                            __uint_as_float(r2[4 * i + 3]));
          }
        }
        __syncwarp();
        const bool inner = n0 + Strip<PAIR>::kCols <= g.N && m0 + 32 <= g.M;
        if (x.slot >= 0) {
          sums_strip<PAIR, BN>(g, strip, x.slot, (int)rank * 128 + quarter * 32, c, c + kOut, lane);
        } else {
          T *out = inner && g.e.vec ? out_rows<T>(g.e, m0) : nullptr;
          if (out != nullptr) inner_strip<T, PAIR>(g.e, strip, out, m0, n0, lane);
          else edge_strip<T, PAIR>(g.e, strip, m0, n0, g.M, g.N, lane);
        }
        __syncwarp();
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

// The sums of a split tile's units, in order, and the epilogue.  CTA (split tile, 8 rows), 8 columns a thread.
template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(256) tile_sum_kernel(const __grid_constant__ GemmArgs g) {
  constexpr int kLanes = (PAIR ? BN / 2 : BN) / 8;
  lets_next_start();
  after_previous();
  int m0, n0;
  place_of<BN, PAIR>(g, g.whole + (int)blockIdx.x, m0, n0);
  for (int j = threadIdx.x; j < 8 * kLanes; j += 256) {
    const int row = (int)blockIdx.y * 8 + j / kLanes, col = j % kLanes * 8;
    if (row >= g.rows || m0 + row >= g.M || n0 + col >= g.N) continue;
    const float *s = g.partial + ((long long)blockIdx.x * g.splits * g.rows + row) * BN + col;
    float p[8] = {}, q[8] = {};
    const long long step = (long long)g.rows * BN;
    for (int i = 0; i < g.splits; i += 4) {  // four units' loads at a time, added in order
      float v[4][8], w[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool is = i + j < g.splits;
        load_row<float, 8>(s + (is ? j * step : 0), true, 8, v[j]);
        if (PAIR) load_row<float, 8>(s + (is ? j * step : 0) + BN / 2, true, 8, w[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i + j >= g.splits) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          p[k] += v[j][k];
          if (PAIR) q[k] += w[j][k];
        }
      }
      s += 4 * step;
    }
    if (PAIR) finish_pair<T, 8>(g.e, m0 + row, n0 + col, g.N, p, q);
    else finish_one<T, 8>(g.e, m0 + row, n0 + col, g.N, p);
  }
}

}  // namespace

int make_map_2d(CUtensorMap *m, const void *p, int dtype, int64_t inner, int64_t outer, int64_t ld, int rows) {
  tile::EncodeTiledFn enc = tile::encode_fn();
  if (enc == nullptr) return LA_ERR_CUDA;
  static thread_local bool bound = false;  // the encoder needs the device's context current on this thread
  if (!bound) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return LA_ERR_CUDA;
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

namespace {

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
  const int rc = launch_early(gemm_kernel<T, A_MN, B_MN, BN, PAIR>, dim3((unsigned)grid), kThreads, C::kSmem, st, 0, g);
  const int cut = g.m_tiles * g.n_tiles - g.whole;
  if (rc != LA_OK || cut == 0) return rc;
  return launch_early(tile_sum_kernel<T, BN, PAIR>, dim3((unsigned)cut, (unsigned)((g.rows + 7) / 8)), 256, 0, st, 0, g);
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

// Estimates the kernel's time for tiles of 256 and 128 columns, whole or split: every tile in s units, or the tiles of the last,
// incomplete round in as many units as there are pairs for (tiles of 256 only: whole rounds of narrow ones run at the power
// limit and move more operands: with them 44 products in which they would be taken, which is 1 in 36 of a grid of sizes, needed 2 %
// more on average; as results 0.85 .. 1.10 of the time, 2 % less, as dW 0.87 .. 1.21, 2 % more, as dx 0.94 .. 1.43, 6 % more).
// A stage takes 0.28 us (256 columns) or 0.20, a tile 0.5 us besides, sums another launch (2.5 us) and their way to memory
// and back (4 TB/s).  Against measurements of 17 shapes with 1 .. 16 units a tile the estimate's choice was the quickest or
// within 4 % of it in 15, within 9 % in all.  The last round split: 4096 x 16384 x 4096 387 -> 383 and in another run 378 -> 366 us,
// 256 tokens through a pair of 11008 x 4096 55 -> 50.
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K0, int64_t K1, bool pair) {
  const int64_t pairs = sm_count() / 2;
  const int64_t mt = (M + kRows - 1) / kRows, rows = M < kRows ? M : kRows;
  const int64_t kb = (K0 + kStepK - 1) / kStepK + (K1 + kStepK - 1) / kStepK;
  GemmPlan best = {};
  double best_us = 1e30;
  for (int bn = 256; bn >= 128; bn /= 2) {
    const int64_t cols = pair ? bn / 2 : bn;
    const int64_t tiles = mt * ((N + cols - 1) / cols);
    const double step = bn == 256 ? 0.28 : 0.20;
    auto consider = [&](int64_t whole, int64_t s) {
      const int64_t cut = (tiles - whole) * s;
      double us = 2.0 + (whole + pairs - 1) / pairs * (kb * step + 0.5);
      if (cut > 0) {
        const double most = (double)s * M * N * (pair ? 2 : 1), sums = (double)cut * rows * bn;  // rows past M are not written
        us += (cut + pairs - 1) / pairs * ((kb + s - 1) / s * step + 0.5) + 2.5 + (sums < most ? sums : most) * 8 / 4e6;
      }
      if (us >= best_us) return;
      best_us = us;
      best = GemmPlan{bn, (int)s, whole, rows, cut * rows * bn * 4};
    };
    consider(tiles, 1);
    for (int64_t s = 2; s <= 16 && s * 4 <= kb + 3; ++s) {
      if (tiles * (s - 1) < pairs * 4) consider(0, s);
      if (bn == 256 && tiles > pairs && tiles % pairs * s <= pairs) consider(tiles / pairs * pairs, s);
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
  if (!status_word_for(st, &g.status)) return LA_ERR_CUDA;
  g.M = (int)p.M; g.N = (int)p.N;
  const int cols = p.pair ? half : plan.bn;
  const int64_t mt = (p.M + kRows - 1) / kRows, nt = (p.N + cols - 1) / cols;
  const int64_t all = plan.whole + (mt * nt - plan.whole) * plan.splits;
  if (all > INT32_MAX / 2) return LA_ERR_TOO_LARGE;
  g.m_tiles = (int)mt; g.n_tiles = (int)nt;
  g.whole = (int)plan.whole; g.splits = plan.splits; g.rows = (int)plan.rows;
  const int units = (int)all;
  if (dtype == LA_BF16)
    return plan.bn == 256 ? launch_t<__nv_bfloat16, 256>(p, g, units, st) : launch_t<__nv_bfloat16, 128>(p, g, units, st);
  return plan.bn == 256 ? launch_t<__half, 256>(p, g, units, st) : launch_t<__half, 128>(p, g, units, st);
}

}  // namespace lin
}  // namespace la
