// linear_fn and gated_linear_fn for up to 128 tokens, 16-bit types: the step of a serving batch, where the weights' bytes
// are the work.
//
// The weights take the place of the rows: a CTA works on 128 weight rows (64 of Wg and the same 64 of Wu for a pair), the
// tokens are the columns of its accumulator (16 .. 128 of them, 128 x tokens in tensor memory), and no row of a tile is
// wasted on tokens that are not there.  A cluster of S CTAs shares the contraction: each streams its part of the rows through
// a ring of TMA boxes, leaves its sums in its shared memory, and finishes a part of the tokens by adding up the sums of
// all S through distributed shared memory, in order.  One launch, no scratch, equal calls give equal bits.
//
// Bound by HBM: 64 tokens through 2 x 11008 rows of 4096 (bf16) are 27.6 us at the measured copy bandwidth; 35 .. 37 here, 50
// with 256-token tiles and a second kernel for the splits of the contraction.  1 token, 4096 rows of 4096: 5.1, 9.5, 17.6.
// The epilogue's rows in accesses of 8 bytes: 128 tokens through 4096 x 4096 17.6 -> 17.4 us, through 8192 x 1024 14.75 -> 14.5.
// What is left there is the launch, the first loads' way and the two cluster barriers; at 64 tokens the tokens' own boxes, which
// every CTA reads from L2, take half of what the weights take.
#include "linear.cuh"
#include "sm100_ptx.cuh"
#include "tile_common.cuh"

namespace la {
namespace lin {
namespace {

using namespace la::ptx;

constexpr int kRowsW = 128;               // weight rows of a CTA
constexpr int kStepK = 64;
constexpr int kMaxCluster = 8;
constexpr int kMaxRing = 12;
constexpr int kPerSm = 3;                 // CTAs of an SM, at most
constexpr int kThreads = 192;             // warps: 0 loads, 1 multiplies, 2..5 read tensor memory and finish
constexpr uint32_t kWBytes = kRowsW * 128;

template <int MT> struct Cfg {            // MT: columns, the tokens rounded up to 16, 32, 64 or 128
  static constexpr uint32_t kStage = kWBytes + MT * 128;
  static constexpr uint32_t kBeside = 1024 + 16 * kMaxRing + 64;  // alignment, barriers
  // stages of a CTA's ring where `per_sm` of them share an SM's 228 KB (1 KB of each is the system's); the CTA's sums take
  // its place in the end, MT x 512 bytes, which two stages hold
  static int ring(int per_sm, int stages) {
    int n = (int)((228u * 1024 / (unsigned)per_sm - 1024 - kBeside) / kStage);
    if (n > stages) n = stages;
    if (n > kMaxRing) n = kMaxRing;
    return n < 2 ? 2 : n;
  }
  static constexpr uint32_t kCols = MT < 32 ? 32 : MT;
};

struct FewArgs {
  CUtensorMap w[2], x;
  Epilogue e;
  int *status;
  int M, N, stages, ring;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}

template <typename T, int MT, bool PAIR>
__global__ void __launch_bounds__(kThreads) few_tokens_kernel(const __grid_constant__ FewArgs g) {
  typedef Cfg<MT> C;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = base + g.ring * C::kStage, empty = full + 8 * g.ring, done = empty + 8 * g.ring;
  const uint32_t tmem_at = done + 8;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(raw + (tmem_at + 4 - smem_u32(raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int tile = blockIdx.x / size;
  const int k0 = (int)((long long)g.stages * rank / size), k1 = (int)((long long)g.stages * (rank + 1) / size);

  lets_next_start();
  if (threadIdx.x == 0) {
    for (int s = 0; s < g.ring; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_at, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(raw + (tmem_at - smem_u32(raw)));

  bool ok = true;
  if (warp == 0) {
    int s = 0, parity = 1;
    for (int kb = k0; kb < k1; ++kb) {
      ok = warp_wait(empty + 8 * s, parity, abort_flag, g.status, 321);
      if (!ok) break;
      const uint32_t ws = base + s * C::kStage, xs = ws + kWBytes, bar = full + 8 * s;
      const int k = kb * kStepK;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar, C::kStage);
        if (PAIR) {
          load_box(ws, &g.w[0], bar, k, tile * 64);
          load_box(ws + kWBytes / 2, &g.w[1], bar, k, tile * 64);
        } else {
          load_box(ws, &g.w[0], bar, k, tile * kRowsW);
        }
        load_box(xs, &g.x, bar, k, 0);
      }
      __syncwarp();
      if (++s == g.ring) {
        s = 0;
        parity ^= 1;
      }
    }
    if (!ok) {  // a wait gave up: let the copies in flight land
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = instr_desc(tile::Fmt<T>::kAB, 0, 0, kRowsW, MT);
    int s = 0, parity = 0;
    for (int kb = k0; kb < k1; ++kb) {
      ok = warp_wait(full + 8 * s, parity, abort_flag, g.status, 322);
      if (!ok) break;
      tc_fence_after();
      const uint32_t ws = base + s * C::kStage, xs = ws + kWBytes;
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < kStepK / 16; ++i)
          mma_ss(tmem, desc_kmajor(ws + i * 32), desc_kmajor(xs + i * 32), idesc, kb > k0 || i > 0);
        mma_commit(kb + 1 == k1 ? done : empty + 8 * s);
      }
      __syncwarp();
      if (++s == g.ring) {
        s = 0;
        parity ^= 1;
      }
    }
  } else {
    // the CTA's sums: [token][weight row], fp32, where the ring was (its last reader is done)
    ok = warp_wait(done, 0, abort_flag, g.status, 323);
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;
    float *sums = reinterpret_cast<float *>(raw + (base - smem_u32(raw)));
#pragma unroll 1
    for (int c = 0; c < MT; c += 16) {
      uint32_t r[16];
      tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(c + j) * kRowsW + row] = __uint_as_float(r[j]);
    }
    tc_fence_before();
  }
  __syncwarp();
  cluster_sync();
  if (warp >= 2) {
    // this CTA's tokens: every size-th of them.  A warp takes one (a pair: two, 16 lanes each) at a time, a lane 4 columns.
    constexpr int kOut = PAIR ? 64 : kRowsW, kLanes = kOut / 4, kTokens = 32 / kLanes;
    const int col = lane % kLanes * 4, n = tile * kOut + col;
    const int step = (int)size * 4 * kTokens;
    for (int m = (int)rank + (int)size * ((warp - 2) * kTokens + lane / kLanes); m < g.M; m += step) {
      float p[4] = {}, q[4] = {};
#pragma unroll 4
      for (uint32_t c = 0; c < size; ++c) {
        const uint32_t at = in_cta(base, c) + (uint32_t)(m * kRowsW + col) * 4u;
        const float4 v = load_cluster(at);
        p[0] += v.x; p[1] += v.y; p[2] += v.z; p[3] += v.w;
        if (PAIR) {
          const float4 w = load_cluster(at + 256u);
          q[0] += w.x; q[1] += w.y; q[2] += w.z; q[3] += w.w;
        }
      }
      if (PAIR) finish_pair<T, 4>(g.e, m, n, g.N, p, q);
      else finish_one<T, 4>(g.e, m, n, g.N, p);
    }
  }
  __syncwarp();
  cluster_sync();  // the sums stay until everyone has read them
  if (warp == 1) tmem_dealloc(tmem, C::kCols);
}

// The cluster's size: the largest whose clusters all fit at once (more would leave a last round with few bytes in flight), of
// at least three stages a CTA; from 64 tokens on 4 are enough for 32 tiles, since every token's sums come from all CTAs of a
// cluster.  How many clusters fit is asked for once per kernel and device; the answer counts one CTA an SM, up to three
// run there.  Measured with sizes 1 .. 8 in us, 1 token: 172 tiles of K 4096 32.5 31.3 34 34 37 37 40 39 (2 taken), 96 tiles 22.2
// 20.4 19.3 19.4 23 23 24 23 (4), 64 tiles of K 8192 35 26 24.4 23.6 23.5 23.8 29 28 (6), 32 tiles of K 4096 19 12 10.3 10.3 9.7 9.6
// 9.8 9.2 (8); 128 tokens, 32 tiles of K 4096: 32 21 17.7 14.5 16.3 16.0 17.9 17.7 (4), 16 tiles of K 2048: 23 16 13 10.3 10.6
// 10.9 11.1 9.7 (8); 32 tokens, 32 tiles of K 768: 7.7 5.8 5.8 5.5 6.3 6.5 6.6 7.0 (4).  Up to 4 against up to 8 CTAs, 64 and 128
// tokens, K 1024 .. 8192: 32 to 64 tiles 3 .. 20 % less (one of 32 shapes 4 % more), from 80 tiles on no more than 4 fit, 16 and 24 tiles
// 8 % less at K 1024, up to 11 % more at 8192.
template <typename T, int MT, bool PAIR>
int launch_cfg(FewArgs g, int tiles, cudaStream_t st) {
  typedef Cfg<MT> C;
  static bool set[64] = {false};
  static int fit[64][kMaxCluster + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LA_ERR_CUDA;
  if (!set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(few_tokens_kernel<T, MT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         227 * 1024);
    for (int s = 1; s <= kMaxCluster && e == cudaSuccess; ++s) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)s;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)s);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = C::kBeside + C::ring(kPerSm, kMaxRing) * C::kStage;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&fit[dev][s], few_tokens_kernel<T, MT, PAIR>, &cfg);
    }
    if (e != cudaSuccess) {
      cudaGetLastError();
      note_cuda_error(e, "few_tokens_kernel");
      return LA_ERR_CUDA;
    }
    set[dev] = true;
  }
  int size = MT >= 64 && tiles >= 32 ? 4 : kMaxCluster;
  if (size > g.stages / 3) size = g.stages < 3 ? 1 : g.stages / 3;
  while (size > 1 && kPerSm * fit[dev][size] < tiles) --size;
  // few CTAs an SM: the more stages each
  int per_sm = (tiles + fit[dev][size] - 1) / fit[dev][size];
  if (per_sm > kPerSm) per_sm = kPerSm;
  g.ring = C::ring(per_sm, (g.stages + size - 1) / size);
  return launch_early(few_tokens_kernel<T, MT, PAIR>, dim3((unsigned)(tiles * size)), kThreads,
                      C::kBeside + g.ring * C::kStage, st, size, g);
}

template <typename T, bool PAIR>
int launch_m(const FewArgs &g, int mt, int tiles, cudaStream_t st) {
  switch (mt) {
    case 16: return launch_cfg<T, 16, PAIR>(g, tiles, st);
    case 32: return launch_cfg<T, 32, PAIR>(g, tiles, st);
    case 64: return launch_cfg<T, 64, PAIR>(g, tiles, st);
  }
  return launch_cfg<T, 128, PAIR>(g, tiles, st);
}

}  // namespace

bool few_tokens_fit(const Product &p, int dtype) {
  return dtype != LA_F32 && p.M <= 128 && p.segments == 1 && !p.a[0].mn_major && !p.b[0].mn_major;
}

int few_tokens_launch(const Product &p, int dtype, cudaStream_t st) {
  FewArgs g = {};
  int mt = 16;
  while (mt < p.M) mt *= 2;
  const int rows = p.pair ? 64 : kRowsW;
  int rc = make_map_2d(&g.x, p.a[0].p, dtype, p.K[0], p.M, p.a[0].ld, mt);
  for (int i = 0; i < (p.pair ? 2 : 1) && rc == LA_OK; ++i)
    rc = make_map_2d(&g.w[i], p.b[i].p, dtype, p.K[0], p.N, p.b[i].ld, rows);
  if (rc != LA_OK) return rc;
  g.e = p.e;
  if (!status_word_for(st, &g.status)) return LA_ERR_CUDA;
  g.M = (int)p.M; g.N = (int)p.N;
  g.stages = (int)((p.K[0] + kStepK - 1) / kStepK);
  const int64_t tiles = (p.N + rows - 1) / rows;
  if (tiles * kMaxCluster > INT32_MAX) return LA_ERR_TOO_LARGE;
  if (dtype == LA_BF16)
    return p.pair ? launch_m<__nv_bfloat16, true>(g, mt, (int)tiles, st)
                  : launch_m<__nv_bfloat16, false>(g, mt, (int)tiles, st);
  return p.pair ? launch_m<__half, true>(g, mt, (int)tiles, st)
                : launch_m<__half, false>(g, mt, (int)tiles, st);
}

}  // namespace lin
}  // namespace la
