// linear_fn and gated_linear_fn: the host plan of both directions, the fp32 product, and the passes around the
// matrix products (derivative of the activation, sums over rows).
//
//   linear        z = x W^T + b             y = act(z) + r
//                 dz = dy act'(z)           dx = dz W      dW = dz^T x      db = sum over rows of dz
//   gated pair    g = x Wg^T + bg, u = x Wu^T + bu         h = act(g) u
//                 dg = dh u act'(g), du = dh act(g)        dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, sums
//
// x (M, K), W (N, K).  Every product is accumulated in fp32 and rounded once, after bias, activation, product of
// the pair and residual.  What the backward needs of the forward is z, or g and u: for 16-bit types kept as the upper 24
// bits of their fp32 values (computing them again would cost a third of the forward's and backward's products together; kept
// in 16 bits their two roundings made the gradients of a pair 1.8 times as far off as rounding the gradients alone
// does, in 24 bits 1.42 times, which is what the rounding of dz leaves).  dz, dg and du are rounded to the type of x, since they are
// operands of two products; in fp16 one above 65504 becomes infinite, as a loss scale has to see to.
#include "linear.cuh"

namespace la {
namespace lin {

int sm_count() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  if (sms[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    sms[dev] = n;
  }
  return sms[dev];
}

namespace {

// ------------------------------------------------------------------------------ fp32 product on the CUDA cores
struct SimtArgs {
  Operand a[2], b[2];
  long long K[2];
  int vec_a[2], vec_b[2];
  long long M, N;
  int n_tiles, splits;
  long long steps[2];  // 16-wide steps of each segment
  Epilogue e;
};

__device__ __forceinline__ void cluster_all() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// four floats at this CTA's shared address `at`, of the cluster's CTA `rank`
__device__ __forceinline__ float4 load_of(uint32_t at, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at), "r"(rank) : "memory");
  return v;
}

constexpr int kStep = 16;
template <int TILE> constexpr int simt_threads() { return TILE == 128 ? 256 : 128; }

// A thread's share of the TILE x 16 tiles of an operand, step after step: two quads, along the contraction or along the rows
// (mn_major).
template <int TILE> struct SimtLoad {
  const float *p[2];
  long long step;
  int left;  // along the contraction: bits of the rows that exist; along the rows: rows that exist from the quad's first on
  bool mn, vec;
  __device__ __forceinline__ void init(const Operand &o, int vec_, long long r0, long long R, long long k0) {
    const int t = threadIdx.x;
    const float *base = static_cast<const float *>(o.p);
    mn = o.mn_major;
    vec = vec_;
    left = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!mn) {
        const long long r = r0 + (t >> 2) + TILE / 2 * i;
        p[i] = base + r * o.ld + k0 + (t & 3) * 4;
        left |= (r < R) << i;
      } else {
        const long long r = r0 + t % (TILE / 4) * 4;
        p[i] = base + (k0 + t / (TILE / 4) + 8 * i) * o.ld + r;
        left = R - r < 4 ? (int)(R - r) : 4;
      }
    }
    step = mn ? kStep * o.ld : kStep;
  }
  // the next step, of which k_left terms exist
  __device__ __forceinline__ void fetch(int k_left, float (&v)[8]) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float (&q)[4] = reinterpret_cast<float (&)[4]>(v[4 * i]);
      const int exist = !mn ? (left >> i & 1 ? k_left - (t & 3) * 4 : 0) : (t / (TILE / 4) + 8 * i < k_left ? left : 0);
      load_row<float, 4>(p[i], vec, exist, q);
      p[i] += step;
    }
  }
};
template <int TILE>
__device__ __forceinline__ void simt_put(bool mn, float (*s)[TILE + 4], const float (&v)[8]) {
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!mn) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[(t & 3) * 4 + j][(t >> 2) + TILE / 2 * i] = v[4 * i + j];
    } else {
      *reinterpret_cast<float4 *>(&s[t / (TILE / 4) + 8 * i][t % (TILE / 4) * 4]) =
          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  }
}

// One TILE x TILE tile (of one split) per CTA, 8 x 4 results a thread (TILE 64, 128 threads) or 8 x 8 (TILE 128, 256 threads),
// packed over pairs of rows; the next step's operands are in registers while the current step's are multiplied.  The splits
// of a tile are a cluster: each CTA adds everyone's sums for a part of the tile, in order, out of shared memory.  2048 x 2048 x
// 2048 402 us (43 TFLOP/s: 256 tiles in 296 places, and shared memory and the instructions beside the products, which leave
// the multipliers two thirds of their time; elements of B kept twice in shared memory, to save doubling them in registers, 860
// us).  514 x 512 x 512 14.3 us, 128 x 16384 x 128 52; with the splits' sums through global memory and a second launch 16.7 and
// 61, but 16 x 4096 x 4096 61 instead of 67 (clusters of 9 fill the SMs less evenly).
template <int TILE, bool PAIR>
__global__ void __launch_bounds__(simt_threads<TILE>(), TILE == 128 ? 2 : (PAIR ? 3 : 5)) simt_product_kernel(const SimtArgs a) {
  constexpr int TN = TILE / 16;  // columns a thread: 4 from tx * 4 on, and for TILE 128 4 from 64 + tx * 4 on
  constexpr int P = PAIR ? 2 : 1;
  union Shared {
    struct {
      float a[2][kStep][TILE + 4], b[2][P][kStep][TILE + 4];
    } in;
    float4 sums[P][TILE][16];  // 64 columns
  };
  __shared__ __align__(16) Shared mem;
  auto &sa = mem.in.a;
  auto &sb = mem.in.b;
  // a warp has 8 x 4 threads' results: fewer bytes out of shared memory than with 16 x 2 (2048 cubed 416 -> 401 us)
  const int tx = (threadIdx.x >> 5 & 1) * 8 + (threadIdx.x & 7), ty = (threadIdx.x >> 6) * 4 + (threadIdx.x >> 3 & 3);
  const long long tile = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x - tile * a.splits);
  const long long m0 = tile / a.n_tiles * TILE, n0 = tile % a.n_tiles * TILE;
  const long long all = a.steps[0] + a.steps[1];
  const long long s0 = all * split / a.splits, s1 = all * (split + 1) / a.splits;
  float2 acc[4][TN] = {}, acc2[PAIR ? 4 : 1][TN] = {};  // rows 2 i and 2 i + 1, column j
  float va[8], vb[8], vb2[8];
  lets_next_start();
  after_previous();
  SimtLoad<TILE> la, lb, lb2;
  long long k_left = 0;  // terms of the segment from the next step on
  auto fetch = [&](long long s) {
    if (s == s0 || s == a.steps[0]) {  // the first step here, or of the second segment
      const int g = s >= a.steps[0];
      const long long k0 = (g ? s - a.steps[0] : s) * kStep;
      la.init(a.a[g], a.vec_a[g], m0, a.M, k0);
      lb.init(a.b[g], a.vec_b[g], n0, a.N, k0);
      if (PAIR) lb2.init(a.b[1], a.vec_b[1], n0, a.N, k0);
      k_left = a.K[g] - k0;
    }
    const int some = k_left < kStep ? (int)k_left : kStep;
    la.fetch(some, va);
    lb.fetch(some, vb);
    if (PAIR) lb2.fetch(some, vb2);
    k_left -= kStep;
  };
  auto put = [&](int at) {  // both operands of a step lie the same way in both segments
    simt_put<TILE>(la.mn, sa[at], va);
    simt_put<TILE>(lb.mn, sb[at][0], vb);
    if (PAIR) simt_put<TILE>(lb2.mn, sb[at][PAIR ? 1 : 0], vb2);
  };
  if (s0 < s1) {
    fetch(s0);
    put(0);
  }
  __syncthreads();
  for (long long s = s0; s < s1; ++s) {
    const int at = (int)(s - s0) & 1;
    if (s + 1 < s1) fetch(s + 1);
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      float2 x[4];
      float y[TN];
      *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(&sa[at][k][ty * 8]);
      *reinterpret_cast<float4 *>(x + 2) = *reinterpret_cast<const float4 *>(&sa[at][k][ty * 8 + 4]);
#pragma unroll
      for (int j = 0; j < TN; j += 4)
        *reinterpret_cast<float4 *>(y + j) = *reinterpret_cast<const float4 *>(&sb[at][0][k][tx * 4 + 16 * j]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = fma2(x[i], make_float2(y[j], y[j]), acc[i][j]);
      if (PAIR) {
#pragma unroll
        for (int j = 0; j < TN; j += 4)
          *reinterpret_cast<float4 *>(y + j) = *reinterpret_cast<const float4 *>(&sb[at][PAIR ? 1 : 0][k][tx * 4 + 16 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc2[PAIR ? i : 0][j] = fma2(x[i], make_float2(y[j], y[j]), acc2[PAIR ? i : 0][j]);
      }
    }
    if (s + 1 < s1) put(at ^ 1);
    __syncthreads();
  }
  auto take = [&](int i, int h, float (&p)[4], float (&q)[4]) {  // row i, columns 4 h .. 4 h + 3 of this thread
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = i % 2 ? acc[i / 2][4 * h + j].y : acc[i / 2][4 * h + j].x;
      q[j] = i % 2 ? acc2[PAIR ? i / 2 : 0][4 * h + j].y : acc2[PAIR ? i / 2 : 0][4 * h + j].x;
    }
  };
  auto finish = [&](long long m, long long n, float (&p)[4], float (&q)[4]) {
    if (m >= a.M || n >= a.N) return;
    if (PAIR) finish_pair<float, 4>(a.e, m, (int)n, (int)a.N, p, q);
    else finish_one<float, 4>(a.e, m, (int)n, (int)a.N, p);
  };
  if (a.splits == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < TN / 4; ++h) {
        float p[4], q[4];
        take(i, h, p, q);
        finish(m0 + ty * 8 + i, n0 + tx * 4 + 64 * h, p, q);
      }
    return;
  }
#pragma unroll
  for (int h = 0; h < TN / 4; ++h) {
    if (h > 0) cluster_all();  // the first 64 columns have been read
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float p[4], q[4];
      take(i, h, p, q);
      mem.sums[0][ty * 8 + i][tx] = make_float4(p[0], p[1], p[2], p[3]);
      if (PAIR) mem.sums[P - 1][ty * 8 + i][tx] = make_float4(q[0], q[1], q[2], q[3]);
    }
    cluster_all();
    for (int u = split * simt_threads<TILE>() + threadIdx.x; u < TILE * 16; u += a.splits * simt_threads<TILE>()) {
      if (m0 + (u >> 4) >= a.M) break;
      const uint32_t at = (uint32_t)__cvta_generic_to_shared(&mem.sums[0][u >> 4][u & 15]);
      float p[4] = {}, q[4] = {};
#pragma unroll 4
      for (int i = 0; i < a.splits; ++i) {
        const float4 v = load_of(at, i);
        p[0] += v.x; p[1] += v.y; p[2] += v.z; p[3] += v.w;
        if (PAIR) {
          const float4 w = load_of(at + TILE * 256u, i);
          q[0] += w.x; q[1] += w.y; q[2] += w.z; q[3] += w.w;
        }
      }
      finish(m0 + (u >> 4), n0 + (u & 15) * 4 + 64 * h, p, q);
    }
  }
  cluster_all();  // the sums stay until everyone has read them
}

// Up to 8 tokens in fp32: the weights' bytes are the work.  A warp streams four weight rows (two of each of a pair) and keeps
// their products with MT tokens; `share` warps of the CTA split the contraction.  At the end a butterfly that halves the
// values at every step leaves lane i with value i.  1 / 8 tokens, 4096 x 4096: 14.3 / 31 us; 10.3 of weights at
// the measured copy bandwidth.
template <int MT, bool PAIR>
__global__ void __launch_bounds__(256) few_tokens_fp32_kernel(const float *x, long long ldx, const float *w0, long long ldw0,
                                                              const float *w1, long long ldw1, int M, int N, int K,
                                                              int share, Epilogue e) {
  constexpr int kRows = PAIR ? 2 : 4, V = 4 * MT;
  __shared__ float part[8][32];
  lets_next_start();
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int at = warp % share;
  const long long n0 = ((long long)blockIdx.x * 8 + warp) / share * kRows;
  const float *w[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const long long n = n0 + r % kRows < N ? n0 + r % kRows : N - 1;
    w[r] = PAIR && r >= 2 ? w1 + n * ldw1 : w0 + n * ldw0;
  }
  float2 acc[4][MT] = {};
#pragma unroll 2
  for (int k = (at * 32 + lane) * 4; k < K; k += share * 128) {
    float4 v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const float4 *>(w[r] + k);
    float4 t[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) t[m] = *reinterpret_cast<const float4 *>(x + (m < M ? m : M - 1) * ldx + k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[r][m] = fma2(make_float2(v[r].z, v[r].w), make_float2(t[m].z, t[m].w),
                         fma2(make_float2(v[r].x, v[r].y), make_float2(t[m].x, t[m].y), acc[r][m]));
  }
  float s[V];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) s[r * MT + m] = acc[r][m].x + acc[r][m].y;
  int off = 16;
#pragma unroll
  for (int n = V; n > 1; n /= 2, off /= 2) {
    const bool up = lane & off;
#pragma unroll
    for (int j = 0; j < V / 2; ++j)
      if (j < n / 2) {
        const float give = up ? s[j] : s[j + n / 2], keep = up ? s[j + n / 2] : s[j];
        s[j] = keep + __shfl_xor_sync(0xffffffffu, give, off);
      }
  }
#pragma unroll
  for (; off > 0; off /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
  constexpr int kStride = 32 / V;  // lanes that hold one value
  if (lane % kStride == 0) part[warp][lane / kStride] = s[0];
  __syncthreads();
  if (at != 0 || lane >= (PAIR ? V / 2 : V)) return;
  float p[1] = {0.f}, q[1] = {0.f};
  for (int i = 0; i < share; ++i) {
    p[0] += part[warp + i][lane];
    if (PAIR) q[0] += part[warp + i][lane + V / 2];
  }
  const int m = lane % MT;
  const long long n = n0 + lane / MT;
  if (m >= M || n >= N) return;
  if (PAIR) finish_pair<float, 1>(e, m, (int)n, N, p, q);
  else finish_one<float, 1>(e, m, (int)n, N, p);
}

// ------------------------------------------------------------------------------ derivative of the activation
struct ActGradArgs {
  const void *dy;           // (M, N)
  Saved z;                  // (M, N) or, for a pair, g and u at columns 0 and z_up
  long long ldy, ldz;
  int z_up;
  void *dz;                 // or null: only the sums
  long long ldd;
  int d_up;
  float *partial;           // (chunks, PAIR ? 2N : N) sums over the chunk's rows, or null
  long long M, N;
  long long rows;           // rows of a chunk
  int act;
};

// VEC values of a row, and VEC kept ones, as they come from memory: nothing touches them until they are needed, so that
// loads issued ahead stay in flight
template <typename T, int VEC> struct RawRow {
  uint4 r;
  __device__ __forceinline__ void load(const T *p) { r = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = Cvt<T>::to_f(h[j]);
  }
};
template <typename T> struct RawRow<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T *p) { r = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = Cvt<T>::to_f(r); }
};
template <typename T, int VEC> struct RawKept {
  uint4 h;
  uint2 l;
  __device__ __forceinline__ void load(const Saved &s, long long off) {
    h = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(s.p) + off);
    l = *reinterpret_cast<const uint2 *>(s.low + off);
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const { kept_values(h, l, v); }
};
template <> struct RawKept<float, 4> {
  RawRow<float, 4> r;
  __device__ __forceinline__ void load(const Saved &s, long long off) { r.load(static_cast<const float *>(s.p) + off); }
  __device__ __forceinline__ void get(float (&v)[4]) const { r.get(v); }
};
template <typename T> struct RawKept<T, 1> {
  float r;
  __device__ __forceinline__ void load(const Saved &s, long long off) { r = kept_value<T>(s, off); }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = r; }
};

// CTA = 32 x VEC columns of one chunk of rows, a warp per row at a time, two rows in flight ahead of the two that are
// worked on.  One read of dy and of what was kept, one write of dz: HBM.
template <typename T, int VEC, bool PAIR>
__global__ void __launch_bounds__(256, PAIR ? 2 : 3) act_grad_kernel(const ActGradArgs a) {
  __shared__ float part[PAIR ? 2 : 1][8][32 * VEC + 1];
  lets_next_start();
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n = ((long long)blockIdx.x * 32 + lane) * VEC;
  const long long r0 = (long long)blockIdx.y * a.rows, r1 = r0 + a.rows < a.M ? r0 + a.rows : a.M;
  const bool kept = a.z.p != nullptr;
  float s0[VEC] = {}, s1[VEC] = {};
  if (n < a.N) {  // N is a multiple of VEC
    RawRow<T, VEC> dy[2];
    RawKept<T, VEC> z[2], u[2];
    long long m = r0 + warp;
    // the next row to load and to store; rows of a warp are 8 apart
    const T *dyp = static_cast<const T *>(a.dy) + m * a.ldy + n;
    long long zo = m * a.ldz + n;
    T *op = a.dz == nullptr ? nullptr : static_cast<T *>(a.dz) + m * a.ldd + n;
    const long long dys = 8 * a.ldy, zs = 8 * a.ldz, os = 8 * a.ldd;
    auto fetch = [&](int i) {
      dy[i].load(dyp);
      if (kept) z[i].load(a.z, zo);
      if (PAIR) u[i].load(a.z, zo + a.z_up);
      dyp += dys;
      zo += zs;
    };
    const int rows = m < r1 ? (int)((r1 - m + 7) / 8) : 0;  // of this warp
    if (rows > 0) fetch(0);
    if (rows > 1) fetch(1);
    for (int row = 0; row < rows; row += 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (row + i >= rows) break;
        float d[VEC], p[VEC], q[VEC], g[VEC];
        dy[i].get(d);
        if (kept) z[i].get(p);
        if (PAIR) u[i].get(q);
        if (row + i + 2 < rows) fetch(i);
        if (kept) {
          activate_grad<T, VEC>(p, g, a.act);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (PAIR) {
              p[j] *= d[j];
              d[j] *= q[j];
              s1[j] += p[j];
            }
            d[j] *= g[j];
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) s0[j] += d[j];
        if (op != nullptr) {
          store_row<T, VEC>(op, VEC > 1, VEC, d);
          if (PAIR) store_row<T, VEC>(op + a.d_up, VEC > 1, VEC, p);
          op += os;
        }
      }
    }
  }
  if (a.partial == nullptr) return;  // uniform over the grid
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    part[0][warp][lane * VEC + j] = s0[j];
    if (PAIR) part[PAIR ? 1 : 0][warp][lane * VEC + j] = s1[j];
  }
  __syncthreads();
  const long long width = PAIR ? 2 * a.N : a.N;
  for (int c = threadIdx.x; c < 32 * VEC; c += 256) {
    const long long col = (long long)blockIdx.x * 32 * VEC + c;
    if (col >= a.N) break;
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      v0 += part[0][w][c];
      if (PAIR) v1 += part[PAIR ? 1 : 0][w][c];
    }
    a.partial[blockIdx.y * width + col] = v0;
    if (PAIR) a.partial[blockIdx.y * width + a.N + col] = v1;
  }
}

// db[c] = sum over the chunks, in a fixed order.  Columns from N on belong to the second bias.
template <typename T>
__global__ void __launch_bounds__(256) bias_sum_kernel(const float *partial, int chunks, long long width, long long N,
                                                       void *db0, void *db1) {
  __shared__ float s[8][33];
  lets_next_start();
  after_previous();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + tx;
  float v = 0.f;
  if (c < width)
    for (int i = ty; i < chunks; i += 8) v += partial[i * width + c];
  s[ty][tx] = v;
  __syncthreads();
  if (ty != 0 || c >= width) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) v += s[i][tx];
  T *db = static_cast<T *>(c < N ? db0 : db1);
  if (db != nullptr) db[c < N ? c : c - N] = Cvt<T>::from_f(v);
}

// ------------------------------------------------------------------------------ relu's border in fp32
// relu's derivative jumps at 0: a pre-activation whose fp32 sum comes out on the other side of 0 than the sum itself moves dx,
// dW and db by a whole dy (one of 263,168 in one of 150 runs of 514 x 512 x 512: 1e-3 to 7e-3 of dx, where fp32 rounding leaves 2e-7).
// So the kept values near 0 are computed again in 64 bits.  Near: each of the sum's K roundings is at most 2^-24 |x_m| |w_n|,
// since no partial sum is above |x_m| |w_n|; with independent signs they add up to sqrt(K) of that, and six times as much is
// taken: for normally distributed values a share of 3e-7 K of the elements.  Only the derivative reads what is kept, so a
// forward without gradients has no such pass.  16-bit types do without: on the tensor cores 6 of 20 million values are on the
// other side at K 2048 and 31 at 8192, and the passes that find and mend them were built and cost more than they are worth there
// (16384 x 4096 x 4096 390 -> 500 us, 16384 x 768 x 2048 60 -> 90, 1024 x 4096 x 4096 31 -> 54).
// Forward that keeps its values, relu / sigmoid: 514 x 512 x 512 19.2 / 14.6 us, 1024 x 4096 x 4096 846 / 786 (810 if no value is
// near 0), 8 x 4096 x 4096 39 / 21.
//
// near_zero[m] = 6 sqrt(K) 2^-24 |x_m|, near_zero[M + n] = |w_n| (rows of values so far from 1 that their squares leave the
// range of fp32 are not looked at).  A warp a row, every operand once: HBM or L2.
template <int V>
__global__ void __launch_bounds__(256) row_size_kernel(const float *x, long long ldx, const float *w, long long ldw,
                                                       long long M, long long N, long long K, float *near_zero) {
  lets_next_start();
  after_previous();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= M + N) return;
  const float *p = row < M ? x + row * ldx : w + (row - M) * ldw;
  float s = 0.f;
#pragma unroll 4
  for (long long k = lane * V; k < K; k += 32 * V) {  // K is a multiple of V
    float v[V];
    load_row<float, V>(p + k, true, V, v);
#pragma unroll
    for (int j = 0; j < V; ++j) s = fmaf(v[j], v[j], s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) near_zero[row] = sqrtf(s) * (row < M ? 3.5762787e-7f * sqrtf((float)K) : 1.f);
}

// A warp looks at 32 columns of a row of z (M, N) at a time and takes the elements near 0 one after the other, all its lanes
// along the contraction.
template <int V>
__global__ void __launch_bounds__(256) relu_border_kernel(const float *x, long long ldx, const float *w, long long ldw,
                                                          const float *bias, float *z, long long ldz, long long M,
                                                          long long N, long long K, const float *near_zero) {
  lets_next_start();
  after_previous();
  const int lane = threadIdx.x & 31;
  const long long strips = (N + 31) / 32, all = M * strips;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * 8) {
    const long long m = i / strips, n0 = (i - m * strips) * 32, mine = n0 + lane;
    const float tau = mine < N ? near_zero[m] * near_zero[M + mine] : 0.f;  // infinite or NaN: left as it is
    const bool near = mine < N && fabsf(z[m * ldz + mine]) < tau && tau <= 3.402823466e38f;
    for (unsigned left = __ballot_sync(0xffffffffu, near); left != 0; left &= left - 1) {
      const long long n = n0 + __ffs(left) - 1;
      const float *p = x + m * ldx, *q = w + n * ldw;
      double s = 0;
#pragma unroll 4
      for (long long k = lane * V; k < K; k += 32 * V) {
        float u[V], v[V];
        load_row<float, V>(p + k, true, V, u);
        load_row<float, V>(q + k, true, V, v);
#pragma unroll
        for (int j = 0; j < V; ++j) s = fma((double)u[j], (double)v[j], s);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) z[m * ldz + n] = (float)(bias == nullptr ? s : s + (double)bias[n]);
    }
  }
}

// ------------------------------------------------------------------------------ rows on 16-byte boundaries
// dst[r][c] = src[r][c] for c < cols, rows of dst `ldd` = cols rounded up to 8 apart; 8 elements a thread.  The tensor
// cores' loads want rows that start on 16 bytes; operands with other strides (odd widths) go through this copy.
__global__ void __launch_bounds__(256) copy_rows_kernel(const uint16_t *src, long long lds, uint16_t *dst, long long ldd,
                                                        long long rows, long long cols) {
  lets_next_start();
  after_previous();
  const long long packs = ldd / 8, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * packs) return;
  const long long r = i / packs, c = (i - r * packs) * 8;
  uint16_t v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? src[r * lds + c + j] : 0;
  uint4 o;
  o.x = v[0] | (uint32_t)v[1] << 16;
  o.y = v[2] | (uint32_t)v[3] << 16;
  o.z = v[4] | (uint32_t)v[5] << 16;
  o.w = v[6] | (uint32_t)v[7] << 16;
  *reinterpret_cast<uint4 *>(dst + r * ldd + c) = o;
}

// ------------------------------------------------------------------------------ host
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Scratch in pieces out of the caller's workspace; with base null it only counts.
struct Scratch {
  char *base;
  int64_t used = 0;
  explicit Scratch(void *p) : base(static_cast<char *>(p)) {}
  void *take(int64_t bytes) {
    void *p = base == nullptr ? nullptr : base + used;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

// bytes of the kept pre-activations (fp32: and of row_size_kernel's results behind them), and their two parts in a buffer
int64_t saved_bytes(int64_t M, int64_t N, int dtype, bool pair) {
  const int64_t values = M * (pair ? 2 * N : N);
  return dtype == LA_F32 ? (values + M + N) * 4 : (values * 2 + 15) / 16 * 16 + values;
}
Saved saved_in(const void *p, int64_t rows, int64_t cols, int dtype) {
  Saved s = {const_cast<void *>(p), nullptr};
  if (p != nullptr && dtype != LA_F32)
    s.low = static_cast<uint8_t *>(const_cast<void *>(p)) + (rows * cols * 2 + 15) / 16 * 16;
  return s;
}

int epilogue_vec(const Epilogue &e, int dtype) {
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  return aligned16(e.bias[0]) && aligned16(e.bias[1]) && aligned16(e.residual) && aligned16(e.out) && aligned16(e.out2) &&
         aligned16(e.save.p) && e.ldr % per == 0 && e.ldo % per == 0 && e.lds % per == 0 && e.save_up % per == 0;
}

// Tile and splits of an fp32 product.  Tiles of 128 where the result is wider than 64 both ways and they and their splits
// fill the GPU, else of 64.  With tiles of 64 / of 128: 1024 x 1024 x 1024 76 / 57 us, 4096 x 1024 x 4096 772 / 679, 16 x 4096 x
// 4096 67 / 141.  Splits of at least 64 terms for four CTAs of 64 an SM (five fit: 30 shapes 3 % behind the quickest of 1 .. 16
// splits on average), those of a pair by pair_splits.  Those of 128, two an SM, split into the power of two, of at least 256 terms,
// that leaves the least of the last round idle: 3.1 us a step of two CTAs, 2.2 of one alone, 4 us a round beside, 10 with the
// sums (1500 x 768 x 2048 in 1, 2, 4: 156, 120, 122; 4096 x 1024 x 4096 679, 692, 748; three, 133 and 769, do not pack as two CTAs an SM).
struct SimtPlan {
  int tile, splits;
};
// Splits of a pair's tiles.  Three of its CTAs fit on an SM, but fewer clusters than that would make (142 of three: a cluster's
// SMs lie together), so their number is asked for once per device.  A step takes 1.2, 1.84 or 2.76 us with one to three CTAs on
// every SM; clusters of three and more do not spread evenly (48 CTAs 1.3, 148 2.26, 222 2.6); sums 1 us a round.  Against four CTAs
// an SM, the rule of single products (37, 74, 100, 111, 148, 185, 296 tiles of K 2048): 39 / 48 us, 71 / 79, 85 / 102, 106 / 116,
// 118 / 141, 165 / 171, 230 / 219; over 75 shapes 7 % less on average, 8 % more at most.
int pair_splits(int64_t tiles, int64_t k) {
  static bool set[64] = {false};
  static int fit[64][17];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 1;
  }
  const int64_t sms = sm_count();
  if (!set[dev]) {
    bool ok = cudaFuncSetAttribute(simt_product_kernel<64, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    for (int s = 1; s <= 16; ++s) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)s;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)s);
      cfg.blockDim = dim3(simt_threads<64>());
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      ok = ok && cudaOccupancyMaxActiveClusters(&fit[dev][s], simt_product_kernel<64, true>, &cfg) == cudaSuccess;
      if (!ok) fit[dev][s] = 0;
    }
    cudaGetLastError();
    set[dev] = true;
  }
  auto step = [&](int64_t ctas, int s) {
    if (ctas <= 0) return 0.;
    if (s <= 2) return ctas <= sms ? 1.2 : ctas <= 2 * sms ? 1.84 : 2.76;
    const double us = 0.7 + 1.56 * ctas / sms;
    return us < 1.2 ? 1.2 : us > 2.76 ? 2.76 : us;
  };
  int best = 1;
  double best_us = 1e30;
  for (int s = 1; s <= 16 && (s == 1 || k / s >= 64); ++s) {
    const int64_t at_once = fit[dev][s];
    if (at_once < 1) continue;
    const int64_t rounds = tiles / at_once, rest = tiles % at_once;
    const double us = (double)k / kStep / s * (rounds * step(at_once * s, s) + step(rest * s, s)) + (s == 1 ? 0 : rounds + 1);
    if (us < best_us) {
      best_us = us;
      best = s;
    }
  }
  return best;
}
SimtPlan simt_plan(const Product &p) {
  const int64_t k = p.K[0] + (p.segments > 1 ? p.K[1] : 0), sms = sm_count();
  if (!p.pair && p.M > 64 && p.N > 64) {
    const int64_t tiles = (p.M + 127) / 128 * ((p.N + 127) / 128);
    int best = 1;
    double best_us = 1e30;
    for (int s = 1; s <= 8 && (s == 1 || k / s >= 256); s *= 2) {
      const int64_t rounds = tiles * s / (2 * sms), rest = tiles * s % (2 * sms);
      const double step = rest == 0 ? 0 : rest <= sms && (rounds > 0 || s == 1) ? 2.2 : 3.1;
      const double us = (k / kStep / s) * (rounds * 3.1 + step) + (rounds + (rest > 0)) * (s == 1 ? 4 : 10);
      if (us < best_us) {
        best_us = us;
        best = s;
      }
    }
    if (tiles * best >= sms) return SimtPlan{128, best};
  }
  const int64_t tiles = (p.M + 63) / 64 * ((p.N + 63) / 64);
  if (p.pair) return SimtPlan{64, pair_splits(tiles, k)};
  int64_t splits = 4 * sms / tiles;
  if (splits > k / 64) splits = k / 64;
  if (splits > 16) splits = 16;
  return SimtPlan{64, splits < 1 ? 1 : (int)splits};
}

template <int TILE, bool PAIR>
int simt_launch_tile(const SimtArgs &a, int64_t grid, cudaStream_t st) {
  if (a.splits > 8) {  // clusters of more than 8 are asked for once per kernel and device
    static bool set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LA_ERR_CUDA;
    if (!set[dev]) {
      const cudaError_t e =
          cudaFuncSetAttribute(simt_product_kernel<TILE, PAIR>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) {
        note_cuda_error(e, "cluster size");
        return LA_ERR_CUDA;
      }
      set[dev] = true;
    }
  }
  return launch_early(simt_product_kernel<TILE, PAIR>, dim3((unsigned)grid), simt_threads<TILE>(), 0, st,
                      a.splits > 1 ? a.splits : 0, a);
}

int simt_launch(const Product &p, const SimtPlan &plan, cudaStream_t st) {
  SimtArgs a = {};
  a.M = p.M; a.N = p.N; a.e = p.e;
  for (int s = 0; s < 2; ++s) {
    a.a[s] = p.a[s]; a.b[s] = p.b[s];
    a.K[s] = s < p.segments ? p.K[s] : 0;
    a.steps[s] = (a.K[s] + kStep - 1) / kStep;
    a.vec_a[s] = aligned16(p.a[s].p) && p.a[s].ld % 4 == 0;
    a.vec_b[s] = aligned16(p.b[s].p) && p.b[s].ld % 4 == 0;
  }
  const int64_t mt = (p.M + plan.tile - 1) / plan.tile;
  a.n_tiles = (int)((p.N + plan.tile - 1) / plan.tile);
  a.splits = plan.splits;
  const int64_t grid = mt * a.n_tiles * plan.splits;
  if (grid > INT32_MAX) return LA_ERR_TOO_LARGE;
  if (plan.tile == 128) return simt_launch_tile<128, false>(a, grid, st);
  return p.pair ? simt_launch_tile<64, true>(a, grid, st) : simt_launch_tile<64, false>(a, grid, st);
}

// Whether a product is few_tokens_fp32_kernel's kind, and the launch: enough warps to fill the GPU, each with 256 terms.
bool few_fp32_fit(const Product &p) {
  auto on16 = [](const Operand &o) { return !o.mn_major && aligned16(o.p) && o.ld % 4 == 0; };
  return p.M <= 8 && p.segments == 1 && p.K[0] % 4 == 0 && on16(p.a[0]) && on16(p.b[0]) && (!p.pair || on16(p.b[1]));
}
template <int MT>
int few_fp32_launch(const Product &p, cudaStream_t st) {
  const int64_t groups = (p.N + (p.pair ? 1 : 3)) / (p.pair ? 2 : 4);
  int share = 1;
  while (share < 8 && groups * share < 16 * (int64_t)sm_count() && p.K[0] >= 512 * share) share *= 2;
  const unsigned grid = (unsigned)((groups * share + 7) / 8);
  Epilogue e = p.e;
  e.vec = 0;  // one value a thread
  const float *x = static_cast<const float *>(p.a[0].p), *w0 = static_cast<const float *>(p.b[0].p),
              *w1 = static_cast<const float *>(p.b[1].p);
  return launch_early(p.pair ? few_tokens_fp32_kernel<MT, true> : few_tokens_fp32_kernel<MT, false>, dim3(grid), 256, 0, st, 0, x,
                      p.a[0].ld, w0, p.b[0].ld, w1, p.b[1].ld, (int)p.M, (int)p.N, (int)p.K[0], share, e);
}

// The operand as the tensor cores can read it: itself, or its copy with rows on 16-byte boundaries.
int readable(Operand &o, int64_t rows, int64_t cols, int dtype, Scratch &s, cudaStream_t st) {
  if (dtype == LA_F32 || (aligned16(o.p) && o.ld % 8 == 0)) return LA_OK;
  const int64_t ld = (cols + 7) / 8 * 8;
  uint16_t *dst = static_cast<uint16_t *>(s.take(rows * ld * 2));
  if (s.base != nullptr) {
    const int64_t grid = (rows * (ld / 8) + 255) / 256;
    if (grid > INT32_MAX) return LA_ERR_TOO_LARGE;
    const int rc = launch_early(copy_rows_kernel, dim3((unsigned)grid), 256, 0, st, 0, static_cast<const uint16_t *>(o.p), o.ld,
                                dst, ld, rows, cols);
    if (rc != LA_OK) return rc;
  }
  o.p = dst;
  o.ld = ld;
  return LA_OK;
}

// One product with its epilogue.  With s.base null only the scratch is counted.
int product(Product p, int dtype, Scratch s, int64_t &need, cudaStream_t st) {
  p.e.vec = epilogue_vec(p.e, dtype);
  if (few_tokens_fit(p, dtype)) {
    if (s.used > need) need = s.used;
    return s.base == nullptr ? LA_OK : few_tokens_launch(p, dtype, st);
  }
  if (dtype == LA_F32 && few_fp32_fit(p)) {
    if (s.used > need) need = s.used;
    if (s.base == nullptr) return LA_OK;
    if (p.M == 1) return few_fp32_launch<1>(p, st);
    if (p.M == 2) return few_fp32_launch<2>(p, st);
    return p.M <= 4 ? few_fp32_launch<4>(p, st) : few_fp32_launch<8>(p, st);
  }
  if (dtype == LA_F32) {
    if (s.used > need) need = s.used;
    if (s.base == nullptr) return LA_OK;
    return simt_launch(p, simt_plan(p), st);
  }
  const GemmPlan plan = gemm_plan(p.M, p.N, p.K[0], p.segments > 1 ? p.K[1] : 0, p.pair != 0);
  float *partial = plan.partial_bytes > 0 ? static_cast<float *>(s.take(plan.partial_bytes)) : nullptr;
  if (s.used > need) need = s.used;
  if (s.base == nullptr) return LA_OK;
  return gemm_launch(p, plan, partial, dtype, st);
}

template <typename T, int VEC>
int act_grad_launch(const ActGradArgs &a, bool pair, int chunks, cudaStream_t st) {
  const dim3 grid((unsigned)((a.N + 32 * VEC - 1) / (32 * VEC)), (unsigned)chunks);
  return launch_early(pair ? act_grad_kernel<T, VEC, true> : act_grad_kernel<T, VEC, false>, grid, 256, 0, st, 0, a);
}

// chunks of rows of act_grad_kernel: one wave of the CTAs that fit, at least 8 rows (one per warp) a chunk
int act_grad_chunks(int64_t M, int64_t N, int dtype, bool pair) {
  const int64_t cols = 32 * (16 / (int64_t)dtype_size(dtype));
  int64_t chunks = (pair ? 2 : 3) * (int64_t)sm_count() / ((N + cols - 1) / cols);
  if (chunks > (M + 7) / 8) chunks = (M + 7) / 8;
  if (chunks > 4096) chunks = 4096;
  return chunks < 1 ? 1 : (int)chunks;
}

int act_grad(ActGradArgs a, bool pair, int chunks, void *db0, void *db1, int dtype, cudaStream_t st) {
  a.rows = (a.M + chunks - 1) / chunks;
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  const bool vec = aligned16(a.dy) && aligned16(a.z.p) && aligned16(a.dz) && a.ldy % per == 0 && a.ldz % per == 0 &&
                   a.ldd % per == 0 && a.z_up % per == 0 && a.d_up % per == 0 && a.N % per == 0;
  int rc = LA_ERR_UNSUPPORTED;
  switch (dtype) {
    case LA_F32: rc = vec ? act_grad_launch<float, 4>(a, pair, chunks, st) : act_grad_launch<float, 1>(a, pair, chunks, st); break;
    case LA_BF16:
      rc = vec ? act_grad_launch<__nv_bfloat16, 8>(a, pair, chunks, st) : act_grad_launch<__nv_bfloat16, 1>(a, pair, chunks, st);
      break;
    case LA_F16: rc = vec ? act_grad_launch<__half, 8>(a, pair, chunks, st) : act_grad_launch<__half, 1>(a, pair, chunks, st); break;
  }
  if (rc != LA_OK || a.partial == nullptr) return rc;
  const long long width = pair ? 2 * a.N : a.N;
  auto *kernel = dtype == LA_F32 ? bias_sum_kernel<float> : (dtype == LA_BF16 ? bias_sum_kernel<__nv_bfloat16> : bias_sum_kernel<__half>);
  return launch_early(kernel, dim3((unsigned)((width + 31) / 32)), 256, 0, st, 0, a.partial, chunks, width, a.N, db0, db1);
}

// The kept values z (row stride ldz) of an fp32 relu, those near 0 in 64 bits.
int relu_border(const float *x, int64_t ldx, const float *w, int64_t ldw, const float *bias, float *z, int64_t ldz, int64_t M,
                int64_t N, int64_t K, cudaStream_t st) {
  float *near_zero = z + M * ldz;
  const int64_t rows = (M + N + 7) / 8, strips = (M * ((N + 31) / 32) + 7) / 8, most = 16 * (int64_t)sm_count();
  const bool vec = aligned16(x) && aligned16(w) && (K | ldx | ldw) % 4 == 0;
  const int rc = launch_early(vec ? row_size_kernel<4> : row_size_kernel<1>, dim3((unsigned)rows), 256, 0, st, 0, x, ldx, w,
                              ldw, M, N, K, near_zero);
  if (rc != LA_OK) return rc;
  return launch_early(vec ? relu_border_kernel<4> : relu_border_kernel<1>, dim3((unsigned)(strips < most ? strips : most)), 256,
                      0, st, 0, x, ldx, w, ldw, bias, z, ldz, M, N, K, near_zero);
}

struct FwdArgs {
  const void *x;
  int64_t ldx;
  const void *w[2];
  int64_t ldw[2];
  const void *bias[2], *residual;
  int64_t ldr;
  void *out, *save;
  int64_t M, N, K;
  int dtype, act, pair;
};

int forward(const FwdArgs &f, Scratch s, int64_t &need, cudaStream_t st) {
  Product p = {};
  p.a[0] = Operand{f.x, f.ldx, 0};
  p.b[0] = Operand{f.w[0], f.ldw[0], 0};
  p.b[1] = Operand{f.w[1], f.ldw[1], 0};
  int rc = readable(p.a[0], f.M, f.K, f.dtype, s, st);
  if (rc == LA_OK) rc = readable(p.b[0], f.N, f.K, f.dtype, s, st);
  if (rc == LA_OK && f.pair) rc = readable(p.b[1], f.N, f.K, f.dtype, s, st);
  if (rc != LA_OK) return rc;
  p.K[0] = f.K;
  p.segments = 1;
  p.pair = f.pair;
  p.M = f.M; p.N = f.N;
  p.e.bias[0] = f.bias[0]; p.e.bias[1] = f.bias[1];
  p.e.residual = f.residual; p.e.ldr = f.ldr;
  p.e.out = f.out; p.e.ldo = f.N; p.e.split = INT32_MAX; p.e.live = (int)f.M;
  p.e.save = saved_in(f.save, f.M, f.pair ? 2 * f.N : f.N, f.dtype); p.e.lds = f.pair ? 2 * f.N : f.N; p.e.save_up = f.pair ? (int)f.N : 0;
  p.e.act = f.act;
  rc = product(p, f.dtype, s, need, st);
  if (rc != LA_OK || s.base == nullptr || f.save == nullptr || f.dtype != LA_F32 || f.act != kActRelu) return rc;
  return relu_border(static_cast<const float *>(f.x), f.ldx, static_cast<const float *>(f.w[0]), f.ldw[0],
                     static_cast<const float *>(f.bias[0]), static_cast<float *>(f.save), p.e.lds, f.M, f.N, f.K, st);
}

struct BwdArgs {
  const void *x;
  int64_t ldx;
  const void *w[2];
  int64_t ldw[2];
  const void *saved, *dy;
  int64_t ldy;
  void *dx, *dw[2], *db[2];
  int64_t M, N, K;
  int dtype, act, pair;
};

int backward(const BwdArgs &f, Scratch s, int64_t &need, cudaStream_t st) {
  const bool run = s.base != nullptr;
  const int64_t es = (int64_t)dtype_size(f.dtype);
  const bool want_dw = f.dw[0] != nullptr, want_db = f.db[0] != nullptr || f.db[1] != nullptr;
  const bool products = f.dx != nullptr || want_dw;
  // dz: dy itself without an activation, else a pass of its own; dg and du side by side, each on a 16-byte boundary
  const int64_t np = (f.N + 7) / 8 * 8;
  const bool own_dz = f.pair || f.act != kActNone;
  Operand dz = {f.dy, f.ldy, 0};
  if (own_dz && products) dz = Operand{s.take(f.M * (f.pair ? 2 * np : np) * es), f.pair ? 2 * np : np, 0};
  Operand x = {f.x, f.ldx, 1}, w[2] = {{f.w[0], f.ldw[0], 1}, {f.w[1], f.ldw[1], 1}};
  int rc = LA_OK;
  if (!own_dz && products) rc = readable(dz, f.M, f.N, f.dtype, s, st);
  if (rc == LA_OK && want_dw) rc = readable(x, f.M, f.K, f.dtype, s, st);
  for (int i = 0; i < (f.pair ? 2 : 1) && f.dx != nullptr && rc == LA_OK; ++i)
    rc = readable(w[i], f.N, f.K, f.dtype, s, st);
  if (rc != LA_OK) return rc;
  const int chunks = act_grad_chunks(f.M, f.N, f.dtype, f.pair != 0);
  float *sums = want_db ? static_cast<float *>(s.take((int64_t)chunks * (f.pair ? 2 : 1) * f.N * 4)) : nullptr;
  if (run && ((own_dz && products) || want_db)) {
    ActGradArgs a = {};
    a.dy = f.dy; a.ldy = f.ldy;
    if (own_dz) {
      a.z = saved_in(f.saved, f.M, f.pair ? 2 * f.N : f.N, f.dtype);
      a.ldz = f.pair ? 2 * f.N : f.N;
      a.z_up = f.pair ? (int)f.N : 0;
    }
    if (own_dz && products) {
      a.dz = const_cast<void *>(dz.p);
      a.ldd = dz.ld;
      a.d_up = f.pair ? (int)np : 0;
    }
    a.partial = sums;
    a.M = f.M; a.N = f.N; a.act = f.act;
    if ((rc = act_grad(a, f.pair != 0, chunks, f.db[0], f.db[1], f.dtype, st)) != LA_OK) return rc;
  }
  const void *dz_up = dz.p == nullptr ? nullptr : static_cast<const char *>(dz.p) + np * es;
  if (f.dx != nullptr) {
    Product p = {};
    p.a[0] = dz;
    p.a[1] = Operand{dz_up, dz.ld, 0};
    p.b[0] = w[0];
    p.b[1] = w[1];
    p.K[0] = f.N; p.K[1] = f.pair ? f.N : 0;
    p.segments = f.pair ? 2 : 1;
    p.M = f.M; p.N = f.K;
    p.e.out = f.dx; p.e.ldo = f.K; p.e.split = INT32_MAX; p.e.live = (int)f.M;
    if ((rc = product(p, f.dtype, s, need, st)) != LA_OK) return rc;
  }
  if (want_dw) {
    Product p = {};
    p.a[0] = Operand{dz.p, dz.ld, 1};
    p.b[0] = x;
    p.K[0] = f.M;
    p.segments = 1;
    p.M = f.pair ? np + f.N : f.N;  // a pair: rows [0, N) are dWg, rows [np, np + N) dWu
    p.N = f.K;
    p.e.out = f.dw[0]; p.e.out2 = f.dw[1]; p.e.ldo = f.K;
    p.e.split = f.pair ? (int)np : (int)f.N;
    p.e.live = (int)f.N;
    if ((rc = product(p, f.dtype, s, need, st)) != LA_OK) return rc;
  }
  if (s.used > need) need = s.used;
  return LA_OK;
}

int check_common(int64_t M, int64_t N, int64_t K, int dtype, int act) {
  cudaGetLastError();
  if (M <= 0 || N <= 0 || K <= 0) return LA_ERR_BAD_SHAPE;
  if (!(dtype == LA_F32 || dtype == LA_BF16 || dtype == LA_F16)) return LA_ERR_UNSUPPORTED;
  if (act < kActNone || act > kActGelu) return LA_ERR_UNSUPPORTED;
  if (M > (1 << 30) || N > (1 << 28) || K > (1 << 28)) return LA_ERR_TOO_LARGE;
  return LA_OK;
}

int check_fwd(const FwdArgs &f) {
  if (f.x == nullptr || f.w[0] == nullptr || (f.pair && f.w[1] == nullptr)) return LA_ERR_NULL_POINTER;
  const int rc = check_common(f.M, f.N, f.K, f.dtype, f.act);
  if (rc != LA_OK) return rc;
  if (f.ldx < f.K || f.ldw[0] < f.K || (f.pair && f.ldw[1] < f.K) || (f.residual != nullptr && f.ldr < f.N))
    return LA_ERR_BAD_SHAPE;
  return LA_OK;
}
int check_bwd(const BwdArgs &f) {
  if (f.x == nullptr || f.w[0] == nullptr || (f.pair && f.w[1] == nullptr) || f.dy == nullptr) return LA_ERR_NULL_POINTER;
  const int rc = check_common(f.M, f.N, f.K, f.dtype, f.act);
  if (rc != LA_OK) return rc;
  if ((f.pair || f.act != kActNone) && f.saved == nullptr) return LA_ERR_NULL_POINTER;
  if (f.pair && (f.dw[0] == nullptr) != (f.dw[1] == nullptr)) return LA_ERR_NULL_POINTER;
  if (f.ldx < f.K || f.ldw[0] < f.K || (f.pair && f.ldw[1] < f.K) || f.ldy < f.N) return LA_ERR_BAD_SHAPE;
  return LA_OK;
}

int check_scratch(int64_t need, void *workspace, int64_t workspace_bytes) {
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return LA_ERR_WORKSPACE;
  if (need > 0 && !aligned16(workspace)) return LA_ERR_MISALIGNED;
  return LA_OK;
}

// a base for calls that need no scratch: never read, only told apart from the counting run
char g_no_scratch[16];

int run_fwd(const FwdArgs &f, void *workspace, int64_t workspace_bytes, void *stream) {
  int rc = check_fwd(f);
  if (rc != LA_OK) return rc;
  if (f.out == nullptr) return LA_ERR_NULL_POINTER;
  int64_t need = 0;
  rc = forward(f, Scratch(nullptr), need, nullptr);  // counts the scratch
  if (rc == LA_OK) rc = check_scratch(need, workspace, workspace_bytes);
  if (rc != LA_OK) return rc;
  return forward(f, Scratch(need > 0 ? workspace : g_no_scratch), need, static_cast<cudaStream_t>(stream));
}
int run_bwd(const BwdArgs &f, void *workspace, int64_t workspace_bytes, void *stream) {
  int rc = check_bwd(f);
  if (rc != LA_OK) return rc;
  int64_t need = 0;
  rc = backward(f, Scratch(nullptr), need, nullptr);
  if (rc == LA_OK) rc = check_scratch(need, workspace, workspace_bytes);
  if (rc != LA_OK) return rc;
  return backward(f, Scratch(need > 0 ? workspace : g_no_scratch), need, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace lin
}  // namespace la

using namespace la;
using namespace la::lin;

extern "C" {

int64_t la_linear_saved_bytes(int64_t M, int64_t N, int dtype, int pair) {
  const int rc = check_common(M, N, 1, dtype, kActNone);
  return rc != LA_OK ? rc : saved_bytes(M, N, dtype, pair != 0);
}

int64_t la_linear_fwd_workspace_bytes(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *weight_up,
                                      int64_t ldw_up, int64_t M, int64_t N, int64_t K, int dtype) {
  FwdArgs f = {};
  f.x = x; f.ldx = ldx;
  f.w[0] = weight; f.ldw[0] = ldw; f.w[1] = weight_up; f.ldw[1] = ldw_up;
  f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.pair = weight_up != nullptr;
  int64_t need = 0;
  const int rc = check_fwd(f);
  if (rc != LA_OK) return rc;
  forward(f, Scratch(nullptr), need, nullptr);
  return need;
}

int la_linear_fwd(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const void *residual,
                  int64_t ldr, void *y, void *z, void *workspace, int64_t workspace_bytes, int64_t M, int64_t N, int64_t K,
                  int dtype, int act, void *stream) {
  FwdArgs f = {};
  f.x = x; f.ldx = ldx; f.w[0] = weight; f.ldw[0] = ldw; f.bias[0] = bias;
  f.residual = residual; f.ldr = residual == nullptr ? 0 : ldr;
  f.out = y; f.save = z; f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.act = act;
  return run_fwd(f, workspace, workspace_bytes, stream);
}

int la_gated_linear_fwd(const void *x, int64_t ldx, const void *w_gate, int64_t ld_gate, const void *w_up, int64_t ld_up,
                        const void *b_gate, const void *b_up, void *h, void *gu, void *workspace, int64_t workspace_bytes,
                        int64_t M, int64_t N, int64_t K, int dtype, int act, void *stream) {
  FwdArgs f = {};
  f.x = x; f.ldx = ldx; f.w[0] = w_gate; f.ldw[0] = ld_gate; f.w[1] = w_up; f.ldw[1] = ld_up;
  f.bias[0] = b_gate; f.bias[1] = b_up;
  f.out = h; f.save = gu; f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.act = act; f.pair = 1;
  return run_fwd(f, workspace, workspace_bytes, stream);
}

int64_t la_linear_bwd_workspace_bytes(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *weight_up,
                                      int64_t ldw_up, const void *d_y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                                      int dtype, int act, int want_dx, int want_dw, int want_db) {
  static char any[16];  // stands for an output that is wanted
  BwdArgs f = {};
  f.x = x; f.ldx = ldx; f.w[0] = weight; f.ldw[0] = ldw; f.w[1] = weight_up; f.ldw[1] = ldw_up;
  f.pair = weight_up != nullptr;
  f.saved = any; f.dy = d_y; f.ldy = ldy;
  f.dx = want_dx ? any : nullptr;
  f.dw[0] = f.dw[1] = want_dw ? any : nullptr;
  f.db[0] = want_db ? any : nullptr;
  f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.act = act;
  int64_t need = 0;
  const int rc = check_bwd(f);
  if (rc != LA_OK) return rc;
  backward(f, Scratch(nullptr), need, nullptr);
  return need;
}

int la_linear_bwd(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *z, const void *d_y, int64_t ldy,
                  void *dx, void *dweight, void *dbias, void *workspace, int64_t workspace_bytes, int64_t M, int64_t N,
                  int64_t K, int dtype, int act, void *stream) {
  BwdArgs f = {};
  f.x = x; f.ldx = ldx; f.w[0] = weight; f.ldw[0] = ldw; f.saved = z; f.dy = d_y; f.ldy = ldy;
  f.dx = dx; f.dw[0] = dweight; f.db[0] = dbias;
  f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.act = act;
  return run_bwd(f, workspace, workspace_bytes, stream);
}

int la_gated_linear_bwd(const void *x, int64_t ldx, const void *w_gate, int64_t ld_gate, const void *w_up, int64_t ld_up,
                        const void *gu, const void *d_h, int64_t ldh, void *dx, void *dw_gate, void *dw_up, void *db_gate,
                        void *db_up, void *workspace, int64_t workspace_bytes, int64_t M, int64_t N, int64_t K, int dtype,
                        int act, void *stream) {
  BwdArgs f = {};
  f.x = x; f.ldx = ldx; f.w[0] = w_gate; f.ldw[0] = ld_gate; f.w[1] = w_up; f.ldw[1] = ld_up;
  f.saved = gu; f.dy = d_h; f.ldy = ldh;
  f.dx = dx; f.dw[0] = dw_gate; f.dw[1] = dw_up; f.db[0] = db_gate; f.db[1] = db_up;
  f.M = M; f.N = N; f.K = K; f.dtype = dtype; f.act = act; f.pair = 1;
  return run_bwd(f, workspace, workspace_bytes, stream);
}

}  // extern "C"
