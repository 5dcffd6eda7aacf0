// Norms of queries and keys for each head, with the position rotation in the same pass: what stands
// in front of the attention in a block.  Per row (token, head) of D features, in fp32:
//
//   s = 1 / sqrt(sum x^2 + eps)            y = c x s (.) w
//   a_i = position * freq_i                for the pairs (lo, hi) of the first R features,
//   out_lo = y_lo cos a_i - y_hi sin a_i   (i, i + R/2) or, interleaved, (2i, 2i + 1)
//   out_hi = y_hi cos a_i + y_lo sin a_i   features from R on pass
//
// backward, with dy = the output's gradient rotated by -a, xh = x s, g = c w (.) dy:
//
//   dx = s (g - xh sum(g xh))              dw = sum over rows of c xh (.) dy
//
// Pure HBM streaming: every row is read once and written once (backward: two reads, one write).
//
// A row belongs to LPR lanes; a lane holds N = NP x VEC "pairs", i.e. N low and N high features, so that
// the partner of every feature sits in the same lane and the rotation needs no exchange; the two sums of
// squares / products take log2(LPR) shuffles.  A warp owns TPW tokens and walks a chunk of their heads:
// the angles of a token are found once, the warp's lanes sharing the pairs, and stay in registers for all
// heads.  An angle is position * freq in double, in turns, reduced to a fraction of a turn before it
// becomes fp32: exact to 2^-24 turns for positions up to 2^28, where fp32 products are off by whole turns.
// The weight gradient stays in registers over all rows of a lane, and leaves as one partial row per CTA,
// which a second kernel adds in a fixed order.
#include "common.cuh"

namespace la {
namespace {

constexpr int kMaxD = 512;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMaxCtas = 2048;  // partial rows of the weight gradients

struct QkArgs {
  const void *x[2];           // q, k
  long long sb[2], sn[2], sh[2];
  const void *w[2];           // (D) or null
  int w16;                    // weights have the type of q and k (fp32 otherwise)
  const void *d_out[2];       // backward: gradients of the outputs, contiguous
  void *out[2];               // forward: outputs; backward: dq, dk; contiguous
  float *partial[2];          // backward: (CTAs, D) partial weight gradients or null
  int heads[2];
  int chunk[2];               // heads a warp works on at a time
  int tpw[2], tpw_log2[2];    // tokens a warp works on side by side
  long long items[2];         // (token group, head chunk) pairs
  int chunks[2];
  int ctas[2];                // CTAs on q, then CTAs on k
  const int64_t *pos;         // (B, N) by strides or null
  long long pos_sb, pos_sn, offset;
  const int64_t *cu;          // null or M + 1 boundaries
  int M;
  long long T;                // B * N
  int N, D, R;
  float c, eps;
  double freq[kMaxD / 2];     // turns per position
};

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };
template <typename T, int VEC> struct Pack {
  typedef typename Raw<VEC * (int)sizeof(T)>::type R;
  static __device__ __forceinline__ void unpack(const R &raw, float *v) {
    const T *h = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = Cvt<T>::to_f(h[j]);
  }
  static __device__ __forceinline__ R pack(const float *v) {
    R raw;
    T *h = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] = Cvt<T>::from_f(v[j]);
    return raw;
  }
};

template <int LPR>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// position of token t of sequence b / of a packed stream
__device__ __forceinline__ long long position_of(const QkArgs &a, long long t) {
  if (a.cu != nullptr) {
    int lo = 0, hi = a.M;  // largest i with cu[i] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(a.cu + mid) <= t) lo = mid; else hi = mid - 1;
    }
    return t - __ldg(a.cu + lo) + a.offset;
  }
  const long long b = t / a.N, n = t - b * a.N;
  if (a.pos != nullptr) return __ldg(a.pos + b * a.pos_sb + n * a.pos_sn) + a.offset;
  return n + a.offset;
}

// INTER: interleaved pairs.  VEC > 1: pack p of lane l (p LPR + l = j) is the low features [j VEC, +VEC) of the
// first half of the rotated (or of the passing) features and the matching high ones; with INTER the "low" and
// "high" packs are simply the first and second half of the row, and pairs are neighbours inside a pack.
// VEC == 1: any D, R and alignment, INTER read from `inter`.
template <typename T, bool BWD, bool INTER, int VEC, int LPR, int NP>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const __grid_constant__ QkArgs a, const int inter) {
  typedef Pack<T, VEC> P;
  typedef typename P::R R;
  constexpr int N = VEC * NP, RPW = 32 / LPR;
  constexpr int kAngles = 32 * N;  // RPW rows x LPR lanes x N pairs
  __shared__ float s_cos[kWarps][kAngles], s_sin[kWarps][kAngles];
  __shared__ double s_freq[kMaxD / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % LPR, sub = lane / LPR;
  const int which = blockIdx.x >= (unsigned)a.ctas[0];
  const int cta = which ? blockIdx.x - a.ctas[0] : blockIdx.x;
  const int H = a.heads[which], D = a.D, half = a.R >> 1;
  const int pairs = (D + 1) >> 1;
  for (int i = threadIdx.x; i < half; i += kThreads) s_freq[i] = a.freq[i];
  __syncthreads();

  // features of the lane's packs (one low, one high), and which exist
  int f_lo[NP], f_hi[NP];
  bool on_lo[NP], on_hi[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int j = (p * LPR + gl) * VEC;
    on_lo[p] = j < pairs;
    if (VEC == 1 ? inter != 0 : INTER) {
      f_lo[p] = VEC == 1 ? 2 * j : j;
      f_hi[p] = VEC == 1 ? 2 * j + 1 : j + (D >> 1);
    } else if (j < half) {
      f_lo[p] = j;
      f_hi[p] = j + half;
    } else {
      f_lo[p] = j + half;
      f_hi[p] = j + half + ((D - a.R + 1) >> 1);
    }
    on_hi[p] = on_lo[p] && f_hi[p] < D;
  }
  float w_lo[N], w_hi[N], dw_lo[N], dw_hi[N];
  const void *wp = a.w[which];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = i / VEC, j = i % VEC;
    w_lo[i] = w_hi[i] = a.c;
    if (wp != nullptr) {
      if (on_lo[p])
        w_lo[i] *= a.w16 ? Cvt<T>::to_f(static_cast<const T *>(wp)[f_lo[p] + j]) : static_cast<const float *>(wp)[f_lo[p] + j];
      if (on_hi[p])
        w_hi[i] *= a.w16 ? Cvt<T>::to_f(static_cast<const T *>(wp)[f_hi[p] + j]) : static_cast<const float *>(wp)[f_hi[p] + j];
    }
    dw_lo[i] = dw_hi[i] = 0.f;
  }
  const T *xp = static_cast<const T *>(a.x[which]);
  const T *dp = BWD ? static_cast<const T *>(a.d_out[which]) : nullptr;
  T *op = static_cast<T *>(a.out[which]);
  const int tpw = a.tpw[which], rpt = RPW >> a.tpw_log2[which];  // rows of a token side by side
  const int tsub = sub / rpt, hsub = sub - tsub * rpt;
  const R zero = {};
  R r_lo[NP], r_hi[NP], d_lo[NP], d_hi[NP];

  for (long long item = (long long)cta * kWarps + warp; item < a.items[which];
       item += (long long)a.ctas[which] * kWarps) {
    const long long group = item / a.chunks[which];
    const int h0 = (int)(item - group * a.chunks[which]) * a.chunk[which];
    const int h1 = min(h0 + a.chunk[which], H);
    const long long t = group * tpw + tsub;
    const bool t_on = t < a.T;
    const long long tc = t_on ? t : a.T - 1;
    const long long b = tc / a.N, n = tc - b * a.N;
    const T *xrow = xp + b * a.sb[which] + n * a.sn[which];
    const long long crow = tc * H;  // rows of the contiguous tensors
    // rows past the chunk or the last token: a row that exists, with a gradient of 0, so that such a lane adds
    // 0 times a value of that row to the weight's gradient
    auto fetch = [&](int h) {
      const bool in = t_on && h < h1;
      const int hc = h < h1 ? h : h1 - 1;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const T *x = xrow + hc * a.sh[which];
        r_lo[p] = on_lo[p] ? *reinterpret_cast<const R *>(x + f_lo[p]) : zero;
        r_hi[p] = on_hi[p] ? *reinterpret_cast<const R *>(x + f_hi[p]) : zero;
        if (BWD) {
          const T *d = dp + (crow + hc) * D;
          d_lo[p] = on_lo[p] && in ? *reinterpret_cast<const R *>(d + f_lo[p]) : zero;
          d_hi[p] = on_hi[p] && in ? *reinterpret_cast<const R *>(d + f_hi[p]) : zero;
        }
      }
    };
    fetch(h0 + hsub);
    // the angles of the warp's tokens, each found by one lane
    for (int i = lane; i < tpw * half; i += 32) {
      const int ts = i / half, pr = i - ts * half;
      const long long tt = group * tpw + ts;
      double turns = (double)position_of(a, tt < a.T ? tt : a.T - 1) * s_freq[pr];
      turns -= rint(turns);
      float sn, cs;
      sincospif(2.f * (float)turns, &sn, &cs);
      s_cos[warp][i] = cs;
      s_sin[warp][i] = sn;
    }
    __syncwarp();
    float cs[N], sn[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i / VEC, j = i % VEC;
      int pr = (p * LPR + gl) * VEC + j;   // the lane's i-th pair
      if (INTER && VEC > 1)                // first half of the values: pairs of the low pack, then of the high pack
        pr = ((j < VEC / 2 ? f_lo[p] : f_hi[p]) >> 1) + j % (VEC / 2 > 0 ? VEC / 2 : 1);
      const bool rot = pr < half;
      cs[i] = rot ? s_cos[warp][tsub * half + pr] : 1.f;
      sn[i] = rot ? s_sin[warp][tsub * half + pr] : 0.f;
    }
    __syncwarp();  // the next item's angles overwrite these

    for (int hb = h0; hb < h1; hb += rpt) {
      const int h = hb + hsub;
      const bool live = t_on && h < h1;
      float xl[N], xh[N], gl_[N], gh_[N];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        P::unpack(r_lo[p], xl + p * VEC);
        P::unpack(r_hi[p], xh + p * VEC);
        if (BWD) {
          P::unpack(d_lo[p], gl_ + p * VEC);
          P::unpack(d_hi[p], gh_ + p * VEC);
        }
      }
      if (hb + rpt < h1) fetch(h + rpt);
      float s2 = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s2 += xl[i] * xl[i] + xh[i] * xh[i];
      // (u, v) rotated by the i-th pair's angle (backward: by its negative)
      auto rotate = [&](float *lo, float *hi) {
        if (INTER && VEC > 1) {
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              const int e = p * VEC + 2 * j, cl = p * VEC + j, ch = cl + VEC / 2;
              const float s_l = BWD ? -sn[cl] : sn[cl], s_h = BWD ? -sn[ch] : sn[ch];
              const float a0 = lo[e], a1 = lo[e + 1], b0 = hi[e], b1 = hi[e + 1];
              lo[e] = a0 * cs[cl] - a1 * s_l;
              lo[e + 1] = a1 * cs[cl] + a0 * s_l;
              hi[e] = b0 * cs[ch] - b1 * s_h;
              hi[e + 1] = b1 * cs[ch] + b0 * s_h;
            }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float s = BWD ? -sn[i] : sn[i], u = lo[i], v = hi[i];
            lo[i] = u * cs[i] - v * s;
            hi[i] = v * cs[i] + u * s;
          }
        }
      };
      if (!BWD) {
        const float rs = rsqrtf(lane_sum<LPR>(s2) + a.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          xl[i] = xl[i] * rs * w_lo[i];
          xh[i] = xh[i] * rs * w_hi[i];
        }
        rotate(xl, xh);
      } else {
        rotate(gl_, gh_);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) dot += gl_[i] * w_lo[i] * xl[i] + gh_[i] * w_hi[i] * xh[i];
        const float rs = rsqrtf(lane_sum<LPR>(s2) + a.eps);
        dot = lane_sum<LPR>(dot) * rs;  // sum of g xh
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float nl = xl[i] * rs, nh = xh[i] * rs;
          dw_lo[i] += nl * gl_[i];
          dw_hi[i] += nh * gh_[i];
          xl[i] = (gl_[i] * w_lo[i] - nl * dot) * rs;
          xh[i] = (gh_[i] * w_hi[i] - nh * dot) * rs;
        }
      }
      if (live) {
        T *o = op + (crow + h) * D;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          if (on_lo[p]) *reinterpret_cast<R *>(o + f_lo[p]) = P::pack(xl + p * VEC);
          if (on_hi[p]) *reinterpret_cast<R *>(o + f_hi[p]) = P::pack(xh + p * VEC);
        }
      }
    }
  }
  if (BWD && a.partial[which] != nullptr) {  // uniform over the CTA
    __shared__ float part[kWarps][2 * LPR * N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        dw_lo[i] += __shfl_xor_sync(0xffffffffu, dw_lo[i], o);
        dw_hi[i] += __shfl_xor_sync(0xffffffffu, dw_hi[i], o);
      }
      const int p = i / VEC, j = i % VEC;
      if (sub == 0) {
        if (on_lo[p]) part[warp][f_lo[p] + j] = dw_lo[i];
        if (on_hi[p]) part[warp][f_hi[p] + j] = dw_hi[i];
      }
    }
    __syncthreads();
    for (int f = threadIdx.x; f < D; f += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) s += part[k][f];
      a.partial[which][(long long)cta * D + f] = s * a.c;
    }
  }
}

// dw[f] = sum over the CTAs' partial rows, in a fixed order.  Block (32 features, 32 row slots); grid.y = q, k.
template <typename T>
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float *pq, const float *pk, int rows_q, int rows_k, int D,
                                                          void *dwq, void *dwk, int w16) {
  __shared__ float s[32][33];
  const int k = blockIdx.y, rows = k ? rows_k : rows_q;
  const float *p = k ? pk : pq;
  void *dw = k ? dwk : dwq;
  if (dw == nullptr) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, f = blockIdx.x * 32 + tx;
  float v = 0.f;
  if (f < D)
    for (int r = ty; r < rows; r += 32) v += p[(long long)r * D + f];
  s[ty][tx] = v;
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) {
    if (ty < o) s[ty][tx] += s[ty + o][tx];
    __syncthreads();
  }
  if (ty == 0 && f < D) {
    if (w16) static_cast<T *>(dw)[f] = Cvt<T>::from_f(s[0][tx]);
    else static_cast<float *>(dw)[f] = s[0][tx];
  }
}

int sm_count() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
  return sms[dev];
}

template <typename T, bool BWD, bool INTER, int VEC, int LPR, int NP>
int launch_cfg(QkArgs &a, int inter, cudaStream_t st) {
  constexpr int RPW = 32 / LPR;
  const int sms = sm_count();
  if (sms <= 0) return LA_ERR_CUDA;
  constexpr int resident = BWD ? 4 : 6;  // CTAs per SM
  const long long warps = (long long)sms * resident * kWarps;
  for (int k = 0; k < 2; ++k) {
    const int H = a.heads[k];
    // tokens side by side: rows of one token fill as much of the warp as there are heads
    int rpt = 1, log2 = 0;
    while (rpt < RPW && rpt < H) rpt <<= 1;
    while ((RPW >> log2) > rpt) ++log2;
    a.tpw[k] = 1 << log2;
    a.tpw_log2[k] = log2;
    const long long groups = (a.T + a.tpw[k] - 1) / a.tpw[k];
    // all heads of a token in one warp where tokens alone fill the GPU: the angles are found once
    int chunk = H;
    while (chunk > rpt && groups * ((H + chunk - 1) / chunk) < warps) chunk = (chunk + 1) / 2;
    chunk = (chunk + rpt - 1) / rpt * rpt;
    a.chunk[k] = chunk;
    a.chunks[k] = (H + chunk - 1) / chunk;
    a.items[k] = groups * a.chunks[k];
  }
  // CTAs in proportion to the rows, one at least, none without work
  const long long total = a.items[0] + a.items[1];
  const long long cap = (long long)sms * resident;
  for (int k = 0; k < 2; ++k) {
    const long long want = (a.items[k] + kWarps - 1) / kWarps;
    long long n = want;
    if ((total + kWarps - 1) / kWarps > cap) {
      n = cap * a.heads[k] / (a.heads[0] + a.heads[1]);
      if (n < 1) n = 1;
      if (n > want) n = want;
    }
    a.ctas[k] = (int)(n < kMaxCtas / 2 ? n : kMaxCtas / 2);
  }
  qk_norm_kernel<T, BWD, INTER, VEC, LPR, NP><<<a.ctas[0] + a.ctas[1], kThreads, 0, st>>>(a, inter);
  return launch_status();
}

template <typename T, bool BWD, bool INTER, int VEC>
int launch_vec(QkArgs &a, int inter, cudaStream_t st) {
  const int lanes = ((a.D + 1) / 2 + VEC - 1) / VEC;
  if constexpr (VEC == 1) {
    if (lanes <= 32) return launch_cfg<T, BWD, false, 1, 32, 1>(a, inter, st);
    if (lanes <= 64) return launch_cfg<T, BWD, false, 1, 32, 2>(a, inter, st);
    if (lanes <= 128) return launch_cfg<T, BWD, false, 1, 32, 4>(a, inter, st);
    return launch_cfg<T, BWD, false, 1, 32, 8>(a, inter, st);
  } else {
    if constexpr (VEC == 8) {
      if (lanes <= 2) return launch_cfg<T, BWD, INTER, VEC, 2, 1>(a, inter, st);
    }
    if (lanes <= 4) return launch_cfg<T, BWD, INTER, VEC, 4, 1>(a, inter, st);
    if (lanes <= 8) return launch_cfg<T, BWD, INTER, VEC, 8, 1>(a, inter, st);
    if (lanes <= 16) return launch_cfg<T, BWD, INTER, VEC, 16, 1>(a, inter, st);
    if (lanes <= 32) return launch_cfg<T, BWD, INTER, VEC, 32, 1>(a, inter, st);
    if constexpr (VEC == 4) return launch_cfg<T, BWD, INTER, VEC, 32, 2>(a, inter, st);
    return LA_ERR_UNSUPPORTED;
  }
}

// The widest access that sizes, strides and addresses allow: VEC features must lie in one half of a pair
// (VEC | R/2 and (D - R)/2; interleaved: VEC | D/2) and start on a multiple of the access.
template <typename T, bool BWD>
int launch_t(QkArgs &a, int inter, cudaStream_t st) {
  auto fits = [&](int vec) {
    if (a.D % 2) return false;
    if (inter ? (a.D / 2) % vec != 0 : ((a.R / 2) % vec != 0 || ((a.D - a.R) / 2) % vec != 0)) return false;
    uintptr_t bytes = 0;
    long long strides = a.D;
    for (int k = 0; k < 2; ++k) {
      bytes |= reinterpret_cast<uintptr_t>(a.x[k]) | reinterpret_cast<uintptr_t>(a.out[k]) |
               reinterpret_cast<uintptr_t>(a.d_out[k]);
      strides |= a.sb[k] | a.sn[k] | a.sh[k];
    }
    return strides % vec == 0 && bytes % (vec * sizeof(T)) == 0;
  };
  if constexpr (sizeof(T) == 2) {
    if (fits(8)) return inter ? launch_vec<T, BWD, true, 8>(a, inter, st) : launch_vec<T, BWD, false, 8>(a, inter, st);
  }
  if (fits(4)) return inter ? launch_vec<T, BWD, true, 4>(a, inter, st) : launch_vec<T, BWD, false, 4>(a, inter, st);
  return launch_vec<T, BWD, false, 1>(a, inter, st);
}

int check(const void *q, const void *k, const int64_t *cu, int64_t M, const int64_t *positions, const double *inv_freq,
          int64_t B, int64_t N, int64_t H, int64_t HK, int64_t D, int64_t R, int dtype, int weight_dtype) {
  cudaGetLastError();
  if (q == nullptr || k == nullptr || (R > 0 && inv_freq == nullptr)) return LA_ERR_NULL_POINTER;
  if (B <= 0 || N <= 0 || H <= 0 || HK <= 0 || D <= 0 || R < 0 || R > D || R % 2) return LA_ERR_BAD_SHAPE;
  if (cu != nullptr ? (B != 1 || M < 1 || positions != nullptr) : M != 0) return LA_ERR_BAD_SHAPE;
  if (!(dtype == LA_F32 || dtype == LA_BF16 || dtype == LA_F16)) return LA_ERR_UNSUPPORTED;
  if (weight_dtype != LA_F32 && weight_dtype != dtype) return LA_ERR_UNSUPPORTED;
  if (D > kMaxD) return LA_ERR_UNSUPPORTED;
  if (N > INT32_MAX || M > INT32_MAX - 1 || H > (1 << 20) || HK > (1 << 20) || B > INT64_MAX / N / 2) return LA_ERR_TOO_LARGE;
  return LA_OK;
}

void fill(QkArgs &a, const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const void *k, int64_t k_sb, int64_t k_sn,
          int64_t k_sh, const void *wq, const void *wk, int weight_dtype, const int64_t *positions, int64_t pos_sb,
          int64_t pos_sn, int64_t offset, const int64_t *cu, int64_t M, const double *inv_freq, int64_t B, int64_t N,
          int64_t H, int64_t HK, int64_t D, int64_t R, float c, float eps) {
  a.x[0] = q; a.x[1] = k;
  a.sb[0] = q_sb; a.sn[0] = q_sn; a.sh[0] = q_sh;
  a.sb[1] = k_sb; a.sn[1] = k_sn; a.sh[1] = k_sh;
  a.w[0] = wq; a.w[1] = wk; a.w16 = weight_dtype != LA_F32;
  a.heads[0] = (int)H; a.heads[1] = (int)HK;
  a.pos = positions; a.pos_sb = pos_sb; a.pos_sn = pos_sn; a.offset = offset;
  a.cu = cu; a.M = (int)M; a.T = B * N; a.N = (int)N; a.D = (int)D; a.R = (int)R; a.c = c; a.eps = eps;
  for (int64_t i = 0; i < R / 2; ++i) a.freq[i] = inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
}

template <bool BWD>
int dispatch(QkArgs &a, int dtype, int inter, cudaStream_t st) {
  switch (dtype) {
    case LA_F32: return launch_t<float, BWD>(a, inter, st);
    case LA_BF16: return launch_t<__nv_bfloat16, BWD>(a, inter, st);
    case LA_F16: return launch_t<__half, BWD>(a, inter, st);
  }
  return LA_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace la

using namespace la;

extern "C" {

int la_qk_norm_rope_fwd(const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const void *k, int64_t k_sb,
                        int64_t k_sn, int64_t k_sh, const void *q_weight, const void *k_weight, int weight_dtype,
                        const int64_t *positions, int64_t pos_sb, int64_t pos_sn, int64_t offset,
                        const int64_t *cu_seqlens, int64_t M, const double *inv_freq, void *q_out, void *k_out,
                        int64_t B, int64_t N, int64_t H, int64_t HK, int64_t D, int64_t R, int dtype, int interleaved,
                        float c, float eps, void *stream) {
  const int rc = check(q, k, cu_seqlens, M, positions, inv_freq, B, N, H, HK, D, R, dtype, weight_dtype);
  if (rc != LA_OK) return rc;
  if (q_out == nullptr || k_out == nullptr) return LA_ERR_NULL_POINTER;
  QkArgs a = {};
  fill(a, q, q_sb, q_sn, q_sh, k, k_sb, k_sn, k_sh, q_weight, k_weight, weight_dtype, positions, pos_sb, pos_sn, offset,
       cu_seqlens, M, inv_freq, B, N, H, HK, D, R, c, eps);
  a.out[0] = q_out; a.out[1] = k_out;
  return dispatch<false>(a, dtype, interleaved != 0, static_cast<cudaStream_t>(stream));
}

int64_t la_qk_norm_rope_bwd_workspace_bytes(int64_t D) { return D <= 0 ? 0 : (int64_t)kMaxCtas * D * 4; }

int la_qk_norm_rope_bwd(const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const void *k, int64_t k_sb,
                        int64_t k_sn, int64_t k_sh, const void *q_weight, const void *k_weight, int weight_dtype,
                        const int64_t *positions, int64_t pos_sb, int64_t pos_sn, int64_t offset,
                        const int64_t *cu_seqlens, int64_t M, const double *inv_freq, const void *d_q_out,
                        const void *d_k_out, void *dq, void *dk, void *dq_weight, void *dk_weight, void *workspace,
                        int64_t workspace_bytes, int64_t B, int64_t N, int64_t H, int64_t HK, int64_t D, int64_t R,
                        int dtype, int interleaved, float c, float eps, void *stream) {
  const int rc = check(q, k, cu_seqlens, M, positions, inv_freq, B, N, H, HK, D, R, dtype, weight_dtype);
  if (rc != LA_OK) return rc;
  if (d_q_out == nullptr || d_k_out == nullptr || dq == nullptr || dk == nullptr) return LA_ERR_NULL_POINTER;
  const bool want_dw = dq_weight != nullptr || dk_weight != nullptr;
  if (want_dw) {
    if (workspace == nullptr || workspace_bytes < la_qk_norm_rope_bwd_workspace_bytes(D)) return LA_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 3u) return LA_ERR_MISALIGNED;
  }
  QkArgs a = {};
  fill(a, q, q_sb, q_sn, q_sh, k, k_sb, k_sn, k_sh, q_weight, k_weight, weight_dtype, positions, pos_sb, pos_sn, offset,
       cu_seqlens, M, inv_freq, B, N, H, HK, D, R, c, eps);
  a.d_out[0] = d_q_out; a.d_out[1] = d_k_out;
  a.out[0] = dq; a.out[1] = dk;
  if (dq_weight != nullptr) a.partial[0] = static_cast<float *>(workspace);
  if (dk_weight != nullptr) a.partial[1] = static_cast<float *>(workspace) + (int64_t)kMaxCtas / 2 * D;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc2 = dispatch<true>(a, dtype, interleaved != 0, st);
  if (rc2 != LA_OK || !want_dw) return rc2;
  const dim3 grid((unsigned)((D + 31) / 32), 2);
  if (dtype == LA_F16)
    qk_norm_dw_kernel<__half><<<grid, 1024, 0, st>>>(a.partial[0], a.partial[1], a.ctas[0], a.ctas[1], (int)D, dq_weight,
                                                     dk_weight, a.w16);
  else
    qk_norm_dw_kernel<__nv_bfloat16><<<grid, 1024, 0, st>>>(a.partial[0], a.partial[1], a.ctas[0], a.ctas[1], (int)D,
                                                            dq_weight, dk_weight, a.w16 && dtype != LA_F32);
  return launch_status();
}

}  // extern "C"
