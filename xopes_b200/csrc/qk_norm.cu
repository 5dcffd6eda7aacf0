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
//
// Two kernels.  qk_norm_stream_kernel, for large calls whose heads lie next to each other: every warp keeps a ring of
// slots in shared memory full by bulk copies of several heads of a token, so that the bytes in flight do not depend on
// registers.  qk_norm_kernel, for small calls, other strides and few heads: loads straight into registers, one step ahead.
// 8 x 8192 tokens of 32 + 32 heads of 128 (bf16), forward / backward: 375-390 / 535 us by the first (2.15 / 3.22 GB, 328 /
// 492 us at the measured copy bandwidth), 531 / 932 by the second.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace la {
namespace {

constexpr int kMaxD = 512;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMaxCtas = 2048;  // partial rows of the weight gradients
constexpr long long kStreamFrom = 1 << 20;  // elements of a tensor (launch_both)

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

// The features of a lane and its share of the weights and their gradients.
// INTER: interleaved pairs.  VEC > 1: pack p of lane l (p LPR + l = j) is the low features [j VEC, +VEC) of the
// first half of the rotated (or of the passing) features and the matching high ones; with INTER the "low" and
// "high" packs are simply the first and second half of the row, and pairs are neighbours inside a pack.
// VEC == 1: any D, R and alignment, INTER read from `inter`.
template <typename T, bool INTER, int VEC, int LPR, int NP> struct Lane {
  static constexpr int N = VEC * NP;
  int f_lo[NP], f_hi[NP];
  bool on_lo[NP], on_hi[NP];
  float w_lo[N], w_hi[N];  // c w

  __device__ __forceinline__ void init(const QkArgs &a, int which, int inter, int gl) {
    const int D = a.D, half = a.R >> 1, pairs = (D + 1) >> 1;
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
    }
  }
  // the lane's angles out of a token's (SIGN: of the rotation)
  __device__ __forceinline__ void angles(const float *c, const float *s, int half, int gl, float sign, float (&cs)[N],
                                         float (&sn)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i / VEC, j = i % VEC;
      int pr = (p * LPR + gl) * VEC + j;  // the lane's i-th pair
      if (INTER && VEC > 1)               // first half of the values: pairs of the low pack, then of the high pack
        pr = ((j < VEC / 2 ? f_lo[p] : f_hi[p]) >> 1) + j % (VEC / 2 > 0 ? VEC / 2 : 1);
      const bool rot = pr < half;
      cs[i] = rot ? c[pr] : 1.f;
      sn[i] = rot ? sign * s[pr] : 0.f;
    }
  }
  static __device__ __forceinline__ void rotate(float *lo, float *hi, const float (&cs)[N], const float (&sn)[N]) {
    if (INTER && VEC > 1) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const int e = p * VEC + 2 * j, cl = p * VEC + j, ch = cl + VEC / 2;
          const float a0 = lo[e], a1 = lo[e + 1], b0 = hi[e], b1 = hi[e + 1];
          lo[e] = a0 * cs[cl] - a1 * sn[cl];
          lo[e + 1] = a1 * cs[cl] + a0 * sn[cl];
          hi[e] = b0 * cs[ch] - b1 * sn[ch];
          hi[e + 1] = b1 * cs[ch] + b0 * sn[ch];
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = lo[i], v = hi[i];
        lo[i] = u * cs[i] - v * sn[i];
        hi[i] = v * cs[i] + u * sn[i];
      }
    }
  }
  // (xl, xh): a row in, its output out
  __device__ __forceinline__ void forward(float (&xl)[N], float (&xh)[N], const float (&cs)[N], const float (&sn)[N],
                                          float eps) const {
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s2 += xl[i] * xl[i] + xh[i] * xh[i];
    const float rs = rsqrtf(lane_sum<LPR>(s2) + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      xl[i] = xl[i] * rs * w_lo[i];
      xh[i] = xh[i] * rs * w_hi[i];
    }
    rotate(xl, xh, cs, sn);
  }
  // (xl, xh): a row in, its gradient out; (dl, dh): the output's gradient; sn negative: the rotation back
  __device__ __forceinline__ void backward(float (&xl)[N], float (&xh)[N], float (&dl)[N], float (&dh)[N],
                                           const float (&cs)[N], const float (&sn)[N], float eps, float (&dw_lo)[N],
                                           float (&dw_hi)[N]) const {
    rotate(dl, dh, cs, sn);
    float s2 = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s2 += xl[i] * xl[i] + xh[i] * xh[i];
      dot += dl[i] * w_lo[i] * xl[i] + dh[i] * w_hi[i] * xh[i];
    }
    const float rs = rsqrtf(lane_sum<LPR>(s2) + eps);
    dot = lane_sum<LPR>(dot) * rs;  // sum of g xh
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float nl = xl[i] * rs, nh = xh[i] * rs;
      dw_lo[i] += nl * dl[i];
      dw_hi[i] += nh * dh[i];
      xl[i] = (dl[i] * w_lo[i] - nl * dot) * rs;
      xh[i] = (dh[i] * w_hi[i] - nh * dot) * rs;
    }
  }
  // the CTA's partial weight gradient: sums over the warps' rows
  __device__ __forceinline__ void leave(float (&dw_lo)[N], float (&dw_hi)[N], float (*part)[2 * LPR * N], float *out,
                                        const QkArgs &a, int warp, int sub) const {
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
    for (int f = threadIdx.x; f < a.D; f += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) s += part[k][f];
      out[f] = s * a.c;
    }
  }
};

// angle of a position as cosine and sine
__device__ __forceinline__ void angle_of(long long position, double freq, float &c, float &s) {
  double turns = (double)position * freq;
  turns -= rint(turns);
  sincospif(2.f * (float)turns, &s, &c);
}

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
  lets_next_start();
  for (int i = threadIdx.x; i < half; i += kThreads) s_freq[i] = a.freq[i];
  __syncthreads();
  after_previous();
  Lane<T, INTER, VEC, LPR, NP> ln;
  ln.init(a, which, inter, gl);
  float dw_lo[N] = {}, dw_hi[N] = {};
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
        r_lo[p] = ln.on_lo[p] ? *reinterpret_cast<const R *>(x + ln.f_lo[p]) : zero;
        r_hi[p] = ln.on_hi[p] ? *reinterpret_cast<const R *>(x + ln.f_hi[p]) : zero;
        if (BWD) {
          const T *d = dp + (crow + hc) * D;
          d_lo[p] = ln.on_lo[p] && in ? *reinterpret_cast<const R *>(d + ln.f_lo[p]) : zero;
          d_hi[p] = ln.on_hi[p] && in ? *reinterpret_cast<const R *>(d + ln.f_hi[p]) : zero;
        }
      }
    };
    fetch(h0 + hsub);
    // the angles of the warp's tokens, each found by one lane
    for (int i = lane; i < tpw * half; i += 32) {
      const int ts = i / half, pr = i - ts * half;
      const long long tt = group * tpw + ts;
      angle_of(position_of(a, tt < a.T ? tt : a.T - 1), s_freq[pr], s_cos[warp][i], s_sin[warp][i]);
    }
    __syncwarp();
    float cs[N], sn[N];
    ln.angles(s_cos[warp] + tsub * half, s_sin[warp] + tsub * half, half, gl, BWD ? -1.f : 1.f, cs, sn);
    __syncwarp();  // the next item's angles overwrite these

    for (int hb = h0; hb < h1; hb += rpt) {
      const int h = hb + hsub;
      const bool live = t_on && h < h1;
      float xl[N], xh[N], dl[N], dh[N];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        P::unpack(r_lo[p], xl + p * VEC);
        P::unpack(r_hi[p], xh + p * VEC);
        if (BWD) {
          P::unpack(d_lo[p], dl + p * VEC);
          P::unpack(d_hi[p], dh + p * VEC);
        }
      }
      if (hb + rpt < h1) fetch(h + rpt);
      if (BWD) ln.backward(xl, xh, dl, dh, cs, sn, a.eps, dw_lo, dw_hi);
      else ln.forward(xl, xh, cs, sn, a.eps);
      if (live) {
        T *o = op + (crow + h) * D;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          if (ln.on_lo[p]) *reinterpret_cast<R *>(o + ln.f_lo[p]) = P::pack(xl + p * VEC);
          if (ln.on_hi[p]) *reinterpret_cast<R *>(o + ln.f_hi[p]) = P::pack(xh + p * VEC);
        }
      }
    }
  }
  if (BWD && a.partial[which] != nullptr) {  // uniform over the CTA
    __shared__ float part[kWarps][2 * LPR * N];
    ln.leave(dw_lo, dw_hi, part, a.partial[which] + (long long)cta * D, a, warp, sub);
  }
}

// ------------------------------------------------------------------------------ large calls
constexpr int kDepth = 2;                                                      // slots of a warp's ring
template <bool BWD> constexpr int slot_bytes() { return BWD ? 2048 : 4096; }  // of each tensor that is read
template <bool BWD> constexpr int stream_smem() { return kWarps * kDepth * slot_bytes<BWD>() * (BWD ? 2 : 1); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The rotation of a lane's N low and N high features as packed pairs of fp32, two neighbouring features each, out of the
// token's cosines and sines in shared memory (16-byte pieces; pairs past the rotated ones are 1 and 0 there).
//   lo' = lo a + {hi, or with INTER its own neighbour} b      hi' likewise with c and d
// Forward with the weights multiplied in; back (BWD) without them, and a = c, b = -d where pairs are not neighbours.
template <int N, bool INTER, bool BWD> struct Turn {
  static constexpr int P = N / 2, Q = BWD && !INTER ? 0 : P;
  float2 a[P], b[P], c[Q ? Q : 1], d[P];
  __device__ __forceinline__ void set(const float *cs, const float *sn, int gl, int half_row, const float (&w_lo)[N],
                                      const float (&w_hi)[N]) {
    float co[N], si[N];
    if (INTER) {  // N / 2 pairs of the low pack, N / 2 of the high one
      read<P>(cs + gl * P, co);
      read<P>(sn + gl * P, si);
      read<P>(cs + half_row + gl * P, co + P);
      read<P>(sn + half_row + gl * P, si + P);
    } else {
      read<N>(cs + gl * N, co);
      read<N>(sn + gl * N, si);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float l0 = BWD ? 1.f : w_lo[2 * i], l1 = BWD ? 1.f : w_lo[2 * i + 1];
      const float h0 = BWD ? 1.f : w_hi[2 * i], h1 = BWD ? 1.f : w_hi[2 * i + 1];
      if (INTER) {
        const float cl = co[i], ch = co[i + P], sl = BWD ? -si[i] : si[i], sh = BWD ? -si[i + P] : si[i + P];
        a[i] = make_float2(l0 * cl, l1 * cl);
        b[i] = make_float2(-l1 * sl, l0 * sl);
        c[Q ? i : 0] = make_float2(h0 * ch, h1 * ch);
        d[i] = make_float2(-h1 * sh, h0 * sh);
      } else {
        const float s0 = BWD ? -si[2 * i] : si[2 * i], s1 = BWD ? -si[2 * i + 1] : si[2 * i + 1];
        a[i] = make_float2(l0 * co[2 * i], l1 * co[2 * i + 1]);
        b[i] = make_float2(-h0 * s0, -h1 * s1);
        if (Q) c[Q ? i : 0] = make_float2(h0 * co[2 * i], h1 * co[2 * i + 1]);
        d[i] = make_float2(l0 * s0, l1 * s1);
      }
    }
  }
  __device__ __forceinline__ void apply(float2 (&lo)[P], float2 (&hi)[P]) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 u = lo[i], v = hi[i];
      if (INTER) {
        lo[i] = fma2(u, a[i], mul2(make_float2(u.y, u.x), b[i]));
        hi[i] = fma2(v, c[Q ? i : 0], mul2(make_float2(v.y, v.x), d[i]));
      } else {
        lo[i] = fma2(u, a[i], mul2(v, b[i]));
        hi[i] = fma2(v, Q ? c[Q ? i : 0] : a[i], mul2(u, d[i]));
      }
    }
  }
  template <int W> static __device__ __forceinline__ void read(const float *p, float *v) {
    if constexpr (W == 2) {
      const float2 x = *reinterpret_cast<const float2 *>(p);
      v[0] = x.x; v[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const float4 x = *reinterpret_cast<const float4 *>(p + i);
        v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
      }
    }
  }
};

// A CTA owns a range of tokens, its warps take them in turn; a warp walks a token's heads in chunks of a.chunk rows = one
// slot, one slot ahead.  Heads lie next to each other (D elements apart) and rows are a multiple of 16 bytes on
// 16-byte boundaries.  The arithmetic is in packed pairs: with one fp32 operation an instruction the kernel issued 274 / 488
// instructions for four rows of 128 features (forward / backward), 415 / 710 us for the call above; with 16 features a
// lane it kept 16 warps an SM, which waited for shuffles and shared memory (376 / 691 us).
template <typename T, bool BWD, bool INTER, int VEC, int LPR>
__global__ void __launch_bounds__(kThreads, VEC == 8 ? 4 : (BWD ? 5 : 6)) qk_norm_stream_kernel(const __grid_constant__ QkArgs a, int *status) {
  typedef Pack<T, VEC> P;
  typedef typename P::R R;
  constexpr int N = VEC, RPW = 32 / LPR, kSlot = slot_bytes<BWD>();
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(16) float s_cos[kWarps][LPR * N], s_sin[kWarps][LPR * N];
  __shared__ double s_freq[kMaxD / 2];
  __shared__ __align__(8) uint64_t bars[kWarps][kDepth];
  __shared__ volatile int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % LPR, sub = lane / LPR;
  const int which = blockIdx.x >= (unsigned)a.ctas[0];
  const int cta = which ? blockIdx.x - a.ctas[0] : blockIdx.x;
  const int H = a.heads[which], D = a.D, half = a.R >> 1;
  for (int i = threadIdx.x; i < half; i += kThreads) s_freq[i] = a.freq[i];
  for (int i = half + lane; i < LPR * N; i += 32) {  // pairs that pass
    s_cos[warp][i] = 1.f;
    s_sin[warp][i] = 0.f;
  }
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < kDepth) ptx::mbar_init(ptx::smem_u32(&bars[warp][lane]), 1);
  ptx::fence_barrier_init();
  lets_next_start();
  __syncthreads();
  after_previous();
  Lane<T, INTER, VEC, LPR, 1> ln;
  ln.init(a, which, 0, gl);
  float2 dw_lo[N / 2] = {}, dw_hi[N / 2] = {};
  uint8_t *slots = ring + warp * kDepth * kSlot * (BWD ? 2 : 1);
  const int chunk = a.chunk[which], chunks = a.chunks[which];
  const int f_lo = ln.f_lo[0], f_hi = ln.f_hi[0];
  const bool on = ln.on_lo[0];  // D is even: low and high features exist together
  const long long t0 = a.T * cta / a.ctas[which] + warp, t1 = a.T * (cta + 1) / a.ctas[which];
  const R zero = {};

  // the next slot to fill: chunk fc of token ft = (fb, fn)
  long long ft = t0, fb = t0 / a.N;
  int fn = (int)(t0 - fb * a.N), fc = 0, fs = 0;
  auto fill = [&]() {
    if (ft >= t1) return;
    if (lane == 0) {
      const int h0 = fc * chunk;
      const uint32_t bytes = (uint32_t)(min(chunk, H - h0) * D * (int)sizeof(T));
      const uint32_t bar = ptx::smem_u32(&bars[warp][fs]), dst = ptx::smem_u32(slots + fs * kSlot * (BWD ? 2 : 1));
      ptx::mbar_arrive_expect_tx(bar, BWD ? 2 * bytes : bytes);
      bulk_load(dst, static_cast<const T *>(a.x[which]) + fb * a.sb[which] + fn * a.sn[which] + h0 * D, bytes, bar);
      if (BWD) bulk_load(dst + kSlot, static_cast<const T *>(a.d_out[which]) + (ft * H + h0) * D, bytes, bar);
    }
    if (++fs == kDepth) fs = 0;
    if (++fc == chunks) {
      fc = 0;
      ft += kWarps;
      fn += kWarps;
      while (fn >= a.N) {
        fn -= a.N;
        ++fb;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) fill();

  int slot = 0, parity = 0;
  bool ok = true;
  long long b = t0 / a.N, doc0 = 0, doc1 = -1;  // sequence; the document a token was last found in
  int n = (int)(t0 - b * a.N);
  for (long long t = t0; t < t1 && ok; t += kWarps) {
    long long position = n;
    if (a.cu != nullptr) {
      if (t >= doc1) {
        int lo = 0, hi = a.M;  // largest i with cu[i] <= t
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (__ldg(a.cu + mid) <= t) lo = mid; else hi = mid - 1;
        }
        doc0 = __ldg(a.cu + lo);
        doc1 = lo < a.M ? __ldg(a.cu + lo + 1) : a.T;
      }
      position = t - doc0;
    } else if (a.pos != nullptr) {
      position = __ldg(a.pos + b * a.pos_sb + n * a.pos_sn);
    }
    position += a.offset;
    n += kWarps;
    while (n >= a.N) {
      n -= a.N;
      ++b;
    }
    for (int i = lane; i < half; i += 32) angle_of(position, s_freq[i], s_cos[warp][i], s_sin[warp][i]);
    __syncwarp();
    Turn<N, INTER, BWD> turn;
    turn.set(s_cos[warp], s_sin[warp], gl, D >> 2, ln.w_lo, ln.w_hi);
    T *orow = static_cast<T *>(a.out[which]) + t * H * D;
    for (int c = 0; c < chunks; ++c) {
      fill();  // into the slot whose last reader has passed the barrier below
      const int rows = min(chunk, H - c * chunk);
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bars[warp][slot]), parity, &abort_flag, status, 311));
      if (!ok) break;
      const T *xs = reinterpret_cast<const T *>(slots + slot * kSlot * (BWD ? 2 : 1));
      const T *ds = reinterpret_cast<const T *>(slots + slot * kSlot * 2 + kSlot);
      for (int r = sub; r - sub < rows; r += RPW) {
        const bool live = r < rows;
        const int at = (live ? r : rows - 1) * D;  // past the chunk: a row that exists, with a gradient of 0
        float2 xl[N / 2], xh[N / 2];
        P::unpack(on ? *reinterpret_cast<const R *>(xs + at + f_lo) : zero, reinterpret_cast<float *>(xl));
        P::unpack(on ? *reinterpret_cast<const R *>(xs + at + f_hi) : zero, reinterpret_cast<float *>(xh));
        float2 s2 = mul2(xl[0], xl[0]);
        s2 = fma2(xh[0], xh[0], s2);
#pragma unroll
        for (int i = 1; i < N / 2; ++i) s2 = fma2(xh[i], xh[i], fma2(xl[i], xl[i], s2));
        if (!BWD) {
          const float2 rs = both(rsqrtf(lane_sum<LPR>(s2.x + s2.y) + a.eps));
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            xl[i] = mul2(xl[i], rs);
            xh[i] = mul2(xh[i], rs);
          }
          turn.apply(xl, xh);
        } else {
          float2 dl[N / 2], dh[N / 2];
          P::unpack(on && live ? *reinterpret_cast<const R *>(ds + at + f_lo) : zero, reinterpret_cast<float *>(dl));
          P::unpack(on && live ? *reinterpret_cast<const R *>(ds + at + f_hi) : zero, reinterpret_cast<float *>(dh));
          turn.apply(dl, dh);
          const float2 *wl = reinterpret_cast<const float2 *>(ln.w_lo), *wh = reinterpret_cast<const float2 *>(ln.w_hi);
          float2 dot = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < N / 2; ++i) dot = fma2(mul2(dh[i], wh[i]), xh[i], fma2(mul2(dl[i], wl[i]), xl[i], dot));
          const float rs1 = rsqrtf(lane_sum<LPR>(s2.x + s2.y) + a.eps);
          const float2 rs = both(rs1), nd = both(-lane_sum<LPR>(dot.x + dot.y) * rs1);  // - sum of g xh
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            xl[i] = mul2(xl[i], rs);
            xh[i] = mul2(xh[i], rs);
            dw_lo[i] = fma2(xl[i], dl[i], dw_lo[i]);
            dw_hi[i] = fma2(xh[i], dh[i], dw_hi[i]);
            xl[i] = mul2(fma2(dl[i], wl[i], mul2(xl[i], nd)), rs);  // the product again: 16 registers less
            xh[i] = mul2(fma2(dh[i], wh[i], mul2(xh[i], nd)), rs);
          }
        }
        if (live && on) {
          *reinterpret_cast<R *>(orow + at + f_lo) = P::pack(reinterpret_cast<const float *>(xl));
          *reinterpret_cast<R *>(orow + at + f_hi) = P::pack(reinterpret_cast<const float *>(xh));
        }
      }
      orow += chunk * D;
      if (++slot == kDepth) {
        slot = 0;
        parity ^= 1;
      }
      __syncwarp();
    }
  }
  if (!ok) {  // a wait gave up: let the copies in flight land
    const uint64_t since = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - since < 1000000ull) __nanosleep(1000);
  }
  if (BWD && a.partial[which] != nullptr) {  // uniform over the CTA
    __shared__ float part[kWarps][2 * LPR * N];
    ln.leave(reinterpret_cast<float (&)[N]>(dw_lo), reinterpret_cast<float (&)[N]>(dw_hi), part,
             a.partial[which] + (long long)cta * D, a, warp, sub);
  }
}

// dw[f] = sum over the CTAs' partial rows, in a fixed order.  Block (32 features, 32 row slots); grid.y = q, k.
template <typename T>
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float *pq, const float *pk, int rows_q, int rows_k, int D,
                                                          void *dwq, void *dwk, int w16) {
  __shared__ float s[32][33];
  lets_next_start();
  after_previous();
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

// CTAs in proportion to the rows of the tensors that have items, one at least, none without work
void share_ctas(QkArgs &a, long long cap) {
  const long long total = a.items[0] + a.items[1];
  const long long rows = (a.items[0] ? a.heads[0] : 0) + (a.items[1] ? a.heads[1] : 0);
  for (int k = 0; k < 2; ++k) {
    const long long want = (a.items[k] + kWarps - 1) / kWarps;
    long long n = want;
    if (want > 0 && (total + kWarps - 1) / kWarps > cap) {
      n = cap * a.heads[k] / rows;
      if (n < 1) n = 1;
      if (n > want) n = want;
    }
    a.ctas[k] = (int)(n < kMaxCtas / 2 ? n : kMaxCtas / 2);
  }
}

template <typename T, bool BWD, bool INTER, int VEC, int LPR, int NP>
int launch_cfg(QkArgs &a, int inter, const bool (&mine)[2], cudaStream_t st) {
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
    a.items[k] = mine[k] ? groups * a.chunks[k] : 0;
  }
  share_ctas(a, (long long)sms * resident);
  return launch_early(qk_norm_kernel<T, BWD, INTER, VEC, LPR, NP>, dim3(a.ctas[0] + a.ctas[1]), kThreads, 0, st, 0, a, inter);
}

template <typename T, bool BWD, bool INTER, int VEC, int LPR>
int launch_stream(QkArgs &a, const bool (&mine)[2], cudaStream_t st) {
  constexpr int RPW = 32 / LPR, kSmem = stream_smem<BWD>();
  static bool set[64] = {false};
  static int resident[64] = {0};
  int dev = 0;
  const int sms = sm_count();
  if (sms <= 0 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LA_ERR_CUDA;
  if (!set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(qk_norm_stream_kernel<T, BWD, INTER, VEC, LPR>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident[dev], qk_norm_stream_kernel<T, BWD, INTER, VEC, LPR>,
                                                        kThreads, kSmem);
    if (e != cudaSuccess || resident[dev] < 1) {
      note_cuda_error(e, "qk_norm shared memory");
      return LA_ERR_CUDA;
    }
    set[dev] = true;
  }
  for (int k = 0; k < 2; ++k) {
    int chunk = slot_bytes<BWD>() / (a.D * (int)sizeof(T)) / RPW * RPW;
    if (chunk > a.heads[k]) chunk = a.heads[k];
    a.chunk[k] = chunk;
    a.chunks[k] = (a.heads[k] + chunk - 1) / chunk;
    a.items[k] = mine[k] ? a.T : 0;
  }
  share_ctas(a, (long long)sms * resident[dev]);
  int *status = nullptr;
  if (!status_word_for(st, &status)) return LA_ERR_CUDA;
  return launch_early(qk_norm_stream_kernel<T, BWD, INTER, VEC, LPR>, dim3(a.ctas[0] + a.ctas[1]), kThreads, kSmem, st, 0, a,
                      status);
}

// Streamed: tensors whose heads lie next to each other and fill a warp's rows, from 2^20 elements on.  Measured, forward /
// backward in us, streamed against direct: 16 heads of 128 (bf16), 2^18 elements 5.0 / 9.1 against 4.8 / 8.8, 2^20
// 5.6 / 10.7 against 8.8 / 16.5, 2^24 28 / 44 against 40 / 75; 32 heads of 128 (fp32), 2^18 8.3 / 14.4 against 4.3 / 8.2,
// 2^20 8.5 / 15.3 against 9.1 / 14.3, 2^23 27 / 44 against 29 / 46.
template <typename T, bool BWD, bool INTER, int VEC, int LPR>
int launch_both(QkArgs &a, cudaStream_t st) {
  // streamed 16-bit rows are taken in 8-byte pieces: half the features, and so half the registers, a lane
  constexpr bool kHalf = VEC == 8 && LPR <= 16;
  constexpr int SVEC = kHalf ? 4 : VEC, SLPR = kHalf ? 2 * LPR : LPR, RPW = 32 / SLPR;
  constexpr int kPer = 16 / (int)sizeof(T);
  bool stream[2], direct[2];
  for (int k = 0; k < 2; ++k) {
    const bool on16 = (reinterpret_cast<uintptr_t>(a.x[k]) | reinterpret_cast<uintptr_t>(a.d_out[k])) % 16 == 0 &&
                      a.D % kPer == 0 && a.sb[k] % kPer == 0 && a.sn[k] % kPer == 0;
    stream[k] = on16 && a.heads[k] >= RPW && (a.heads[k] == 1 || a.sh[k] == a.D) &&
                RPW * a.D * (int)sizeof(T) <= slot_bytes<BWD>() && a.T * a.heads[k] * a.D >= kStreamFrom;
    direct[k] = !stream[k];
  }
  int ctas[2] = {0, 0}, rc = LA_OK;
  if (stream[0] || stream[1]) {
    rc = launch_stream<T, BWD, INTER, SVEC, SLPR>(a, stream, st);
    ctas[0] = a.ctas[0];
    ctas[1] = a.ctas[1];
  }
  if (rc == LA_OK && (direct[0] || direct[1])) {
    rc = launch_cfg<T, BWD, INTER, VEC, LPR, 1>(a, INTER, direct, st);
    ctas[0] += a.ctas[0];
    ctas[1] += a.ctas[1];
  }
  a.ctas[0] = ctas[0];  // partial rows of each tensor
  a.ctas[1] = ctas[1];
  return rc;
}

template <typename T, bool BWD, bool INTER, int VEC>
int launch_vec(QkArgs &a, int inter, cudaStream_t st) {
  const bool both[2] = {true, true};
  const int lanes = ((a.D + 1) / 2 + VEC - 1) / VEC;
  if constexpr (VEC == 1) {
    if (lanes <= 32) return launch_cfg<T, BWD, false, 1, 32, 1>(a, inter, both, st);
    if (lanes <= 64) return launch_cfg<T, BWD, false, 1, 32, 2>(a, inter, both, st);
    if (lanes <= 128) return launch_cfg<T, BWD, false, 1, 32, 4>(a, inter, both, st);
    return launch_cfg<T, BWD, false, 1, 32, 8>(a, inter, both, st);
  } else if constexpr (VEC * sizeof(T) == 16) {
    if constexpr (VEC == 8) {
      if (lanes <= 2) return launch_both<T, BWD, INTER, VEC, 2>(a, st);
    }
    if (lanes <= 4) return launch_both<T, BWD, INTER, VEC, 4>(a, st);
    if (lanes <= 8) return launch_both<T, BWD, INTER, VEC, 8>(a, st);
    if (lanes <= 16) return launch_both<T, BWD, INTER, VEC, 16>(a, st);
    if (lanes <= 32) return launch_both<T, BWD, INTER, VEC, 32>(a, st);
    if constexpr (VEC == 4) return launch_cfg<T, BWD, INTER, VEC, 32, 2>(a, inter, both, st);
    return LA_ERR_UNSUPPORTED;
  } else {  // 8-byte accesses of 16-bit types
    if (lanes <= 8) return launch_cfg<T, BWD, INTER, VEC, 8, 1>(a, inter, both, st);
    if (lanes <= 16) return launch_cfg<T, BWD, INTER, VEC, 16, 1>(a, inter, both, st);
    if (lanes <= 32) return launch_cfg<T, BWD, INTER, VEC, 32, 1>(a, inter, both, st);
    return launch_cfg<T, BWD, INTER, VEC, 32, 2>(a, inter, both, st);
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
  const int w16 = a.w16 && dtype != LA_F32;
  return launch_early(dtype == LA_F16 ? qk_norm_dw_kernel<__half> : qk_norm_dw_kernel<__nv_bfloat16>, grid, 1024, 0, st, 0,
                      a.partial[0], a.partial[1], a.ctas[0], a.ctas[1], (int)D, dq_weight, dk_weight, w16);
}

}  // extern "C"
