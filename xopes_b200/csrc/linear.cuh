// Pieces shared by the kernels of linear_fn and gated_linear_fn: what happens to a product before it is written
// (bias, activation, product of the pair, residual), and the interface between the host plan (linear.cu) and the
// matrix kernels (gemm_sm100.cu).
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace la {
namespace lin {

enum { kActNone = 0, kActRelu = 1, kActSigmoid = 2, kActSilu = 3, kActGelu = 4 };

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float ex2(float x) {  // 2^x, one instruction
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 ex2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
// 1 / x; 0 for x above 2^126
__device__ __forceinline__ float2 inverse2(float2 x) { return make_float2(__fdividef(1.f, x.x), __fdividef(1.f, x.y)); }
constexpr float kLog2e = 1.4426950408889634f;

// Sigmoid and the normal distribution's integral in two forms.  fp32 results: by expf (2 ulp) and erff, one value at a time.
// Results that are rounded to 16 bits: by 2^x and 1 / x of the special function unit, two values in packed arithmetic.

// 1 / (1 + e^-z)
__device__ __forceinline__ float2 sigmoid2(float2 z) { return inverse2(add2(both(1.f), ex2(mul2(z, both(-kLog2e))))); }
__device__ __forceinline__ float sigmoid_exact(float z) { return 1.f / (1.f + expf(-z)); }
// Phi(z), and e = e^(-z^2 / 2).  The tail Phi(-a) = e R(a) with R(a) as a polynomial in t = 1 / (1 + p a), the form of Hastings
// (Approximations for Digital Computers, 1955); p and the six coefficients minimise the largest relative error over 0 .. 14.5
// (a linear program), 4.1e-6, so that the lower tail keeps its bits: Abramowitz and Stegun 7.1.26, which has five coefficients
// and bounds the absolute error, is off by 5e-4 at -3.5 and 4e-3 at -6, where half a step is 4.9e-4 (fp16) and 3.9e-3 (bf16).
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2 &e) {
  e = ex2(mul2(mul2(z, z), both(-0.5f * kLog2e)));
  const float2 t = inverse2(fma2(both(0.308636275f), make_float2(fabsf(z.x), fabsf(z.y)), both(1.f)));
  float2 q = fma2(t, both(-0.0750100687f), both(0.186830327f));
  q = fma2(t, q, both(0.00985927228f));
  q = fma2(t, q, both(0.135590911f));
  q = fma2(t, q, both(0.119369581f));
  q = mul2(mul2(t, e), fma2(t, q, both(0.123357952f)));
  return make_float2(z.x < 0.f ? q.x : 1.f - q.x, z.y < 0.f ? q.y : 1.f - q.y);
}
// by erfcf, which keeps its bits in the lower tail (1 + erff is a multiple of 2^-24 there)
__device__ __forceinline__ float normal_cdf_exact(float z) { return 0.5f * erfcf(z * -0.70710678118654752f); }

// z[j] = act(z[j]); the kind is the same for the whole launch, so the choice is a branch around a row's loop
template <typename T, int W>
__device__ __forceinline__ void activate(float (&z)[W], int kind) {
  if (kind == kActRelu) {
#pragma unroll
    for (int j = 0; j < W; ++j) z[j] = z[j] > 0.f || z[j] != z[j] ? z[j] : 0.f;
    return;
  }
  if constexpr (sizeof(T) == 2 && W % 2 == 0) {
    float2 (&v)[W / 2] = reinterpret_cast<float2 (&)[W / 2]>(z);
    if (kind == kActSigmoid) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) v[j] = sigmoid2(v[j]);
    } else if (kind == kActSilu) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) v[j] = mul2(v[j], sigmoid2(v[j]));
    } else if (kind == kActGelu) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        float2 e;
        v[j] = mul2(v[j], normal_cdf2(v[j], e));
      }
    }
  } else {
    if (kind == kActSigmoid) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] = sigmoid_exact(z[j]);
    } else if (kind == kActSilu) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] *= sigmoid_exact(z[j]);
    } else if (kind == kActGelu) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] *= normal_cdf_exact(z[j]);
    }
  }
}

// z[j] = act(z[j]) and d[j] = act'(z[j])
template <typename T, int W>
__device__ __forceinline__ void activate_grad(float (&z)[W], float (&d)[W], int kind) {
  constexpr float kDensity = 0.3989422804014327f;  // 1 / sqrt(2 pi)
  if (kind == kActRelu) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      d[j] = z[j] <= 0.f ? 0.f : 1.f;  // NaN: the gradient passes, as the value does
      z[j] = z[j] > 0.f || z[j] != z[j] ? z[j] : 0.f;
    }
    return;
  }
  if (kind == kActNone) {
#pragma unroll
    for (int j = 0; j < W; ++j) d[j] = 1.f;
    return;
  }
  if constexpr (sizeof(T) == 2 && W % 2 == 0) {
    float2 (&v)[W / 2] = reinterpret_cast<float2 (&)[W / 2]>(z), (&g)[W / 2] = reinterpret_cast<float2 (&)[W / 2]>(d);
#pragma unroll
    for (int j = 0; j < W / 2; ++j) {
      if (kind == kActGelu) {
        float2 e;
        const float2 cdf = normal_cdf2(v[j], e);
        g[j] = fma2(mul2(v[j], both(kDensity)), e, cdf);
        v[j] = mul2(v[j], cdf);
      } else {
        const float2 s = sigmoid2(v[j]), rest = fma2(s, both(-1.f), both(1.f));
        if (kind == kActSilu) {
          v[j] = mul2(v[j], s);
          g[j] = fma2(v[j], rest, s);
        } else {
          v[j] = s;
          g[j] = mul2(s, rest);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (kind == kActGelu) {
        const float cdf = normal_cdf_exact(z[j]);
        d[j] = cdf + z[j] * kDensity * expf(-0.5f * z[j] * z[j]);
        z[j] *= cdf;
      } else {
        const float s = sigmoid_exact(z[j]);
        if (kind == kActSilu) {
          d[j] = s * (1.f + z[j] * (1.f - s));
          z[j] *= s;
        } else {
          z[j] = s;
          d[j] = s * (1.f - s);
        }
      }
    }
  }
}

// Pre-activations kept for the backward: fp32 values, or (16-bit types) the upper 24 bits of fp32 values, 16 of them in
// p and 8 in low.
struct Saved {
  void *p;
  uint8_t *low;
};

// What becomes of a product.  One product: out = act(p + bias[0]) + residual, save = p + bias[0].  A pair (g, u):
// out = act(g + bias[0]) * (u + bias[1]), save = g + bias[0] in columns [0, N) and u + bias[1] in [save_up, +N).
// Rows: row m < split goes to out if m < live, else row m - split to out2 if that is < live (the two weight
// gradients of a pair are one product); otherwise split is above every row and live = all rows.
struct Epilogue {
  const void *bias[2];
  const void *residual;
  long long ldr;
  void *out, *out2;
  long long ldo;
  int split, live;
  Saved save;
  long long lds;
  int save_up;
  int act;
  int vec;  // every pointer 16-byte aligned, every row stride and save_up a multiple of 16 bytes in the type of x
};

// W consecutive elements from / to p, `left` of them exist; vec: in accesses of 8 or 16 bytes where W elements fill them
template <typename T, int W>
__device__ __forceinline__ void load_row(const T *p, bool vec, int left, float (&v)[W]) {
  constexpr int kBytes = W * (int)sizeof(T), kPer = 16 / (int)sizeof(T);
  if constexpr (kBytes == 8) {
    if (vec && left >= W) {
      const uint2 r = *reinterpret_cast<const uint2 *>(p);
      const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = Cvt<T>::to_f(h[j]);
      return;
    }
  } else if constexpr (kBytes % 16 == 0) {
    if (vec && left >= W) {
#pragma unroll
      for (int i = 0; i < W / kPer; ++i) {
        const uint4 r = *reinterpret_cast<const uint4 *>(p + i * kPer);
        const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[i * kPer + j] = Cvt<T>::to_f(h[j]);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = j < left ? Cvt<T>::to_f(p[j]) : 0.f;
}
template <typename T, int W>
__device__ __forceinline__ void store_row(T *p, bool vec, int left, const float (&v)[W]) {
  constexpr int kBytes = W * (int)sizeof(T), kPer = 16 / (int)sizeof(T);
  if constexpr (kBytes == 8) {
    if (vec && left >= W) {
      uint2 r;
      T *h = reinterpret_cast<T *>(&r);
#pragma unroll
      for (int j = 0; j < W; ++j) h[j] = Cvt<T>::from_f(v[j]);
      *reinterpret_cast<uint2 *>(p) = r;
      return;
    }
  } else if constexpr (kBytes % 16 == 0) {
    if (vec && left >= W) {
#pragma unroll
      for (int i = 0; i < W / kPer; ++i) {
        uint4 r;
        T *h = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int j = 0; j < kPer; ++j) h[j] = Cvt<T>::from_f(v[i * kPer + j]);
        *reinterpret_cast<uint4 *>(p + i * kPer) = r;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < left) p[j] = Cvt<T>::from_f(v[j]);
}

// W kept values at offset `off` (W a multiple of 8 where vec is set for a 16-bit type)
template <typename T, int W>
__device__ __forceinline__ void store_saved(const Saved &s, long long off, bool vec, int left, const float (&v)[W]) {
  if constexpr (sizeof(T) == 4) {
    store_row<float, W>(static_cast<float *>(s.p) + off, vec, left, v);
  } else {
    uint16_t *hi = static_cast<uint16_t *>(s.p) + off;
    uint8_t *lo = s.low + off;
    if constexpr (W % 8 == 0) {
      if (vec && left >= W) {
#pragma unroll
        for (int i = 0; i < W; i += 8) {
          uint32_t u[8], h[4], l[2];
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(v[i + j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = __byte_perm(u[2 * j], u[2 * j + 1], 0x7632);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            l[j] = __byte_perm(__byte_perm(u[4 * j], u[4 * j + 1], 0x0051), __byte_perm(u[4 * j + 2], u[4 * j + 3], 0x0051),
                               0x5410);
          *reinterpret_cast<uint4 *>(hi + i) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint2 *>(lo + i) = make_uint2(l[0], l[1]);
        }
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < left) {
        hi[j] = (uint16_t)(__float_as_uint(v[j]) >> 16);
        lo[j] = (uint8_t)(__float_as_uint(v[j]) >> 8);
      }
  }
}
// Eight kept values of 24 bits out of their upper 16 and lower 8.  The 8 bits that were cut off are filled with a copy of
// the lower 8: one instruction a value, and the errors of the cut are centred.
__device__ __forceinline__ void kept_values(const uint4 &h4, const uint2 &l2, float *v) {
  const uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[2] = {l2.x, l2.y};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] = __uint_as_float(__byte_perm(l[j / 4], h[j / 2], (j % 4) * 0x11 + (j % 2 ? 0x7600 : 0x5400)));
}
// one kept value, with the same filling
template <typename T> __device__ __forceinline__ float kept_value(const Saved &s, long long off) {
  if constexpr (sizeof(T) == 4) return static_cast<const float *>(s.p)[off];
  else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(s.p)[off] << 16 | (uint32_t)s.low[off] * 0x101u);
}

template <typename T, int W>
__device__ __forceinline__ void add_row(const void *p, long long off, bool vec, int left, float (&v)[W]) {
  if (p == nullptr) return;
  float b[W];
  load_row<T, W>(static_cast<const T *>(p) + off, vec, left, b);
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] += b[j];
}

// where row m of the result goes, or null
template <typename T>
__device__ __forceinline__ T *out_row(const Epilogue &e, long long m) {
  if (m < e.split) return m < e.live ? static_cast<T *>(e.out) + m * e.ldo : nullptr;
  return m - e.split < e.live ? static_cast<T *>(e.out2) + (m - e.split) * e.ldo : nullptr;
}

// columns [n, n + W) of row m (N columns in all); p, g, u hold the raw products and are overwritten
template <typename T, int W>
__device__ __forceinline__ void finish_one(const Epilogue &e, long long m, int n, int N, float (&p)[W]) {
  const int left = N - n;
  T *row = out_row<T>(e, m);
  if (left <= 0 || row == nullptr) return;
  add_row<T, W>(e.bias[0], n, e.vec, left, p);
  if (e.save.p != nullptr) store_saved<T, W>(e.save, m * e.lds + n, e.vec, left, p);
  activate<T, W>(p, e.act);
  add_row<T, W>(e.residual, m * e.ldr + n, e.vec, left, p);
  store_row<T, W>(row + n, e.vec, left, p);
}
template <typename T, int W>
__device__ __forceinline__ void finish_pair(const Epilogue &e, long long m, int n, int N, float (&g)[W], float (&u)[W]) {
  const int left = N - n;
  T *row = out_row<T>(e, m);
  if (left <= 0 || row == nullptr) return;
  add_row<T, W>(e.bias[0], n, e.vec, left, g);
  add_row<T, W>(e.bias[1], n, e.vec, left, u);
  if (e.save.p != nullptr) {
    store_saved<T, W>(e.save, m * e.lds + n, e.vec, left, g);
    store_saved<T, W>(e.save, m * e.lds + e.save_up + n, e.vec, left, u);
  }
  activate<T, W>(g, e.act);
#pragma unroll
  for (int j = 0; j < W; ++j) g[j] *= u[j];
  store_row<T, W>(row + n, e.vec, left, g);
}

// One operand of a product: element (r, k) of row r and contraction index k at p[r * ld + k], or, with the rows
// next to each other (mn_major), at p[k * ld + r].
struct Operand {
  const void *p;
  long long ld;
  int mn_major;
};

// C[m][n] = sum over segments s and k < K[s] of A_s(m, k) B_s(n, k); a pair: segment 0 of B gives g, segment 1 gives u,
// both with A_0 and K[0].
struct Product {
  Operand a[2], b[2];
  int64_t K[2];
  int segments, pair;
  int64_t M, N;
  Epilogue e;
};

int sm_count();  // of the current device (148 where there is none); linear.cu

// gemm_sm100.cu, for 16-bit operands with 16-byte aligned addresses and row strides: columns of a tile, units of a split tile,
// tiles that are done whole, rows of a split tile, and the workspace for their sums.
struct GemmPlan {
  int bn, splits;
  int64_t whole, rows, partial_bytes;
};
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K0, int64_t K1, bool pair);
int gemm_launch(const Product &p, const GemmPlan &plan, float *partial, int dtype, cudaStream_t st);

// Tensor map of an (outer, inner) matrix of 16-bit elements, inner next to each other, rows `ld` elements apart; boxes of 64
// inner elements (128 bytes, swizzled) by `rows` outer ones, zeros outside.
int make_map_2d(CUtensorMap *m, const void *p, int dtype, int64_t inner, int64_t outer, int64_t ld, int rows);

// few_tokens.cu: whether a product is its kind, and the launch (same alignment).
bool few_tokens_fit(const Product &p, int dtype);
int few_tokens_launch(const Product &p, int dtype, cudaStream_t st);

}  // namespace lin
}  // namespace la
