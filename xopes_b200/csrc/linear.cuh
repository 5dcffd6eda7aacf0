// Pieces shared by the kernels of linear_fn and gated_linear_fn: what happens to a product before it is written
// (bias, activation, product of the pair, residual), and the description of a product.
#pragma once
#include "common.cuh"

namespace la {
namespace lin {

enum { kActNone = 0, kActRelu = 1, kActSigmoid = 2, kActSilu = 3, kActGelu = 4 };

// e^x: 2 ulp for fp32 results; the fast form (2 + 1.2 |x| ulp) where the result is rounded to 16 bits
template <typename T> __device__ __forceinline__ float exp_of(float x) { return __expf(x); }
template <> __device__ __forceinline__ float exp_of<float>(float x) { return expf(x); }
template <typename T> __device__ __forceinline__ float inverse_of(float x) { return __fdividef(1.f, x); }
template <> __device__ __forceinline__ float inverse_of<float>(float x) { return 1.f / x; }
// 1 / (1 + e^-z); the fast quotient returns 0 for divisors above 2^126, which is what the sigmoid is there
template <typename T> __device__ __forceinline__ float sigmoid_of(float z) { return inverse_of<T>(1.f + exp_of<T>(-z)); }

template <typename T>
__device__ __forceinline__ float act_of(float z, int kind) {
  switch (kind) {
    case kActRelu: return z > 0.f || z != z ? z : 0.f;
    case kActSigmoid: return sigmoid_of<T>(z);
    case kActSilu: return z * sigmoid_of<T>(z);
    case kActGelu: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  }
  return z;
}

// the activation and its derivative
template <typename T>
__device__ __forceinline__ float act_grad_of(float z, int kind, float &a) {
  switch (kind) {
    case kActRelu: a = z > 0.f || z != z ? z : 0.f; return z > 0.f ? 1.f : 0.f;
    case kActSigmoid: a = sigmoid_of<T>(z); return a * (1.f - a);
    case kActSilu: {
      const float s = sigmoid_of<T>(z);
      a = z * s;
      return s * (1.f + z * (1.f - s));
    }
    case kActGelu: {
      const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      a = z * cdf;
      return cdf + z * 0.3989422804014327f * exp_of<T>(-0.5f * z * z);
    }
  }
  a = z;
  return 1.f;
}

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
  void *save;
  long long lds;
  int save_up;
  int act;
  int vec;  // every pointer 16-byte aligned, every row stride and save_up a multiple of 16 bytes
};

// W consecutive elements (W sizeof(T) = 8 or a multiple of 16 bytes) from / to p; `left` of them exist
template <typename T, int W>
__device__ __forceinline__ void load_row(const T *p, bool vec, int left, float (&v)[W]) {
  if (vec && left >= W) {
    constexpr int kBytes = W * (int)sizeof(T);
    if constexpr (kBytes == 8) {
      const uint2 r = *reinterpret_cast<const uint2 *>(p);
      const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = Cvt<T>::to_f(h[j]);
    } else {
      constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < W / kPer; ++i) {
        const uint4 r = *reinterpret_cast<const uint4 *>(p + i * kPer);
        const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[i * kPer + j] = Cvt<T>::to_f(h[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = j < left ? Cvt<T>::to_f(p[j]) : 0.f;
  }
}
template <typename T, int W>
__device__ __forceinline__ void store_row(T *p, bool vec, int left, const float (&v)[W]) {
  if (vec && left >= W) {
    constexpr int kBytes = W * (int)sizeof(T);
    if constexpr (kBytes == 8) {
      uint2 r;
      T *h = reinterpret_cast<T *>(&r);
#pragma unroll
      for (int j = 0; j < W; ++j) h[j] = Cvt<T>::from_f(v[j]);
      *reinterpret_cast<uint2 *>(p) = r;
    } else {
      constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < W / kPer; ++i) {
        uint4 r;
        T *h = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int j = 0; j < kPer; ++j) h[j] = Cvt<T>::from_f(v[i * kPer + j]);
        *reinterpret_cast<uint4 *>(p + i * kPer) = r;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < left) p[j] = Cvt<T>::from_f(v[j]);
  }
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
  if (e.save != nullptr) store_row<T, W>(static_cast<T *>(e.save) + m * e.lds + n, e.vec, left, p);
  if (e.act != kActNone) {
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = act_of<T>(p[j], e.act);
  }
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
  if (e.save != nullptr) {
    T *s = static_cast<T *>(e.save) + m * e.lds + n;
    store_row<T, W>(s, e.vec, left, g);
    store_row<T, W>(s + e.save_up, e.vec, left, u);
  }
#pragma unroll
  for (int j = 0; j < W; ++j) g[j] = act_of<T>(g[j], e.act) * u[j];
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

}  // namespace lin
}  // namespace la
