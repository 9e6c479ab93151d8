// Layer norm over the last dimension, forward and backward:
//   xh = (x - mean) rstd,  y = xh w + b;   h = dy w,  dx = rstd (h - mean(h) - xh mean(h xh)),  dw = sum dy xh,  db = sum dy.
//
// Streaming kernels, bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.  A row is held in the
// registers of one warp or of one CTA, so that mean, variance (of the centred values) and result take one read of it.  An
// element lies with the same thread in every row of a CTA: the weight's and the bias's gradients are sums in registers, left
// once per CTA and added up by a second kernel in a fixed order.
// The next row of a CTA is asked for before the reductions of the one at hand.  32,768 x 2,048 of bf16: forward 49 us = 0.84 of the
// copy rate, backward 88 us = 0.70 of it (its registers leave two CTAs of 256 threads on an SM).
#include "pkda_common.cuh"
#include "pkda_launch.h"

#include <algorithm>
#include <type_traits>

namespace pkda {

struct LayerNormParams {
  long long rows;
  int dim;
  float eps, inv_dim;
  const void *x, *dy;
  const float *w, *b;
  void *y, *dx;
  float *mean, *rstd;
  float* part;  // [groups][2][dim], or NULL
  int groups;
};

namespace ln {

// How a thread holds its share of a row: kVecs pieces of kPer elements, piece j at (j * TPR + t) * kPer.
template <typename T, bool kWide> struct Piece;
template <> struct Piece<bf16, true> {
  static constexpr int kPer = 8;
  using Raw = uint4;
  static __device__ __forceinline__ Raw load(const bf16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = unpack_bf16(w[j]);
      f[2 * j] = a.x;
      f[2 * j + 1] = a.y;
    }
  }
  static __device__ __forceinline__ void store(bf16* p, const float* f) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
};
template <> struct Piece<float, true> {
  static constexpr int kPer = 4;
  using Raw = float4;
  static __device__ __forceinline__ Raw load(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
  static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <typename T> struct Piece<T, false> {
  static constexpr int kPer = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw load(const T* p) { return __ldg(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = to_f(r); }
  static __device__ __forceinline__ void store(T* p, const float* f) { *p = from_f<T>(f[0]); }
};

// Elements of a thread: 8 where a row has up to 8 per thread of the widest CTA, else 16.
template <typename T, bool kWide, int kElems> struct Row {
  using P = Piece<T, kWide>;
  static constexpr int kVecs = kElems / P::kPer;
  typename P::Raw raw[kVecs];
  __device__ __forceinline__ void load(const T* row, int t, int tpr, int dim) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int at = (j * tpr + t) * P::kPer;
      raw[j] = typename P::Raw{};
      if (at < dim) raw[j] = P::load(row + at);
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[kElems]) const {  // (zeros past the row)
#pragma unroll
    for (int j = 0; j < kVecs; ++j) P::unpack(raw[j], f + j * P::kPer);
  }
};
template <typename T, bool kWide, int kElems>
__device__ __forceinline__ void store_row(T* row, const float (&f)[kElems], int t, int tpr, int dim) {
  using P = Piece<T, kWide>;
#pragma unroll
  for (int j = 0; j < kElems / P::kPer; ++j) {
    const int at = (j * tpr + t) * P::kPer;
    if (at < dim) P::store(row + at, f + j * P::kPer);
  }
}
// A thread's piece j of a parameter; `none` where there is none.  (Rows in whole pieces have parameters on 16 bytes.)
template <typename T, bool kWide>
__device__ __forceinline__ void load_piece(const float* p, float none, float* f, int at, int dim) {
  constexpr int kPer = Piece<T, kWide>::kPer;
  if constexpr (kWide) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const float4 v = p && at < dim ? __ldg(reinterpret_cast<const float4*>(p + at + i)) : make_float4(none, none, none, none);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else {
    f[0] = p && at < dim ? __ldg(p + at) : none;
  }
}
template <typename T, bool kWide, int kElems>
__device__ __forceinline__ void load_param(const float* p, float none, float (&f)[kElems], int t, int tpr, int dim) {
  constexpr int kPer = Piece<T, kWide>::kPer;
#pragma unroll
  for (int j = 0; j < kElems / kPer; ++j) load_piece<T, kWide>(p, none, f + j * kPer, (j * tpr + t) * kPer, dim);
}

template <int TPR> __host__ __device__ constexpr int threads() { return TPR < 256 ? (TPR == 32 ? 256 : TPR) : TPR; }

// Sums over the TPR threads of a row of one, two or four values at once, every thread gets them.  The first rounds of shuffles
// halve the number of values instead (a lane keeps the half that its bit names), and a warp adds up the sums of all warps, a value
// and warp to a lane: 4 values over 256 threads take 14 shuffles, 36 one by one.  One barrier: what is written there is read
// before the next barrier of the same kind but one, which uses the other half of s_red.
template <int TPR, int kN>
__device__ __forceinline__ void row_sums(float (&v)[kN], float (*s_red)[32], int slot) {
  static_assert(kN == 1 || kN == 2 || kN == 4);
  constexpr int kWarps = TPR / 32, kAll = kWarps * kN, kSpan = 32 / kN;  // (lanes that hold the same value)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float x[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) x[i] = v[i];
#pragma unroll
  for (int o = 16, n = kN / 2; o; o >>= 1, n >>= 1) {
    if (n) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float give = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
        x[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    } else {
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], o);
    }
  }
  if (TPR == 32) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __shfl_sync(0xffffffffu, x[0], i * kSpan);
    return;
  }
  float* red = s_red[slot * kN];
  if (lane % kSpan == 0) red[warp * kN + lane / kSpan] = x[0];
  __syncthreads();
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < kAll; e += 32) a += kAll >= 32 || lane < kAll ? red[e + lane] : 0.f;
#pragma unroll
  for (int o = (kAll < 32 ? kAll : 32) / 2; o >= kN; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = __shfl_sync(0xffffffffu, a, i);
}

// TPR threads a row: a warp (eight rows a CTA), or the whole CTA; kRows rows a turn, whose sums share their barriers.
template <typename T, bool kWide, int TPR, int kElems, int kRows>
__global__ void __launch_bounds__(threads<TPR>()) layer_norm_fwd_kernel(const LayerNormParams p) {
  after_previous();
  __shared__ float s_red[2 * kRows][32];
  constexpr int kTeams = threads<TPR>() / TPR, kPer = Piece<T, kWide>::kPer;
  const int t = threadIdx.x % TPR, dim = p.dim;
  const long long step = (long long)gridDim.x * kTeams * kRows;
  long long r = ((long long)blockIdx.x * kTeams + threadIdx.x / TPR) * kRows;
  const T* x = static_cast<const T*>(p.x);
  Row<T, kWide, kElems> next[kRows];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (row + i < p.rows) next[i].load(x + (size_t)(row + i) * dim, t, TPR, dim);
  };
  fetch(r);
  constexpr bool kHeld = kElems == 8;  // (sixteen of each do not fit beside the row: from the cache, row by row)
  float w[kHeld ? kElems : 1], b[kHeld ? kElems : 1];
  if constexpr (kHeld) {
    load_param<T, kWide, kElems>(p.w, 1.f, w, t, TPR, dim);
    load_param<T, kWide, kElems>(p.b, 0.f, b, t, TPR, dim);
  }
  for (; r < p.rows; r += step) {
    float f[kRows][kElems], mean[kRows], rstd[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      next[i].unpack(f[i]);
      mean[i] = 0.f;
#pragma unroll
      for (int e = 0; e < kElems; ++e) mean[i] += f[i][e];
    }
    fetch(r + step);
    row_sums<TPR, kRows>(mean, s_red, 0);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      mean[i] *= p.inv_dim;
      rstd[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kElems / kPer; ++j) {
        float sq = 0.f;
#pragma unroll
        for (int e = j * kPer; e < (j + 1) * kPer; ++e) {
          f[i][e] -= mean[i];
          sq += f[i][e] * f[i][e];
        }
        rstd[i] += (j * TPR + t) * kPer < dim ? sq : 0.f;
      }
    }
    row_sums<TPR, kRows>(rstd, s_red, 1);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (r + i >= p.rows) break;
      rstd[i] = rsqrtf(rstd[i] * p.inv_dim + p.eps);
#pragma unroll
      for (int j = 0; j < kElems / kPer; ++j) {
        float wr[kPer], br[kPer];
        if constexpr (!kHeld) {
          load_piece<T, kWide>(p.w, 1.f, wr, (j * TPR + t) * kPer, dim);
          load_piece<T, kWide>(p.b, 0.f, br, (j * TPR + t) * kPer, dim);
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          float& y = f[i][j * kPer + e];
          if constexpr (kHeld) y = y * rstd[i] * w[j * kPer + e] + b[j * kPer + e];
          else y = y * rstd[i] * wr[e] + br[e];
        }
      }
      store_row<T, kWide, kElems>(static_cast<T*>(p.y) + (size_t)(r + i) * dim, f[i], t, TPR, dim);
      if (t == 0) {
        if (p.mean) p.mean[r + i] = mean[i];
        if (p.rstd) p.rstd[r + i] = rstd[i];
      }
    }
  }
}

// Sixteen elements a thread leave no registers for the sums over the rows (1,024 x 16 elements: 74 us backward for 1,024 rows of
// bf16 with what that spills): they lie in shared memory then, four floats a thread and access, read and written by their own
// thread alone, and the weight is read row by row from the cache.
template <int TPR, int kElems> __host__ __device__ constexpr bool sums_in_smem() { return kElems == 16; }
template <int TPR, int kElems> __host__ __device__ constexpr int bwd_smem() { return sums_in_smem<TPR, kElems>() ? 2 * kElems * TPR * 4 : 0; }

template <typename T, bool kWide, int TPR, int kElems, int kRows>
__global__ void __launch_bounds__(threads<TPR>()) layer_norm_bwd_kernel(const LayerNormParams p) {
  after_previous();
  extern __shared__ float4 s_acc[];  // [2][kElems / 4][TPR]
  __shared__ float s_red[4 * kRows][32];
  constexpr bool kShared = sums_in_smem<TPR, kElems>();
  constexpr int kTeams = threads<TPR>() / TPR, kPer = Piece<T, kWide>::kPer, kSums = kShared ? 1 : kElems;
  const int t = threadIdx.x % TPR, dim = p.dim;
  const long long step = (long long)gridDim.x * kTeams * kRows;
  long long r = ((long long)blockIdx.x * kTeams + threadIdx.x / TPR) * kRows;
  const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
  Row<T, kWide, kElems> nx[kRows], nd[kRows];
  float n_mean[kRows], n_rstd[kRows];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (row + i < p.rows) {
        nx[i].load(x + (size_t)(row + i) * dim, t, TPR, dim);
        nd[i].load(dy + (size_t)(row + i) * dim, t, TPR, dim);
        n_mean[i] = __ldg(p.mean + row + i);
        n_rstd[i] = __ldg(p.rstd + row + i);
      }
  };
  if (!kShared) fetch(r);
  float w[kSums], dw[kSums], db[kSums];
  if (kShared) {
#pragma unroll
    for (int j = 0; j < 2 * kElems / 4; ++j) s_acc[j * TPR + t] = make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    load_param<T, kWide, kSums>(p.w, 1.f, w, t, TPR, dim);
#pragma unroll
    for (int e = 0; e < kSums; ++e) dw[e] = db[e] = 0.f;
  }
  for (int it = 0; r < p.rows; r += step, ++it) {
    float f[kRows][kElems], d[kRows][kElems], sum[2 * kRows], rstd[kRows];
    if (kShared) fetch(r);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool here = r + i < p.rows;
      nx[i].unpack(f[i]);
      nd[i].unpack(d[i]);
      rstd[i] = n_rstd[i];
      const float mean = n_mean[i];
      sum[2 * i] = sum[2 * i + 1] = 0.f;
      if (!here) {
#pragma unroll
        for (int e = 0; e < kElems; ++e) f[i][e] = d[i][e] = 0.f;
        continue;
      }
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        f[i][e] = (f[i][e] - mean) * rstd[i];  // (elements past the row: their cotangent is zero)
        if (!kShared) {
          dw[e % kSums] += d[i][e] * f[i][e];
          db[e % kSums] += d[i][e];
          d[i][e] *= w[e % kSums];
        }
      }
      if (kShared) {
#pragma unroll
        for (int j = 0; j < kElems / 4; ++j) {
          float4 a = s_acc[j * TPR + t], c = s_acc[(kElems / 4 + j) * TPR + t];
          const int k = 4 * j;
          a.x += d[i][k] * f[i][k];         a.y += d[i][k + 1] * f[i][k + 1];
          a.z += d[i][k + 2] * f[i][k + 2]; a.w += d[i][k + 3] * f[i][k + 3];
          c.x += d[i][k]; c.y += d[i][k + 1]; c.z += d[i][k + 2]; c.w += d[i][k + 3];
          s_acc[j * TPR + t] = a;
          s_acc[(kElems / 4 + j) * TPR + t] = c;
        }
#pragma unroll
        for (int j = 0; j < kElems / kPer; ++j) {
          float wr[kPer];
          load_piece<T, kWide>(p.w, 1.f, wr, (j * TPR + t) * kPer, dim);
#pragma unroll
          for (int e = 0; e < kPer; ++e) d[i][j * kPer + e] *= wr[e];
        }
      }
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        sum[2 * i] += d[i][e];
        sum[2 * i + 1] += d[i][e] * f[i][e];
      }
    }
    if (!kShared) fetch(r + step);
    row_sums<TPR, 2 * kRows>(sum, s_red, it & 1);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (r + i >= p.rows) break;
      const float m1 = sum[2 * i] * p.inv_dim, m2 = sum[2 * i + 1] * p.inv_dim;
#pragma unroll
      for (int e = 0; e < kElems; ++e) d[i][e] = rstd[i] * (d[i][e] - m1 - f[i][e] * m2);
      store_row<T, kWide, kElems>(static_cast<T*>(p.dx) + (size_t)(r + i) * dim, d[i], t, TPR, dim);
    }
  }
  if (!p.part) return;
  float* part = p.part + (size_t)blockIdx.x * 2 * dim;
  if (TPR == 32) {  // the CTA's eight warps hold the same elements: one after the other through shared memory
    __shared__ float s_sum[TPR == 32 ? kTeams : 1][TPR == 32 ? 32 * kElems : 1];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kSums; ++e) s_sum[threadIdx.x / TPR][e * 32 + t] = which ? db[e] : dw[e];
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * kElems; i += threads<TPR>()) {
        const int e = i / 32, at = ((e / kPer) * TPR + i % 32) * kPer + e % kPer;
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < kTeams; ++k) a += s_sum[k][i];
        if (at < dim) part[(size_t)which * dim + at] = a;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
      const int at = ((e / kPer) * TPR + t) * kPer + e % kPer;
      if (at < dim) {
        part[at] = kShared ? reinterpret_cast<const float*>(s_acc)[((e / 4) * TPR + t) * 4 + e % 4] : dw[e % kSums];
        part[dim + at] = kShared ? reinterpret_cast<const float*>(s_acc)[((kElems / 4 + e / 4) * TPR + t) * 4 + e % 4] : db[e % kSums];
      }
    }
  }
}

// Sum over the TPR threads of a row, the same value in each.  `slot` alternates between uses that follow one another, so
// that one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float2 (*s_red)[32], int slot) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (TPR == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) s_red[slot][warp] = v;
  __syncthreads();
  constexpr int kWarps = TPR / 32;
  v = lane < kWarps ? s_red[slot][lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = kWarps / 2; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, v.x, 0), __shfl_sync(0xffffffffu, v.y, 0));
}

// Rows wider than a CTA's registers: three passes over the row (which the cache holds), a CTA per row.
constexpr int kLongThreads = 512;
template <typename T> __global__ void __launch_bounds__(kLongThreads) layer_norm_fwd_long_kernel(const LayerNormParams p) {
  after_previous();
  __shared__ float2 s_red[2][32];
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + (size_t)r * p.dim;
    float s = 0.f;
    for (int i = threadIdx.x; i < p.dim; i += kLongThreads) s += to_f(x[i]);
    const float mean = row_sum2<kLongThreads>(make_float2(s, 0.f), s_red, 0).x * p.inv_dim;
    s = 0.f;
    for (int i = threadIdx.x; i < p.dim; i += kLongThreads) {
      const float c = to_f(x[i]) - mean;
      s += c * c;
    }
    const float rstd = 1.f / sqrtf(row_sum2<kLongThreads>(make_float2(s, 0.f), s_red, 1).x * p.inv_dim + p.eps);
    T* y = static_cast<T*>(p.y) + (size_t)r * p.dim;
    for (int i = threadIdx.x; i < p.dim; i += kLongThreads)
      y[i] = from_f<T>((to_f(x[i]) - mean) * rstd * (p.w ? p.w[i] : 1.f) + (p.b ? p.b[i] : 0.f));
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}
template <typename T> __global__ void __launch_bounds__(kLongThreads) layer_norm_bwd_long_kernel(const LayerNormParams p) {
  after_previous();
  __shared__ float2 s_red[2][32];
  int it = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, ++it) {
    const T* x = static_cast<const T*>(p.x) + (size_t)r * p.dim;
    const T* dy = static_cast<const T*>(p.dy) + (size_t)r * p.dim;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float2 s = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < p.dim; i += kLongThreads) {
      const float h = to_f(dy[i]) * (p.w ? p.w[i] : 1.f);
      s.x += h;
      s.y += h * (to_f(x[i]) - mean) * rstd;
    }
    s = row_sum2<kLongThreads>(s, s_red, it & 1);
    T* dx = static_cast<T*>(p.dx) + (size_t)r * p.dim;
    for (int i = threadIdx.x; i < p.dim; i += kLongThreads) {
      const float h = to_f(dy[i]) * (p.w ? p.w[i] : 1.f), xh = (to_f(x[i]) - mean) * rstd;
      dx[i] = from_f<T>(rstd * (h - s.x * p.inv_dim - xh * s.y * p.inv_dim));
    }
  }
}
// Their parameter gradients: a thread per column and slice of rows.
template <typename T> __global__ void __launch_bounds__(256) layer_norm_dw_long_kernel(const LayerNormParams p) {
  after_previous();
  const long long c = blockIdx.x * 256ll + threadIdx.x, per = (p.rows + gridDim.y - 1) / gridDim.y;
  if (c >= p.dim) return;
  float dw = 0.f, db = 0.f;
  const long long end = min((long long)p.rows, (blockIdx.y + 1) * per);
  for (long long r = blockIdx.y * per; r < end; ++r) {
    const float d = to_f(static_cast<const T*>(p.dy)[(size_t)r * p.dim + c]);
    dw += d * (to_f(static_cast<const T*>(p.x)[(size_t)r * p.dim + c]) - p.mean[r]) * p.rstd[r];
    db += d;
  }
  p.part[(size_t)blockIdx.y * 2 * p.dim + c] = dw;
  p.part[(size_t)blockIdx.y * 2 * p.dim + p.dim + c] = db;
}

// Sums the partials [groups][2 dim] in a fixed order: 32 columns a CTA, 32 warps with every 32nd group each.
__global__ void __launch_bounds__(1024) layer_norm_dw_kernel(const float* part, float* dw, float* db, int dim, int groups) {
  after_previous();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32ll + lane;
  float a = 0.f;
  if (c < 2ll * dim) {
#pragma unroll 4
    for (int g = warp; g < groups; g += 32) a += part[(size_t)g * 2 * dim + c];
  }
  s[warp][lane] = a;
  __syncthreads();
  a = s[lane][warp];  // column `warp` of this CTA, partial `lane`
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const long long col = blockIdx.x * 32ll + warp;
  if (lane == 0 && col < 2ll * dim) {
    if (col < dim) {
      if (dw) dw[col] = a;
    } else if (db) {
      db[col - dim] = a;
    }
  }
}

constexpr int kMostGroups = 148 * 8;
constexpr int kLongDim = 16384;  // rows up to here stay in registers (16 elements of 1,024 threads)

// What is launched for a width: threads of a row and elements of a thread, eight or, from 4,097 elements on, sixteen.
template <typename F> static int by_dim(long long dim, F&& f) {
  using std::integral_constant;
  if (dim <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 8>());
  if (dim <= 512) return f(integral_constant<int, 64>(), integral_constant<int, 8>());
  if (dim <= 1024) return f(integral_constant<int, 128>(), integral_constant<int, 8>());
  if (dim <= 2048) return f(integral_constant<int, 256>(), integral_constant<int, 8>());
  if (dim <= 4096) return f(integral_constant<int, 512>(), integral_constant<int, 8>());
  if (dim <= 8192) return f(integral_constant<int, 512>(), integral_constant<int, 16>());
  return f(integral_constant<int, 1024>(), integral_constant<int, 16>());
}

// The most CTAs of a backward, each of which leaves sums of 2 dim floats: what the threads and the shared memory of 148 SMs hold.
static long long most_groups(long long dim) {
  return 148 * by_dim(dim, [](auto tpr, auto elems) {
    constexpr int TPR = decltype(tpr)::value, smem = bwd_smem<TPR, decltype(elems)::value>();
    return std::min({8, 2048 / threads<TPR>(), smem ? 232448 / (smem + 1024) : 8});
  });
}

// CTAs of a persistent launch: what is resident at once, fewer for few rows, never more than the partials' bound.
template <typename K> static int grid_of(K kernel, int threads, int smem, long long ctas) {
  int per_sm = 1;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
  if (per_sm > 8) per_sm = 8;
  const long long cap = std::min((long long)sm_count() * per_sm, (long long)kMostGroups);
  return (int)std::max(1ll, std::min(ctas, cap));
}

static int check(const pkda_layer_norm_args& a, LayerNormParams& p) {
  if (a.rows < 0 || a.dim < 1 || a.dim > (1ll << 30)) return PKDA_ERR_SHAPE;
  if (a.dtype != PKDA_BF16 && a.dtype != PKDA_F32) return PKDA_ERR_DTYPE;
  p.rows = a.rows; p.dim = (int)a.dim; p.eps = a.eps; p.inv_dim = (float)(1.0 / (double)a.dim);
  p.x = a.x; p.dy = a.dy; p.w = a.weight; p.b = a.bias; p.y = a.y; p.dx = a.dx; p.mean = a.mean; p.rstd = a.rstd;
  p.part = nullptr; p.groups = 0;
  return PKDA_OK;
}

// Whole 16-byte pieces in every row?
static bool wide(const pkda_layer_norm_args& a, std::initializer_list<const void*> ptrs) {
  return a.dim % (a.dtype == PKDA_BF16 ? 8 : 4) == 0 && aligned(ptrs, 16);
}

// Rows a turn: two, which share their barriers, where every SM has turns enough for them, so that the smallest calls still spread
// over the chip.  32,768 x 2,048 of bf16, one / two / four: forward 55 / 49 / 57 us, backward 102 / 88 us / no registers for four.
constexpr long long kManyRows = 148 * 16;

template <typename T, bool kWide, int TPR, int kElems, int kRows> static int launch_fwd_rows(const LayerNormParams& p, cudaStream_t st) {
  const auto kernel = layer_norm_fwd_kernel<T, kWide, TPR, kElems, kRows>;
  constexpr int n = threads<TPR>(), rows = n / TPR * kRows;
  return launch_kernel(kernel, grid_of(kernel, n, 0, (p.rows + rows - 1) / rows), n, 0, st, p);
}
template <typename T, bool kWide> static int launch_fwd(const LayerNormParams& p, cudaStream_t st) {
  return by_dim(p.dim, [&](auto tpr, auto elems) {
    constexpr int TPR = decltype(tpr)::value, kElems = decltype(elems)::value;
    if constexpr (kElems == 8) {
      if (p.rows >= kManyRows) return launch_fwd_rows<T, kWide, TPR, kElems, 2>(p, st);
    }
    return launch_fwd_rows<T, kWide, TPR, kElems, 1>(p, st);
  });
}
template <typename T, bool kWide, int TPR, int kElems, int kRows> static int launch_bwd_rows(LayerNormParams& p, cudaStream_t st) {
  const auto kernel = layer_norm_bwd_kernel<T, kWide, TPR, kElems, kRows>;
  constexpr int n = threads<TPR>(), rows = n / TPR * kRows, smem = bwd_smem<TPR, kElems>();
  if (smem && !ensure_dynamic_smem(kernel, smem)) return PKDA_ERR_LAUNCH;
  // every CTA leaves sums for the second kernel: few rows do not take more CTAs than pay for them
  const long long turns = (p.rows + rows - 1) / rows, least = (turns + 3) / 4, sms = sm_count();
  p.groups = grid_of(kernel, n, smem, std::min(turns < sms ? turns : std::max(least, sms), most_groups(p.dim)));
  return launch_kernel(kernel, p.groups, n, smem, st, p);
}
template <typename T, bool kWide> static int launch_bwd(LayerNormParams& p, cudaStream_t st) {
  return by_dim(p.dim, [&](auto tpr, auto elems) {
    constexpr int TPR = decltype(tpr)::value, kElems = decltype(elems)::value;
    if constexpr (kElems == 8 && TPR < 512) {
      if (p.rows >= kManyRows) return launch_bwd_rows<T, kWide, TPR, kElems, 2>(p, st);
    }
    return launch_bwd_rows<T, kWide, TPR, kElems, 1>(p, st);
  });
}
template <typename T> static int launch_long_bwd(LayerNormParams& p, cudaStream_t st) {
  int rc = launch_kernel(layer_norm_bwd_long_kernel<T>, (int)std::min(p.rows, (long long)sm_count() * 4), kLongThreads, 0, st, p);
  if (rc != PKDA_OK || !p.part) return rc;
  end_stage(st);
  p.groups = (int)std::min(p.rows, 32ll);
  begin_stage(kStageLayerNormDw, st);
  return launch_kernel(layer_norm_dw_long_kernel<T>, dim3((p.dim + 255) / 256, p.groups), 256, 0, st, p);
}

}  // namespace ln

int layer_norm_fwd(const pkda_layer_norm_args* a, cudaStream_t st) {
  LayerNormParams p;
  int rc = ln::check(*a, p);
  if (rc != PKDA_OK || a->rows == 0) return rc;
  if (!a->x || !a->y) return PKDA_ERR_NULL;
  const bool f32 = a->dtype == PKDA_F32;
  begin_stage(kStageLayerNormFwd, st);
  if (a->dim > ln::kLongDim) {
    const int grid = (int)std::min(p.rows, (long long)sm_count() * 4);
    rc = f32 ? launch_kernel(ln::layer_norm_fwd_long_kernel<float>, grid, ln::kLongThreads, 0, st, p)
             : launch_kernel(ln::layer_norm_fwd_long_kernel<bf16>, grid, ln::kLongThreads, 0, st, p);
  } else if (ln::wide(*a, {a->x, a->y, a->weight, a->bias})) {
    rc = f32 ? ln::launch_fwd<float, true>(p, st) : ln::launch_fwd<bf16, true>(p, st);
  } else {
    rc = f32 ? ln::launch_fwd<float, false>(p, st) : ln::launch_fwd<bf16, false>(p, st);
  }
  end_stage(st);
  return rc;
}

size_t layer_norm_bwd_workspace(const pkda_layer_norm_args& a) {
  LayerNormParams p;
  if (ln::check(a, p) != PKDA_OK) return 0;
  const long long groups = a.dim > ln::kLongDim ? 32 : ln::most_groups(a.dim);
  return align_up((size_t)std::min(groups, std::max(a.rows, 1ll)) * 2 * a.dim * sizeof(float));
}

int layer_norm_bwd(const pkda_layer_norm_args* a, cudaStream_t st) {
  LayerNormParams p;
  int rc = ln::check(*a, p);
  if (rc != PKDA_OK) return rc;
  if (a->rows == 0) {
    for (float* d : {a->dweight, a->dbias})
      if (d && cudaMemsetAsync(d, 0, (size_t)a->dim * sizeof(float), st) != cudaSuccess) return launch_code(cudaErrorUnknown);
    return PKDA_OK;
  }
  if (!a->x || !a->dy || !a->dx || !a->mean || !a->rstd) return PKDA_ERR_NULL;
  const bool params = a->dweight || a->dbias, f32 = a->dtype == PKDA_F32;
  if (params) {
    if (!a->workspace || a->workspace_bytes < layer_norm_bwd_workspace(*a)) return PKDA_ERR_WORKSPACE;
    if (!aligned({a->workspace}, 4)) return PKDA_ERR_ALIGN;
    p.part = static_cast<float*>(a->workspace);
  }
  begin_stage(kStageLayerNormBwd, st);
  if (a->dim > ln::kLongDim)
    rc = f32 ? ln::launch_long_bwd<float>(p, st) : ln::launch_long_bwd<bf16>(p, st);
  else if (ln::wide(*a, {a->x, a->dy, a->dx, a->weight}))
    rc = f32 ? ln::launch_bwd<float, true>(p, st) : ln::launch_bwd<bf16, true>(p, st);
  else
    rc = f32 ? ln::launch_bwd<float, false>(p, st) : ln::launch_bwd<bf16, false>(p, st);
  end_stage(st);
  if (rc != PKDA_OK || !params) return rc;
  begin_stage(kStageLayerNormDw, st);
  rc = launch_kernel(ln::layer_norm_dw_kernel, (int)((2 * a->dim + 31) / 32), 1024, 0, st, p.part, a->dweight, a->dbias, p.dim, p.groups);
  end_stage(st);
  return rc;
}

}  // namespace pkda
