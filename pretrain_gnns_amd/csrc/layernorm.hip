// Layer normalisation of rows (torch.nn.LayerNorm over the last axis), with an optional ReLU, forward and backward:
//   mu = mean_c x, v = mean_c (x - mu)^2, r = (v + eps)^-1/2, xh = (x - mu) r, y = relu?(xh gamma + beta)
//   h = dy [xh gamma + beta > 0, with the ReLU], g = h gamma,  dx = r (g - mean_c g - xh mean_c (g xh))
//   dgamma = sum_rows h xh, dbeta = sum_rows h
// Both directions are HBM-bound: 2 and 3 passes over a matrix.  A row is read ONCE: it stays in the registers of the LPR lanes that
// share it (16, a wave or a workgroup), so the variance is that of the centred values (two passes over registers, not the
// difference of two large sums).  Statistics, sums and products are fp32 whatever the rows' type; y and dx are rounded once.  The
// backward keeps its columns' share of dgamma / dbeta in registers over all rows of a lane group, writes one partial per workgroup
// and a second launch adds the partials in float64 in a fixed order: no atomics, bitwise reproducible.
#include <algorithm>
#include <type_traits>

#include "common.h"

using namespace pgnn;

namespace {

constexpr int kBlock = 256;
constexpr int kRegDim = 8192;    // widest row that is kept in registers (256 lanes x 32 values); wider rows are re-read from L2
constexpr int kWideBlock = 1024;

// 16 bytes of a row, at the element's own alignment: odd widths and strides take the same loads (global memory takes any
// alignment; a vector that straddles a line costs one more request)
template <typename T> struct Pack;
template <> struct Pack<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); static constexpr int n = 4; };
template <> struct Pack<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); static constexpr int n = 8; };
template <> struct Pack<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2))); static constexpr int n = 8; };

// the VE values at column c of a row, zero beyond dim
template <typename T, int VE>
__device__ __forceinline__ void load_cols(const T* __restrict__ row, int c, int dim, float (&v)[VE]) {
  if (c + VE <= dim) {
    if constexpr (Pack<T>::n == VE) {
      const typename Pack<T>::type p = *reinterpret_cast<const typename Pack<T>::type*>(row + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = (float)p[e];
    } else {  // fp32 gains beside 16-bit rows: two vectors
      static_assert(VE == 2 * Pack<T>::n, "");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const typename Pack<T>::type p = *reinterpret_cast<const typename Pack<T>::type*>(row + c + h * Pack<T>::n);
#pragma unroll
        for (int e = 0; e < Pack<T>::n; ++e) v[h * Pack<T>::n + e] = (float)p[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = c + e < dim ? (float)row[c + e] : 0.f;
  }
}

// the same as the 16 bytes that they are in memory (a row that is fetched ahead waits in this form)
template <typename T>
__device__ __forceinline__ typename Pack<T>::type load_pack(const T* __restrict__ row, int c, int dim) {
  typename Pack<T>::type p;
  if (c + Pack<T>::n <= dim) {
    p = *reinterpret_cast<const typename Pack<T>::type*>(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < Pack<T>::n; ++e) p[e] = c + e < dim ? row[c + e] : (T)0.f;
  }
  return p;
}

template <typename T, int VE>
__device__ __forceinline__ void store_cols(T* __restrict__ row, int c, int dim, const float (&v)[VE]) {
  if (c + VE <= dim) {
    typename Pack<T>::type p;
#pragma unroll
    for (int e = 0; e < VE; ++e) p[e] = (T)v[e];
    *reinterpret_cast<typename Pack<T>::type*>(row + c) = p;
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (c + e < dim) row[c + e] = (T)v[e];
  }
}

// sums of N values over the LPR lanes of a row; every lane ends with the same bits.  LPR = 256: across the four waves through LDS
// (`slot` alternates between calls, so one barrier per call is enough)
template <int LPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds, int& slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = row16_sum(v[i]);
    if constexpr (LPR >= 64) {
      v[i] += __shfl_xor(v[i], 16);
      v[i] += __shfl_xor(v[i], 32);
    }
  }
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    float* s = lds + slot * W * N;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = s[i];
#pragma unroll
      for (int w = 1; w < W; ++w) t += s[w * N + i];
      v[i] = t;
    }
    slot ^= 1;
  }
}

template <typename W, int VE>
__device__ __forceinline__ void load_gain(const W* __restrict__ p, int c, int dim, float dflt, float (&v)[VE]) {
  if (p) {
    load_cols<W, VE>(p, c, dim, v);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = dflt;
  }
}

template <typename T, typename W, int LPR, int NV>
__global__ void __launch_bounds__(kBlock) k_layer_norm_fwd(const T* __restrict__ x, int64_t ldx, const W* __restrict__ gamma,
                                                           const W* __restrict__ beta, float eps, int relu, T* __restrict__ y, int64_t ldy,
                                                           float* __restrict__ save_mean, float* __restrict__ save_rstd, int64_t rows, int dim) {
  constexpr int VE = Pack<T>::n, G = kBlock / LPR;
  __shared__ float lds[2 * kBlock / 64];
  int slot = 0;
  const int lane = threadIdx.x % LPR;
  const float inv_dim = 1.f / (float)dim;
  float w[NV][VE], b[NV][VE];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    load_gain<W, VE>(gamma, (lane + LPR * q) * VE, dim, 1.f, w[q]);
    load_gain<W, VE>(beta, (lane + LPR * q) * VE, dim, 0.f, b[q]);
  }
  // whole workgroups iterate together when a row is shared by all of it (the barrier in row_sum); lane groups of 16 and 64 do not meet
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / LPR;
  typename Pack<T>::type ahead[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int q = 0; q < NV; ++q) ahead[q] = load_pack<T>(x + row * ldx, (lane + LPR * q) * VE, dim);
  };
  if (r < rows) fetch(r);
  for (; r < rows; r += step) {
    float v[NV][VE];
    float s[1] = {0.f};
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) v[q][e] = (float)ahead[q][e];
    if (r + step < rows) fetch(r + step);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) s[0] += v[q][e];
    row_sum<LPR, 1>(s, lds, slot);
    const float mean = s[0] * inv_dim;
    s[0] = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        v[q][e] -= mean;
        s[0] += (lane + LPR * q) * VE + e < dim ? v[q][e] * v[q][e] : 0.f;
      }
    row_sum<LPR, 1>(s, lds, slot);
    const float rstd = 1.f / sqrtf(s[0] * inv_dim + eps);
    if (lane == 0 && save_mean) {
      save_mean[r] = mean;
      save_rstd[r] = rstd;
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float o = fmaf(v[q][e] * rstd, w[q][e], b[q][e]);
        v[q][e] = relu && o < 0.f ? 0.f : o;  // a NaN stays one
      }
      const int c = (lane + LPR * q) * VE;
      if (c < dim) store_cols<T, VE>(y + r * ldy, c, dim, v[q]);
    }
  }
}

template <typename T, typename W, int LPR, int NV>
__global__ void __launch_bounds__(kBlock) k_layer_norm_bwd(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                           const W* __restrict__ gamma, const W* __restrict__ beta,
                                                           const float* __restrict__ save_mean, const float* __restrict__ save_rstd, int relu,
                                                           T* __restrict__ dx, int64_t lddx, float* __restrict__ partial /*[grid][2][dim]*/,
                                                           int64_t rows, int dim) {
  constexpr int VE = Pack<T>::n, G = kBlock / LPR;
  __shared__ float lds[LPR > 64 ? 4 * kBlock / 64 : kBlock / 64 * LPR * NV * VE];
  int slot = 0;
  const int lane = threadIdx.x % LPR;
  const float inv_dim = 1.f / (float)dim;
  float w[NV][VE], dw[NV][VE], db[NV][VE];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    load_gain<W, VE>(gamma, (lane + LPR * q) * VE, dim, 1.f, w[q]);
#pragma unroll
    for (int e = 0; e < VE; ++e) dw[q][e] = db[q][e] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / LPR;
  // the next row is on its way while this one is summed: a row's round trip through its sums is longer than its memory latency
  typename Pack<T>::type px[NV], pg[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](int64_t row) {
    next_mean = save_mean[row];
    next_rstd = save_rstd[row];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      px[q] = load_pack<T>(x + row * ldx, (lane + LPR * q) * VE, dim);
      pg[q] = load_pack<T>(dy + row * lddy, (lane + LPR * q) * VE, dim);
    }
  };
  if (r < rows) fetch(r);
  for (; r < rows; r += step) {
    float v[NV][VE], g[NV][VE];
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        v[q][e] = (float)px[q][e];
        g[q][e] = (float)pg[q][e];
      }
    const float mean = next_mean, rstd = next_rstd;
    if (r + step < rows) fetch(r + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float b[VE];
      if (relu) load_gain<W, VE>(beta, (lane + LPR * q) * VE, dim, 0.f, b);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        v[q][e] = (v[q][e] - mean) * rstd;                                // beyond dim: finite or not, its g is zero -- see below
        if (relu && fmaf(v[q][e], w[q][e], b[e]) <= 0.f) g[q][e] = 0.f;  // the forward's expression
        if ((lane + LPR * q) * VE + e >= dim) v[q][e] = 0.f;
        dw[q][e] = fmaf(g[q][e], v[q][e], dw[q][e]);
        db[q][e] += g[q][e];
        g[q][e] *= w[q][e];
        s[0] += g[q][e];
        s[1] = fmaf(g[q][e], v[q][e], s[1]);
      }
    }
    if (dx) {  // (uniform: the barrier inside row_sum is met by all or none)
      row_sum<LPR, 2>(s, lds, slot);
      const float m1 = s[0] * inv_dim, m2 = s[1] * inv_dim;
#pragma unroll
      for (int q = 0; q < NV; ++q) {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[q][e] = rstd * (g[q][e] - fmaf(v[q][e], m2, m1));
        const int c = (lane + LPR * q) * VE;
        if (c < dim) store_cols<T, VE>(dx + r * lddx, c, dim, v[q]);
      }
    }
  }
  if (!partial) return;
  float* out = partial + (size_t)blockIdx.x * 2 * dim;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float (&a)[NV][VE] = half ? db : dw;
    if constexpr (LPR <= 64) {  // lane groups of a wave by shuffles, the four waves through LDS
      if constexpr (LPR == 16) {
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            a[q][e] += __shfl_xor(a[q][e], 16);
            a[q][e] += __shfl_xor(a[q][e], 32);
          }
      }
      const int wl = threadIdx.x & 63, wv = threadIdx.x >> 6;
      constexpr int E = NV * VE;
      __syncthreads();
      if (wl < LPR) {
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int e = 0; e < VE; ++e) lds[(wv * E + q * VE + e) * LPR + wl] = a[q][e];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < E * LPR; i += kBlock) {
        const int l = i % LPR, qe = i / LPR, c = (l + LPR * (qe / VE)) * VE + qe % VE;
        if (c < dim) out[half * dim + c] = (lds[i] + lds[i + E * LPR]) + (lds[i + 2 * E * LPR] + lds[i + 3 * E * LPR]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        const int c = (lane + LPR * q) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (c + e < dim) out[half * dim + c + e] = a[q][e];
      }
    }
  }
}

// rows wider than kRegDim: one workgroup of 1024 threads per row, the row read once per sum (the later reads come from L2)
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = row16_sum(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  __syncthreads();  // the previous sum has been read
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < kWideBlock / 64; ++w) t += lds[w];
  return t;
}

template <typename T, typename W>
__global__ void __launch_bounds__(kWideBlock) k_layer_norm_fwd_wide(const T* __restrict__ x, int64_t ldx, const W* __restrict__ gamma,
                                                                    const W* __restrict__ beta, float eps, int relu, T* __restrict__ y, int64_t ldy,
                                                                    float* __restrict__ save_mean, float* __restrict__ save_rstd, int64_t rows,
                                                                    int dim) {
  __shared__ float lds[kWideBlock / 64];
  const float inv_dim = 1.f / (float)dim;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < dim; c += kWideBlock) s += (float)row[c];
    const float mean = block_sum(s, lds) * inv_dim;
    s = 0.f;
    for (int c = threadIdx.x; c < dim; c += kWideBlock) {
      const float d = (float)row[c] - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.f / sqrtf(block_sum(s, lds) * inv_dim + eps);
    if (threadIdx.x == 0 && save_mean) {
      save_mean[r] = mean;
      save_rstd[r] = rstd;
    }
    for (int c = threadIdx.x; c < dim; c += kWideBlock) {
      const float o = fmaf(((float)row[c] - mean) * rstd, gamma ? (float)gamma[c] : 1.f, beta ? (float)beta[c] : 0.f);
      y[r * ldy + c] = (T)(relu && o < 0.f ? 0.f : o);
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kWideBlock) k_layer_norm_bwd_wide(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                                    const W* __restrict__ gamma, const W* __restrict__ beta,
                                                                    const float* __restrict__ save_mean, const float* __restrict__ save_rstd,
                                                                    int relu, T* __restrict__ dx, int64_t lddx, int64_t rows, int dim) {
  __shared__ float lds[kWideBlock / 64];
  const float inv_dim = 1.f / (float)dim;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = save_mean[r], rstd = save_rstd[r];
    auto at = [&](int c, float& xh) {
      xh = ((float)x[r * ldx + c] - mean) * rstd;
      const float w = gamma ? (float)gamma[c] : 1.f;
      const float h = (float)dy[r * lddy + c];
      return relu && fmaf(xh, w, beta ? (float)beta[c] : 0.f) <= 0.f ? 0.f : h * w;
    };
    float s1 = 0.f, s2 = 0.f, xh;
    for (int c = threadIdx.x; c < dim; c += kWideBlock) {
      const float g = at(c, xh);
      s1 += g;
      s2 = fmaf(g, xh, s2);
    }
    const float m1 = block_sum(s1, lds) * inv_dim, m2 = block_sum(s2, lds) * inv_dim;
    for (int c = threadIdx.x; c < dim; c += kWideBlock) {
      const float g = at(c, xh);
      dx[r * lddx + c] = (T)(rstd * (g - fmaf(xh, m2, m1)));
    }
  }
}

// a workgroup sums the rows b, b + gridDim.y, ... for 256 columns
template <typename T, typename W>
__global__ void __launch_bounds__(kBlock) k_layer_norm_gain_wide(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                                 const W* __restrict__ gamma, const W* __restrict__ beta,
                                                                 const float* __restrict__ save_mean, const float* __restrict__ save_rstd, int relu,
                                                                 float* __restrict__ partial, int64_t rows, int dim) {
  const int c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= dim) return;
  const float w = gamma ? (float)gamma[c] : 1.f, b = beta ? (float)beta[c] : 0.f;
  float s1 = 0.f, s2 = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float xh = ((float)x[r * ldx + c] - save_mean[r]) * save_rstd[r];
    const float h = relu && fmaf(xh, w, b) <= 0.f ? 0.f : (float)dy[r * lddy + c];
    s1 = fmaf(h, xh, s1);
    s2 += h;
  }
  float* out = partial + (size_t)blockIdx.y * 2 * dim;
  out[c] = s1;
  out[dim + c] = s2;
}

// 64 columns of [dgamma | dbeta] per workgroup, 16 waves that each take every 16th partial; float64, fixed order
template <typename W>
__global__ void __launch_bounds__(1024) k_layer_norm_gain_final(const float* __restrict__ partial, int nblk, W* __restrict__ dgamma,
                                                                W* __restrict__ dbeta, int dim) {
  __shared__ double lds[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), sl = threadIdx.x >> 6;
  double a[4] = {0.0, 0.0, 0.0, 0.0};
  if (col < 2 * dim) {
    int b = sl;
    for (; b + 48 < nblk; b += 64) {
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] += (double)partial[(size_t)(b + 16 * u) * 2 * dim + col];
    }
    for (; b < nblk; b += 16) a[0] += (double)partial[(size_t)b * 2 * dim + col];
  }
  lds[sl][threadIdx.x & 63] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (sl != 0 || col >= 2 * dim) return;
  double t = 0.0;
  for (int w = 0; w < 16; ++w) t += lds[w][threadIdx.x];
  if (col < dim) {
    if (dgamma) dgamma[col] = (W)(float)t;
  } else if (dbeta) {
    dbeta[col - dim] = (W)(float)t;
  }
}

// lanes per row: the fewest that hold it with fewer than 32 values each -- with 32 the backward's registers leave one wave per SIMD
// (2048 fp32: 104 us on 64 lanes, 90 on 256; 512 bf16: 57 on 16, 48 on 64; but 448 fp32, 28 values: 98 on 16, 110 on 64; 1500 bf16, 24
// values: 55 on 64, 95 on 256; 40 M values each)
inline int lanes_per_row(int64_t dim, int per_vector) {
  const int64_t most = 31 / per_vector * per_vector;
  return dim <= 16 * most ? 16 : dim <= 64 * most ? 64 : 256;
}

// workgroups of the backward: two per CU cover HBM's latency and leave few partials; beyond 4096 columns the registers of a workgroup fill
// a CU and the partials are as large as rows, so one (4882 x 8192 fp32 118 us with 512, 111 with 256, bf16 84 and 65; 9765 x 4096 fp32 98
// and 111).  Rows of a wave or more: at least two per lane group, for the partials' sake (2048 x 1500 bf16 17.1 us with one, 14.1 with two;
// 2048 x 256 on 16 lanes 7.5 with one, 9.6 with two)
inline int64_t bwd_blocks(int64_t rows, int64_t dim) {
  const int64_t groups = dim > kRegDim ? 1 : kBlock / lanes_per_row(dim, 4);  // (of fp32 rows; 16-bit rows may have fewer)
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, groups == 16 ? groups : 2 * groups), dim > 4096 ? 256 : 512));
}

struct FwdArgs {
  const void* x; int64_t ldx; const void *gamma, *beta; float eps; int relu; void* y; int64_t ldy; float *mean, *rstd; int64_t rows; int dim;
  hipStream_t st;
};
struct BwdArgs {
  const void* dy; int64_t lddy; const void* x; int64_t ldx; const void *gamma, *beta; const float *mean, *rstd; int relu; void* dx; int64_t lddx;
  void *dgamma, *dbeta; float* partial; int64_t rows; int dim; hipStream_t st;
};

template <typename T, typename W, int LPR, int NV>
void launch_fwd(const FwdArgs& a) {
  constexpr int G = kBlock / LPR;
  const int64_t grid = std::min<int64_t>(ceil_div(a.rows, G), (int64_t)num_cu() * 8);
  hipLaunchKernelGGL((k_layer_norm_fwd<T, W, LPR, NV>), dim3((unsigned)grid), dim3(kBlock), 0, a.st, (const T*)a.x, a.ldx, (const W*)a.gamma,
                     (const W*)a.beta, a.eps, a.relu, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.dim);
}
template <typename T, typename W, int LPR, int NV>
void launch_bwd(const BwdArgs& a) {
  hipLaunchKernelGGL((k_layer_norm_bwd<T, W, LPR, NV>), dim3((unsigned)bwd_blocks(a.rows, a.dim)), dim3(kBlock), 0, a.st, (const T*)a.dy, a.lddy,
                     (const T*)a.x, a.ldx, (const W*)a.gamma, (const W*)a.beta, a.mean, a.rstd, a.relu, (T*)a.dx, a.lddx, a.partial, a.rows, a.dim);
}

template <typename T, typename W, int LPR, int MAXNV, typename Args, int NV = 1>
void by_vectors(int nv, const Args& a) {
  if constexpr (NV >= MAXNV) {
    if constexpr (std::is_same<Args, FwdArgs>::value) launch_fwd<T, W, LPR, MAXNV>(a); else launch_bwd<T, W, LPR, MAXNV>(a);
  } else {
    if (nv <= NV) {
      if constexpr (std::is_same<Args, FwdArgs>::value) launch_fwd<T, W, LPR, NV>(a); else launch_bwd<T, W, LPR, NV>(a);
    } else {
      by_vectors<T, W, LPR, MAXNV, Args, NV + 1>(nv, a);
    }
  }
}

template <typename T, typename W, typename Args>
void by_width(const Args& a) {
  constexpr int VE = Pack<T>::n, FEW = 31 / VE;  // (vectors per lane: fewer than 32 values, on 256 lanes up to kRegDim columns)
  const int lpr = lanes_per_row(a.dim, VE), nv = (int)ceil_div(a.dim, lpr * VE);
  if (lpr == 16) by_vectors<T, W, 16, FEW>(nv, a);
  else if (lpr == 64) by_vectors<T, W, 64, FEW, Args, FEW / 4 + 1>(nv, a);  // (more than 16 or 64 lanes hold with FEW)
  else by_vectors<T, W, 256, kRegDim / 256 / VE, Args, FEW / 4 + 1>(nv, a);
}

template <typename T, typename W>
void run_fwd(const FwdArgs& a) {
  if (a.dim <= kRegDim) return by_width<T, W>(a);
  const int64_t grid = std::min<int64_t>(a.rows, (int64_t)num_cu() * 2);
  hipLaunchKernelGGL((k_layer_norm_fwd_wide<T, W>), dim3((unsigned)grid), dim3(kWideBlock), 0, a.st, (const T*)a.x, a.ldx, (const W*)a.gamma,
                     (const W*)a.beta, a.eps, a.relu, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.dim);
}

template <typename T, typename W>
void run_bwd(const BwdArgs& a) {
  const int64_t nblk = a.rows ? bwd_blocks(a.rows, a.dim) : 0;
  if (a.rows && a.dim <= kRegDim) {
    by_width<T, W>(a);
  } else if (a.rows) {
    const int64_t grid = std::min<int64_t>(a.rows, (int64_t)num_cu() * 2);
    if (a.dx)
      hipLaunchKernelGGL((k_layer_norm_bwd_wide<T, W>), dim3((unsigned)grid), dim3(kWideBlock), 0, a.st, (const T*)a.dy, a.lddy, (const T*)a.x, a.ldx,
                         (const W*)a.gamma, (const W*)a.beta, a.mean, a.rstd, a.relu, (T*)a.dx, a.lddx, a.rows, a.dim);
    if (a.partial)
      hipLaunchKernelGGL((k_layer_norm_gain_wide<T, W>), dim3((unsigned)ceil_div(a.dim, kBlock), (unsigned)nblk), dim3(kBlock), 0, a.st,
                         (const T*)a.dy, a.lddy, (const T*)a.x, a.ldx, (const W*)a.gamma, (const W*)a.beta, a.mean, a.rstd, a.relu, a.partial,
                         a.rows, a.dim);
  }
  if (a.partial)
    hipLaunchKernelGGL((k_layer_norm_gain_final<W>), dim3((unsigned)ceil_div(2 * (int64_t)a.dim, 64)), dim3(1024), 0, a.st, a.partial, (int)nblk,
                       (W*)a.dgamma, (W*)a.dbeta, a.dim);
}

inline bool known_types(int x_type, int w_type) {
  return (x_type == PGNN_F32 && w_type == PGNN_F32) ||
         ((x_type == PGNN_BF16 || x_type == PGNN_F16) && (w_type == PGNN_F32 || w_type == x_type));
}

template <typename Args>
void by_type(int x_type, int w_type, const Args& a) {
  auto go = [&](auto t, auto w) {
    if constexpr (std::is_same<Args, FwdArgs>::value) run_fwd<decltype(t), decltype(w)>(a); else run_bwd<decltype(t), decltype(w)>(a);
  };
  if (x_type == PGNN_F32) go(float{}, float{});
  else if (x_type == PGNN_BF16 && w_type == PGNN_F32) go(__bf16{}, float{});
  else if (x_type == PGNN_BF16) go(__bf16{}, __bf16{});
  else if (w_type == PGNN_F32) go(_Float16{}, float{});
  else go(_Float16{}, _Float16{});
}

}  // namespace

extern "C" {

int pgnn_layer_norm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, float eps, int relu, void* y, int64_t ldy,
                        float* save_mean, float* save_rstd, int64_t rows, int64_t dim, int x_type, int w_type, pgnn_stream stream) {
  PGNN_REQUIRE(known_types(x_type, w_type), "layer_norm_fwd: rows of type %d with gains of type %d", x_type, w_type);
  PGNN_REQUIRE(rows >= 0 && dim > 0 && dim < (1ll << 30), "layer_norm_fwd: bad shape [%lld, %lld]", (long long)rows, (long long)dim);
  if (rows == 0) return PGNN_OK;
  PGNN_REQUIRE(x && y && ldx >= 0 && ldy >= dim, "layer_norm_fwd: bad pointer or leading dimension");
  PGNN_REQUIRE(!save_mean == !save_rstd, "layer_norm_fwd: save_mean and save_rstd are kept together");
  by_type(x_type, w_type, FwdArgs{x, ldx, gamma, beta, eps, relu, y, ldy, save_mean, save_rstd, rows, (int)dim, (hipStream_t)stream});
  return check_launch("layer_norm_fwd");
}

size_t pgnn_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 0 || dim <= 0) return 0;
  return (size_t)bwd_blocks(rows, dim) * 2 * (size_t)dim * sizeof(float);
}

int pgnn_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* gamma, const void* beta, const float* save_mean,
                        const float* save_rstd, int relu, void* dx, int64_t lddx, void* dgamma, void* dbeta, int64_t rows, int64_t dim,
                        int x_type, int w_type, void* ws, size_t ws_bytes, pgnn_stream stream) {
  PGNN_REQUIRE(known_types(x_type, w_type), "layer_norm_bwd: rows of type %d with gains of type %d", x_type, w_type);
  PGNN_REQUIRE(rows >= 0 && dim > 0 && dim < (1ll << 30), "layer_norm_bwd: bad shape [%lld, %lld]", (long long)rows, (long long)dim);
  const bool gains = dgamma || dbeta;
  if (!gains && (!dx || rows == 0)) return PGNN_OK;
  PGNN_REQUIRE(rows == 0 || (dy && x && save_mean && save_rstd && lddy >= 0 && ldx >= 0 && (!dx || lddx >= dim)),
               "layer_norm_bwd: bad pointer or leading dimension");
  if (gains && (!ws || ws_bytes < pgnn_layer_norm_bwd_workspace_bytes(rows, dim))) {
    set_error("layer_norm_bwd: workspace too small");
    return PGNN_ERR_WORKSPACE;
  }
  by_type(x_type, w_type, BwdArgs{dy, lddy, x, ldx, gamma, beta, save_mean, save_rstd, relu, rows ? dx : nullptr, lddx, dgamma, dbeta,
                                  gains ? (float*)ws : nullptr, rows, (int)dim, (hipStream_t)stream});
  return check_launch("layer_norm_bwd");
}

}  // extern "C"
