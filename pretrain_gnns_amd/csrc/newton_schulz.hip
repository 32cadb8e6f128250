// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step that is built on it:
//   X_0 = G / (|G|_F + eps), transposed if it has more rows than columns (X is k x n, k <= n), then per step
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
// which drives the singular values of X towards 1 and leaves its singular vectors alone.  Muon orthogonalises the momentum:
//   M <- mu M + G,  U = G + mu M (nesterov) or M,  p <- p (1 - lr wd) - rate orthogonal(U)
//
// Everything after the first read of G lives as TWO fp16 planes h + l of s X, s a power of two (two_plane.h): three
// v_mfma_f32_16x16x32_f16 per block (h l, l h, h h) with fp32 accumulation give the error of an fp32 product at 3/16 of the
// matrix-core time of v_mfma_f32_16x16x4_f32, and two planes take the bytes of one fp32 matrix.  The iteration bounds its own
// entries -- |X_ij| <= |X|_2 <= u_t, with u_0 = |G|_F / (|G|_F + eps) and u_{t+1} the maximum of |a x + b x^3 + c x^5| on [0, u_t] --
// so ONE scale per matrix and step is known before a product runs: no row maxima, and no fp16 overflow for any input.
// Both X and X^T are kept, so that all three products contract along rows of both operands (the fragments of an MFMA are 16-byte
// pieces of rows): the epilogue turns its tile through LDS and writes it both ways.  A and B are symmetric: only the tiles on and
// above the diagonal are computed, and written twice.  a X is added behind the product B X, in fp32: as a I inside B it would stand in
// the middle of each long sum and cost the small terms their last bits (4096 x 4096: 6.5e-6 of the 64-bit result instead of 3e-6).
// All matrices of a call share each launch: 2 + 3 steps launches whatever their number.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "two_plane.h"

using namespace pgnn;

namespace {

constexpr int kMaxJobs = 48;         // matrices per launch (the job table travels in the kernel arguments: 3.4 KB at most)
constexpr int kMaxSteps = 32;
constexpr int kMaxParts = 256;       // partial sums of squares per matrix
constexpr int64_t kNormPart = 4096;  // elements per partial sum, at least
constexpr int64_t kChunkBytes = 2ll << 30;  // a call's matrices are taken in chunks of at most this much workspace
constexpr int kBK = 32;              // contraction per stage: one MFMA
constexpr int kPad = 64;             // leading dimensions of the planes are multiples of this, zero beyond the matrix

enum { kGram, kPoly, kApply, kLast };

// where a matrix's planes are in its part of the workspace (bytes): the exponents and the partial sums in front, at fixed places; planes
// of 64 k columns are multiples of 256 bytes by themselves
constexpr int64_t kExps = 0, kParts = 512, kPlanes = kParts + kMaxParts * 8;
static_assert(3 * (kMaxSteps + 1) * 4 <= kParts && kPlanes % 256 == 0, "");
struct Layout {
  int64_t ldk, ldn, x, xt0, xt1, a, b, bytes;
};
__host__ __device__ inline Layout layout_of(int64_t k, int64_t n) {
  Layout l;
  l.ldk = (k + kPad - 1) & ~(int64_t)(kPad - 1);
  l.ldn = (n + kPad - 1) & ~(int64_t)(kPad - 1);
  l.x = kPlanes;
  l.xt0 = l.x + 4 * k * l.ldn;
  l.xt1 = l.xt0 + 4 * n * l.ldk;
  l.a = l.xt1 + 4 * n * l.ldk;
  l.b = l.a + 4 * k * l.ldk;
  l.bytes = l.b + 4 * k * l.ldk;
  return l;
}

struct Jobs {
  int count;
  int first[kMaxJobs + 1];  // first workgroup of a job
  int rows[kMaxJobs], cols[kMaxJobs];
  int64_t off[kMaxJobs];    // its part of the workspace
  const void* src[kMaxJobs];  // G
  int64_t ld[kMaxJobs];
  void* dst[kMaxJobs];      // the result, or the parameter
  char* ws;
};
struct MuonArgs {
  float* momentum[kMaxJobs];
  float rate[kMaxJobs];
  float mu, keep;           // keep = 1 - lr wd
  int nesterov;
};
struct NoMuon { int unused; };  // (not empty: an empty kernel argument is dropped on the device side only)
template <bool MUON> using Muon = typename std::conditional<MUON, MuonArgs, NoMuon>::type;
struct Bounds {             // of the iteration on [0, 1]: max |p| after t steps, max |b x^2 + c x^4| in step t
  float coef[kMaxSteps][3];
  float cap_x[kMaxSteps + 1], cap_b[kMaxSteps];
  int steps;
  float eps;
};

__device__ __forceinline__ int find_job(const int* first, int count, int b) {
  int j = 0, hi = count;
  while (hi - j > 1) {
    const int mid = (j + hi) >> 1;
    if (first[mid] <= b) j = mid; else hi = mid;
  }
  return j;
}

// partial sums of squares in float64 (millions of terms, squares of gradients far below 1); Muon: the momentum is advanced here
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_norm(Jobs jobs, Muon<MUON> mu) {
  const int j = find_job(jobs.first, jobs.count, blockIdx.x);
  const int part = blockIdx.x - jobs.first[j], nparts = jobs.first[j + 1] - jobs.first[j];
  const int64_t rows = jobs.rows[j], cols = jobs.cols[j];
  double s = 0.0;
  const int64_t stride = (int64_t)nparts * 256;
  for (int64_t e = (int64_t)part * 256 + threadIdx.x; e < rows * cols; e += stride) {
    const int64_t r = e / cols, c = e - r * cols;
    float v = (float)static_cast<const T*>(jobs.src[j])[r * jobs.ld[j] + c];
    if constexpr (MUON) {
      const float m = fmaf(mu.mu, mu.momentum[j][e], v);
      mu.momentum[j][e] = m;
      v = mu.nesterov ? fmaf(mu.mu, m, v) : m;
    }
    s += (double)v * (double)v;
  }
  __shared__ double lds[4];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    reinterpret_cast<double*>(jobs.ws + jobs.off[j] + kParts)[part] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
}

// exponent e with bound * 2^e <= 2^13 (entries then stay a factor of 8 below fp16's largest value)
__device__ __forceinline__ int plane_exponent(float bound) { return 12 - ilogbf(bound); }

// X_0 as planes, both ways round, and the exponents of all planes to come
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_split(Jobs jobs, Muon<MUON> mu, Bounds bd) {
  const int j = find_job(jobs.first, jobs.count, blockIdx.x);
  const int64_t rows = jobs.rows[j], cols = jobs.cols[j];
  const bool tall = rows > cols;
  const Layout l = layout_of(min(rows, cols), max(rows, cols));
  char* base = jobs.ws + jobs.off[j];
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int nparts = (int)min((int64_t)kMaxParts, (rows * cols + kNormPart - 1) / kNormPart);
  double s = (int)threadIdx.x < nparts ? reinterpret_cast<const double*>(base + kParts)[threadIdx.x] : 0.0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const float inv = (float)(1.0 / (norm + (double)bd.eps));
  float u = (float)(norm / (norm + (double)bd.eps)) * 1.001f;
  if (!(u >= 0x1p-60f)) u = 0x1p-60f;  // (also a NaN: everything becomes NaN whatever the scale)
  if (!(u <= bd.cap_x[0])) u = bd.cap_x[0];
  const int e0 = plane_exponent(u);
  const int local = blockIdx.x - jobs.first[j];
  if (local == 0 && threadIdx.x == 0) {
    int* e = reinterpret_cast<int*>(base + kExps);
    e[0] = e0;
    for (int t = 0; t < bd.steps; ++t) {
      const float a = fabsf(bd.coef[t][0]), b = fabsf(bd.coef[t][1]), c = fabsf(bd.coef[t][2]);
      const float al = fmaxf(1.001f * u * u, 0x1p-60f);
      e[kMaxSteps + 1 + t] = plane_exponent(al);                                                       // A
      const float be = fmaxf(fminf(1.001f * al * (b + al * c), bd.cap_b[t]), 0x1p-60f);
      e[2 * (kMaxSteps + 1) + t] = plane_exponent(be);                                                 // B
      u = fmaxf(fminf((a + be) * u, bd.cap_x[t + 1]), 0x1p-60f);
      e[t + 1] = plane_exponent(u);                                                                    // X
    }
  }
  const int tc = (int)((cols + 63) / 64), r0 = local / tc * 64, c0 = local % tc * 64;
  const float scale = ldexpf(1.f, e0);
  for (int q = threadIdx.x; q < 4096; q += 256) {
    const int r = q >> 6, c = q & 63;
    float v = 0.f;
    if (r0 + r < rows && c0 + c < cols) {
      v = (float)static_cast<const T*>(jobs.src[j])[(r0 + r) * jobs.ld[j] + c0 + c];
      if constexpr (MUON) {  // the direction, from the momentum that k_ns_norm has advanced
        const float m = mu.momentum[j][(r0 + r) * cols + c0 + c];
        v = mu.nesterov ? fmaf(mu.mu, m, v) : m;
      }
      v = v * inv * scale;
    }
    tile[r][c] = v;
  }
  __syncthreads();
  _Float16* as_is = reinterpret_cast<_Float16*>(base + (tall ? l.xt0 : l.x));
  _Float16* turned = reinterpret_cast<_Float16*>(base + (tall ? l.x : l.xt0));
  const int64_t ld_is = tall ? l.ldk : l.ldn, ld_tu = tall ? l.ldn : l.ldk;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    _Float16* d = half ? turned : as_is;
    const int64_t ld = half ? ld_tu : ld_is, dr0 = half ? c0 : r0, dc0 = half ? r0 : c0, drows = half ? cols : rows;
    for (int q = threadIdx.x; q < 64 * 32; q += 256) {
      const int r = q >> 5, c = (q & 31) * 2;
      if (dr0 + r >= drows) continue;
      uint32_t h, lo;
      split2(half ? tile[c][r] : tile[r][c], half ? tile[c + 1][r] : tile[r][c + 1], h, lo);
      *reinterpret_cast<uint32_t*>(d + (dr0 + r) * ld + dc0 + c) = h;
      *reinterpret_cast<uint32_t*>(d + (drows + dr0 + r) * ld + dc0 + c) = lo;
    }
  }
}

template <typename T> struct Out8 { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };

__device__ __forceinline__ void split8(const float (&v)[8], f16x8& h, f16x8& l) {
  uint32_t hh[4], ll[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) split2(v[2 * q], v[2 * q + 1], hh[q], ll[q]);
  h = __builtin_bit_cast(f16x8, make_uint4(hh[0], hh[1], hh[2], hh[3]));
  l = __builtin_bit_cast(f16x8, make_uint4(ll[0], ll[1], ll[2], ll[3]));
}

// One TT x TT tile of C = P Q^T, P and Q on planes.  Four waves of TT/2 x TT/2; wave w fetches operand array w (P high, P low, Q high,
// Q low) by LDS DMA, STAGES - 1 stages ahead.  A stage holds 32 columns: 64 bytes per row, whose four 16-byte pieces are permuted by
// (row >> 1) & 3, so that the eight rows one LDS cycle reads of a piece lie in eight different bank groups.
template <int TT, int STAGES, int PHASE, typename TO, bool MUON>
__global__ void __launch_bounds__(256) k_ns_product(Jobs jobs, Muon<MUON> mu, int step, float ca, float cb, float cc) {
  constexpr int MI = TT / 32, ARR = TT * kBK * 2, STAGE = 4 * ARR, NJ = TT / 16;
  constexpr int LDT = TT + 4;  // floats per row of the epilogue's tile: 16-byte rows, neighbours four banks apart
  extern __shared__ __align__(16) char smem[];
  const int j = find_job(jobs.first, jobs.count, blockIdx.x);
  const int rows = jobs.rows[j], cols = jobs.cols[j], k = min(rows, cols), n = max(rows, cols);
  const Layout l = layout_of(k, n);
  char* base = jobs.ws + jobs.off[j];
  int ti, tj;
  {
    const int local = blockIdx.x - jobs.first[j];
    if constexpr (PHASE <= kPoly) {  // tile pairs ti <= tj, column by column
      tj = (int)((sqrtf(8.f * (float)local + 1.f) - 1.f) * 0.5f);
      while (tj * (tj + 1) / 2 > local) --tj;
      while ((tj + 1) * (tj + 2) / 2 <= local) ++tj;
      ti = local - tj * (tj + 1) / 2;
    } else {
      const int across = (k + TT - 1) / TT;
      ti = local % across;
      tj = local / across;
    }
  }
  const int* exps = reinterpret_cast<const int*>(base + kExps);
  const int eX = exps[step], eA = exps[kMaxSteps + 1 + step], eB = exps[2 * (kMaxSteps + 1) + step], eY = exps[step + 1];
  const int64_t xt_in = step & 1 ? l.xt1 : l.xt0, xt_out = step & 1 ? l.xt0 : l.xt1;
  // operands: rows, leading dimension, planes
  const _Float16 *P, *Q;
  int prow, qrow, ldp, kk;
  if constexpr (PHASE == kGram) {
    P = Q = reinterpret_cast<const _Float16*>(base + l.x);
    prow = qrow = k;
    ldp = kk = (int)l.ldn;
  } else if constexpr (PHASE == kPoly) {
    P = Q = reinterpret_cast<const _Float16*>(base + l.a);
    prow = qrow = k;
    ldp = kk = (int)l.ldk;
  } else {
    P = reinterpret_cast<const _Float16*>(base + l.b);
    Q = reinterpret_cast<const _Float16*>(base + xt_in);
    prow = k;
    qrow = n;
    ldp = kk = (int)l.ldk;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i0 = ti * TT, j0 = tj * TT;

  // the wave's DMA pieces: 16 rows of 64 bytes each
  const _Float16* src = (wave < 2 ? P + (int64_t)(wave & 1) * prow * ldp : Q + (int64_t)(wave & 1) * qrow * ldp);
  uint32_t offs[NJ];  // in halfs; rows beyond the matrix re-read its last one (their results are not stored)
#pragma unroll
  for (int q = 0; q < NJ; ++q) {
    const int r = q * 16 + (lane >> 2);
    const int row = min((wave < 2 ? i0 : j0) + r, (wave < 2 ? prow : qrow) - 1);
    offs[q] = (uint32_t)row * (uint32_t)ldp + (uint32_t)(((lane & 3) ^ ((r >> 1) & 3)) * 8);
  }
  auto issue = [&](int t) {
    char* dst = smem + (t % STAGES) * STAGE + wave * ARR;
#pragma unroll
    for (int q = 0; q < NJ; ++q)
      __builtin_amdgcn_global_load_lds(PGNN_GPTR(src + (size_t)offs[q] + (size_t)t * kBK), PGNN_LPTR(dst + q * 1024), 16, 0, 0);
  };
  const int wi = (wave >> 1) * (TT / 2), wj = (wave & 1) * (TT / 2);
  const int fr = lane & 15, fc = lane >> 4;
  auto frag = [&](const char* arr, int row) {
    return *reinterpret_cast<const f16x8*>(arr + row * 64 + ((fc ^ ((row >> 1) & 3)) * 16));
  };

  f32x4 acc[MI][MI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nk = kk / kBK;
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t)
    if (t < nk) issue(t);
  for (int t = 0; t < nk; ++t) {
    // stage t has landed; behind the barrier every wave's part of it has, and every wave is done with the buffer refilled below
    if (t + STAGES - 2 < nk) gemm_wait_vmcnt_imm<(STAGES - 2) * NJ>();
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + STAGES - 1 < nk) issue(t + STAGES - 1);
    const char* st = smem + (t % STAGES) * STAGE;
    f16x8 ph[MI], pl[MI], qh[MI], ql[MI];
#pragma unroll
    for (int a = 0; a < MI; ++a) {
      ph[a] = frag(st, wi + a * 16 + fr);
      pl[a] = frag(st + ARR, wi + a * 16 + fr);
      qh[a] = frag(st + 2 * ARR, wj + a * 16 + fr);
      ql[a] = frag(st + 3 * ARR, wj + a * 16 + fr);
    }
#pragma unroll
    for (int b = 0; b < MI; ++b) {  // smallest terms first
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], ql[b], acc[a][b], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a], qh[b], acc[a][b], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], qh[b], acc[a][b], 0, 0, 0);
    }
    asm volatile("" ::: "memory");
  }

  // epilogue: the tile to LDS as fp32 [j][i] (a lane holds four consecutive i of one j), then out row by row, both ways
  __syncthreads();
  float* tile = reinterpret_cast<float*>(smem);
  const float f = PHASE == kGram ? ldexpf(1.f, eA - 2 * eX) : PHASE == kPoly ? ldexpf(cc, -2 * eA)
                : PHASE == kApply ? ldexpf(1.f, eY - eX - eB) : ldexpf(1.f, -eX - eB);
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b)
      *reinterpret_cast<f32x4*>(tile + (wj + b * 16 + fr) * LDT + wi + a * 16 + fc * 4) = acc[a][b] * f;
  __syncthreads();
  constexpr int PIECES = TT / 8;
  const bool tall = rows > cols;
#pragma unroll
  for (int turned = 0; turned < 2; ++turned) {
    // turned = 0: rows j of the transpose, columns i; turned = 1: rows i, columns j
    if constexpr (PHASE == kLast) {
      if (tall == (turned == 1)) continue;  // G's own orientation only
    }
    if (PHASE <= kPoly && turned == 1 && ti == tj) continue;  // a diagonal tile is its own mirror image
    const int r0 = turned ? i0 : j0, c0 = turned ? j0 : i0;
    const int nr = PHASE <= kPoly ? k : turned ? k : n, nc = PHASE <= kPoly ? k : turned ? n : k;
    const int ld = PHASE <= kPoly || !turned ? (int)l.ldk : (int)l.ldn;
    for (int q = threadIdx.x; q < TT * PIECES; q += 256) {
      const int r = q / PIECES, c = (q % PIECES) * 8;
      if (r0 + r >= nr || c0 + c >= ld) continue;
      float v[8];
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[(c + e) * LDT + r];
      } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + r * LDT + c), hi = *reinterpret_cast<const f32x4*>(tile + r * LDT + c + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
      }
      const int64_t at = (int64_t)(r0 + r) * ld + c0 + c;
      if constexpr (PHASE >= kApply) {  // + a X, from X or X^T in this orientation (X is overwritten below by the thread that reads it)
        const _Float16* X = reinterpret_cast<const _Float16*>(base + (turned ? l.x : xt_in));
        const f16x8 h = *reinterpret_cast<const f16x8*>(X + at), lo = *reinterpret_cast<const f16x8*>(X + (int64_t)nr * ld + at);
        const float fa = ldexpf(ca, PHASE == kApply ? eY - eX : -eX);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(fa, (float)h[e] + (float)lo[e], v[e]);
      }
      if constexpr (PHASE == kPoly) {  // + b A, then to B's scale
        const _Float16* A = reinterpret_cast<const _Float16*>(base + l.a);
        const f16x8 h = *reinterpret_cast<const f16x8*>(A + at), lo = *reinterpret_cast<const f16x8*>(A + (int64_t)k * ld + at);
        const float fa = ldexpf(cb, -eA), fs = ldexpf(1.f, eB);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = fmaf(fa, (float)h[e] + (float)lo[e], v[e]);
          v[e] *= fs;
        }
      }
      if constexpr (PHASE != kLast) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + c + e < nc ? v[e] : 0.f;  // the padding that the next product contracts over
        _Float16* d = reinterpret_cast<_Float16*>(base + (PHASE == kGram ? l.a : PHASE == kPoly ? l.b : turned ? l.x : xt_out));
        f16x8 h, lo;
        split8(v, h, lo);
        *reinterpret_cast<f16x8*>(d + at) = h;
        *reinterpret_cast<f16x8*>(d + (int64_t)nr * ld + at) = lo;
      } else {
        TO* d = static_cast<TO*>(jobs.dst[j]) + (int64_t)(r0 + r) * cols + c0 + c;
        const int m = min(8, nc - (c0 + c));
        if (m == 8) {
          typename Out8<TO>::type o;
          if constexpr (MUON) o = *reinterpret_cast<typename Out8<TO>::type*>(d);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (MUON) o[e] = fmaf(-mu.rate[j], v[e], o[e] * mu.keep);
            else o[e] = (TO)v[e];
          }
          *reinterpret_cast<typename Out8<TO>::type*>(d) = o;
        } else {
          for (int e = 0; e < m; ++e) {
            if constexpr (MUON) d[e] = fmaf(-mu.rate[j], v[e], d[e] * mu.keep);
            else d[e] = (TO)v[e];
          }
        }
      }
    }
  }
}

// max over x in [0, u] of |a x^p + b x^(p+2) + c x^(p+4)| for p = 1 and 0, by its stationary points
double odd_max(double a, double b, double c, double u) {
  double m = std::fabs(u * (a + u * u * (b + u * u * c)));
  const double A = 5 * c, B = 3 * b, C = a;  // a + 3 b y + 5 c y^2 = 0, y = x^2
  double ys[2];
  int cnt = 0;
  if (A != 0) {
    const double D = B * B - 4 * A * C;
    if (D >= 0) { ys[cnt++] = (-B + std::sqrt(D)) / (2 * A); ys[cnt++] = (-B - std::sqrt(D)) / (2 * A); }
  } else if (B != 0) {
    ys[cnt++] = -C / B;
  }
  for (int q = 0; q < cnt; ++q)
    if (ys[q] > 0 && ys[q] < u * u) m = std::max(m, std::fabs(std::sqrt(ys[q]) * (a + ys[q] * (b + ys[q] * c))));
  return m;
}
double even_max(double a, double b, double c, double u) {
  const double y = u * u;
  double m = std::max(std::fabs(a), std::fabs(a + y * (b + y * c)));
  if (c != 0) {
    const double s = -b / (2 * c);
    if (s > 0 && s < y) m = std::max(m, std::fabs(a + s * (b + s * c)));
  }
  return m;
}

// 0 if the coefficients are finite and keep the iteration's spectral norm below 2^20
int make_bounds(Bounds& bd, const float* coef, int steps, float eps) {
  bd.steps = steps;
  bd.eps = eps;
  double u = 1.002;
  bd.cap_x[0] = (float)u;
  for (int t = 0; t < steps; ++t) {
    for (int q = 0; q < 3; ++q) {
      if (!std::isfinite(coef[3 * t + q])) return 1;
      bd.coef[t][q] = coef[3 * t + q];
    }
    bd.cap_b[t] = (float)(1.002 * even_max(0.0, coef[3 * t + 1], coef[3 * t + 2], u) + 1e-6);
    u = 1.002 * odd_max(coef[3 * t], coef[3 * t + 1], coef[3 * t + 2], u) + 1e-6;  // (rounding: far below the margin of 2^3 to fp16's range)
    if (!(u < 1048576.0)) return 1;
    bd.cap_x[t + 1] = (float)u;
  }
  return 0;
}

template <int TT>
int tiles_of(int k, int n, bool symmetric) {
  const int64_t a = ceil_div(k, TT), b = ceil_div(n, TT);
  return (int)(symmetric ? a * (a + 1) / 2 : a * b);
}

template <int TT, int STAGES, int PHASE, typename TO, bool MUON>
void launch_product(Jobs& jobs, const Muon<MUON>& mu, int step, const float* c, hipStream_t st) {
  int blocks = 0;
  for (int j = 0; j < jobs.count; ++j) {
    jobs.first[j] = blocks;
    blocks += tiles_of<TT>(std::min(jobs.rows[j], jobs.cols[j]), std::max(jobs.rows[j], jobs.cols[j]), PHASE <= kPoly);
  }
  jobs.first[jobs.count] = blocks;
  constexpr size_t lds = std::max<size_t>((size_t)STAGES * 4 * TT * kBK * 2, (size_t)TT * (TT + 4) * 4);
  const void* fn = (const void*)k_ns_product<TT, STAGES, PHASE, TO, MUON>;
  allow_big_lds(fn, lds);
  hipLaunchKernelGGL((k_ns_product<TT, STAGES, PHASE, TO, MUON>), dim3(blocks), dim3(256), lds, st, jobs, mu, step, c[0], c[1], c[2]);
}

template <int TT, int STAGES, typename TO, bool MUON>
void run_steps(Jobs& jobs, const Muon<MUON>& mu, const Bounds& bd, hipStream_t st) {
  for (int t = 0; t < bd.steps; ++t) {
    launch_product<TT, STAGES, kGram, float, false>(jobs, NoMuon{0}, t, bd.coef[t], st);
    launch_product<TT, STAGES, kPoly, float, false>(jobs, NoMuon{0}, t, bd.coef[t], st);
    if (t + 1 < bd.steps) launch_product<TT, STAGES, kApply, float, false>(jobs, NoMuon{0}, t, bd.coef[t], st);
    else launch_product<TT, STAGES, kLast, TO, MUON>(jobs, mu, t, bd.coef[t], st);
  }
}

template <typename T, bool MUON>
void run_chunk(Jobs& jobs, const Muon<MUON>& mu, const Bounds& bd, hipStream_t st) {
  int blocks = 0;
  for (int j = 0; j < jobs.count; ++j) {
    jobs.first[j] = blocks;
    blocks += (int)std::min<int64_t>(kMaxParts, ceil_div((int64_t)jobs.rows[j] * jobs.cols[j], kNormPart));
  }
  jobs.first[jobs.count] = blocks;
  hipLaunchKernelGGL((k_ns_norm<T, MUON>), dim3(blocks), dim3(256), 0, st, jobs, mu);
  blocks = 0;
  int64_t big = 0;
  for (int j = 0; j < jobs.count; ++j) {
    jobs.first[j] = blocks;
    blocks += (int)(ceil_div(jobs.rows[j], 64) * ceil_div(jobs.cols[j], 64));
    big += tiles_of<128>(std::min(jobs.rows[j], jobs.cols[j]), std::max(jobs.rows[j], jobs.cols[j]), true);
  }
  jobs.first[jobs.count] = blocks;
  hipLaunchKernelGGL((k_ns_split<T, MUON>), dim3(blocks), dim3(256), 0, st, jobs, mu, bd);
  if (big >= num_cu()) run_steps<128, 2, T, MUON>(jobs, mu, bd, st);
  else run_steps<64, 4, T, MUON>(jobs, mu, bd, st);
}

// the matrices [from, to) of a chunk: at most kMaxJobs, and kChunkBytes unless one alone takes more
int64_t chunk_end(const int64_t* rows, const int64_t* cols, int64_t from, int64_t count, size_t& bytes) {
  bytes = 0;
  int64_t j = from;
  for (; j < count && j - from < kMaxJobs; ++j) {
    const size_t b = rows[j] > 0 && cols[j] > 0 ? (size_t)layout_of(std::min(rows[j], cols[j]), std::max(rows[j], cols[j])).bytes : 0;
    if (j > from && bytes + b > (size_t)kChunkBytes) break;
    bytes += b;
  }
  return j;
}

int check_shapes(const char* what, const int64_t* rows, const int64_t* cols, int64_t count) {
  PGNN_REQUIRE(count >= 0 && (count == 0 || (rows && cols)), "%s: bad list of matrices", what);
  for (int64_t j = 0; j < count; ++j)  // 32-bit offsets inside a plane
    PGNN_REQUIRE(rows[j] >= 0 && cols[j] >= 0 && rows[j] <= 32768 && cols[j] <= 32768, "%s: matrix %lld is %lld x %lld (0 to 32768 each way)", what,
                 (long long)j, (long long)rows[j], (long long)cols[j]);
  return PGNN_OK;
}

template <typename Fill>
int run_all(const char* what, const int64_t* rows, const int64_t* cols, int64_t count, const float* coef, int steps, float eps, void* ws,
            size_t ws_bytes, Fill fill) {
  if (int rc = check_shapes(what, rows, cols, count)) return rc;
  PGNN_REQUIRE(coef && steps >= 1 && steps <= kMaxSteps, "%s: 1 to %d steps", what, kMaxSteps);
  PGNN_REQUIRE(eps >= 0.f && std::isfinite(eps), "%s: bad eps", what);
  Bounds bd;
  PGNN_REQUIRE(make_bounds(bd, coef, steps, eps) == 0, "%s: with these coefficients the iteration leaves every bound", what);
  size_t most = 0;  // everything is checked before the first launch
  for (int64_t from = 0; from < count;) {
    size_t need;
    from = chunk_end(rows, cols, from, count, need);
    most = std::max(most, need);
  }
  if (most && (!ws || ws_bytes < most)) {
    set_error("%s: workspace too small", what);
    return PGNN_ERR_WORKSPACE;
  }
  for (int64_t j = 0; j < count; ++j)
    PGNN_REQUIRE(rows[j] == 0 || cols[j] == 0 || fill.valid(j), "%s: bad pointer or leading dimension of matrix %lld", what, (long long)j);
  bool launched = false;
  for (int64_t from = 0; from < count;) {
    size_t need;
    const int64_t to = chunk_end(rows, cols, from, count, need);
    Jobs jobs{};
    MuonArgs mu{};
    jobs.ws = (char*)ws;
    int64_t off = 0;
    for (int64_t j = from; j < to; ++j) {
      if (rows[j] == 0 || cols[j] == 0) continue;
      const int q = jobs.count++;
      jobs.rows[q] = (int)rows[j];
      jobs.cols[q] = (int)cols[j];
      jobs.off[q] = off;
      off += layout_of(std::min(rows[j], cols[j]), std::max(rows[j], cols[j])).bytes;
      fill.set(jobs, mu, q, j);
    }
    if (jobs.count) fill.run(jobs, mu, bd);
    launched |= jobs.count > 0;
    from = to;
  }
  return launched ? check_launch(what) : PGNN_OK;
}

struct FillPlain {
  const void* const* src; const int64_t* ld; void* const* dst; const int64_t* cols; int type; hipStream_t st;
  bool valid(int64_t j) const { return src[j] && dst[j] && ld[j] >= 0; }
  void set(Jobs& jobs, MuonArgs&, int q, int64_t j) const {
    jobs.src[q] = src[j];
    jobs.dst[q] = dst[j];
    jobs.ld[q] = ld[j];
  }
  void run(Jobs& jobs, const MuonArgs&, const Bounds& bd) const {
    if (type == PGNN_F32) run_chunk<float, false>(jobs, NoMuon{0}, bd, st);
    else if (type == PGNN_BF16) run_chunk<__bf16, false>(jobs, NoMuon{0}, bd, st);
    else run_chunk<_Float16, false>(jobs, NoMuon{0}, bd, st);
  }
};
struct FillMuon {
  float* const* params; const float* const* grads; float* const* momentum; const float* rates; const int64_t* cols; float mu, keep; int nesterov;
  hipStream_t st;
  bool valid(int64_t j) const { return params[j] && grads[j] && momentum[j]; }
  void set(Jobs& jobs, MuonArgs& m, int q, int64_t j) const {
    jobs.src[q] = grads[j];
    jobs.dst[q] = params[j];
    jobs.ld[q] = cols[j];
    m.momentum[q] = momentum[j];
    m.rate[q] = rates[j];
  }
  void run(Jobs& jobs, MuonArgs& m, const Bounds& bd) const {
    m.mu = mu;
    m.keep = keep;
    m.nesterov = nesterov;
    run_chunk<float, true>(jobs, m, bd, st);
  }
};

}  // namespace

extern "C" {

size_t pgnn_newton_schulz_workspace_bytes(const int64_t* rows, const int64_t* cols, int64_t count) {
  if (check_shapes("newton_schulz_workspace_bytes", rows, cols, count)) return 0;
  size_t most = 0;
  for (int64_t from = 0; from < count;) {
    size_t b;
    from = chunk_end(rows, cols, from, count, b);
    most = std::max(most, b);
  }
  return most;
}

int pgnn_newton_schulz(const void* const* src, const int64_t* ld_src, void* const* dst, const int64_t* rows, const int64_t* cols, int64_t count,
                       int type, const float* coefficients, int steps, float eps, void* ws, size_t ws_bytes, pgnn_stream stream) {
  PGNN_REQUIRE(type == PGNN_F32 || type == PGNN_BF16 || type == PGNN_F16, "newton_schulz: type %d", type);
  PGNN_REQUIRE(count <= 0 || (src && ld_src && dst), "newton_schulz: bad list of matrices");
  return run_all("newton_schulz", rows, cols, count, coefficients, steps, eps, ws, ws_bytes,
                 FillPlain{src, ld_src, dst, cols, type, (hipStream_t)stream});
}

int pgnn_muon_step(float* const* params, const float* const* grads, float* const* momentum, const float* rates, const int64_t* rows,
                   const int64_t* cols, int64_t count, float mu, int nesterov, float keep, const float* coefficients, int steps, float eps,
                   void* ws, size_t ws_bytes, pgnn_stream stream) {
  PGNN_REQUIRE(count <= 0 || (params && grads && momentum && rates), "muon_step: bad list of matrices");
  return run_all("muon_step", rows, cols, count, coefficients, steps, eps, ws, ws_bytes,
                 FillMuon{params, grads, momentum, rates, cols, mu, keep, nesterov, (hipStream_t)stream});
}

}  // extern "C"
