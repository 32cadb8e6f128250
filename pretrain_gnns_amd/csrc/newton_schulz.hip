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
// X is kept as X^T only: the product B X contracts along rows of B and of X^T (the fragments of an MFMA are 16-byte pieces of rows),
// and X X^T contracts down the rows of X^T, whose fragments ds_read_b64_tr_b16 turns on their way out of LDS (keeping X as well
// doubled what the last product writes and reads: ten 300 x 600 14.0 instead of 12.5 us).  A and B are symmetric: only the tiles on
// and above the diagonal are computed, and written twice.  a X is added behind the product B X, in fp32: as a I inside B it would stand in
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

constexpr int kGram = 0, kPoly = 1, kApply = 2, kLast = 3;  // (not an unnamed enum: its name in a kernel differs between host and device)

__host__ __device__ inline int parts_of(int64_t k, int64_t n) {
  const int64_t p = (k * n + kNormPart - 1) / kNormPart;
  return (int)(p < kMaxParts ? p : kMaxParts);
}

// where a matrix's planes are in its part of the workspace (bytes): the exponents and the partial sums in front, at fixed places; planes
// of 64 k columns are multiples of 256 bytes by themselves
constexpr int64_t kExps = 0, kParts = 512, kPlanes = kParts + kMaxParts * 8;
static_assert(3 * (kMaxSteps + 1) * 4 <= kParts && kPlanes % 256 == 0, "");
struct Layout {
  int64_t ldk, rows, xt0, xt1, a, b, bytes;  // X^T: `rows` rows, n of them and zeros up to whole stages
};
__host__ __device__ inline Layout layout_of(int64_t k, int64_t n) {
  Layout l;
  l.ldk = (k + kPad - 1) & ~(int64_t)(kPad - 1);
  l.rows = (n + kBK - 1) & ~(int64_t)(kBK - 1);
  l.xt0 = kPlanes;
  l.xt1 = l.xt0 + 4 * l.rows * l.ldk;
  l.a = l.xt1 + 4 * l.rows * l.ldk;
  l.b = l.a + 4 * k * l.ldk;
  l.bytes = l.b + 4 * k * l.ldk;
  return l;
}

// a matrix of the call: its first workgroup in this launch, its sizes (k <= n), whether G has more rows than columns, its workspace
struct Job {
  int first, k, n, tall;
  int64_t off;
};
struct Jobs {
  int count, blocks, xcds;
  char* ws;
  Job job[kMaxJobs];
};
struct Sources {
  const void* src[kMaxJobs];  // G
  int64_t ld[kMaxJobs];
};
struct Results {
  void* dst[kMaxJobs];        // the orthogonal matrix, or the parameter
};
struct MuonArgs {
  float* momentum[kMaxJobs];
  float rate[kMaxJobs];
  float mu, keep;           // keep = 1 - lr wd
  int nesterov;
};
struct Nothing { int unused; };  // (not empty: an empty kernel argument is dropped on the device side only)
template <bool MUON> using Muon = typename std::conditional<MUON, MuonArgs, Nothing>::type;
template <int PHASE> using Last = typename std::conditional<PHASE == kLast, Results, Nothing>::type;
struct Bounds {             // of the iteration on [0, 1]: max |p| after t steps, max |b x^2 + c x^4| in step t
  float coef[kMaxSteps][3];
  float cap_x[kMaxSteps + 1], cap_b[kMaxSteps];
  int steps;
  float eps;
};

// the job of a workgroup, found by one vector load and a ballot: a bisection is a chain of scalar loads, each of which waits for the
// kernel arguments anew
__device__ __forceinline__ int find_job(const Jobs& jobs, int b) {
  const int lane = threadIdx.x & 63;
  const int first = lane < jobs.count ? jobs.job[lane].first : 0x7fffffff;
  return __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(first <= b)) - 1);
}
// 16 bytes of G at the element's own alignment
template <typename T> struct Piece { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); static constexpr int n = 16 / sizeof(T); };

// partial sums of squares in float64 (millions of terms, squares of gradients far below 1); Muon: the momentum is advanced here
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_norm(Jobs jobs, Sources from, Muon<MUON> mu) {
  const int j = find_job(jobs, blockIdx.x);
  const Job job = jobs.job[j];
  const int rows = job.tall ? job.n : job.k, cols = job.tall ? job.k : job.n;
  const int nparts = parts_of(job.k, job.n), part = blockIdx.x - job.first;
  const T* g = static_cast<const T*>(from.src[j]);
  const int64_t ld = from.ld[j];
  constexpr int E = Piece<T>::n;
  double s = 0.0;
  auto add = [&](float v, float& m) {
    if constexpr (MUON) {
      m = fmaf(mu.mu, m, v);
      v = mu.nesterov ? fmaf(mu.mu, m, v) : m;
    }
    s += (double)v * (double)v;
  };
  // a dense matrix is one long row; else the workgroup's lanes walk the pieces of row after row
  const bool dense = ld == cols || rows == 1;
  const int64_t width = dense ? (int64_t)rows * cols : cols, pieces = (width + E - 1) / E;
  const int64_t stride = (int64_t)nparts * 256, start = (int64_t)part * 256 + threadIdx.x;
  int64_t r = 0, c = start;
  if (!dense) { r = start / pieces; c = start - r * pieces; }
  const int64_t dr = dense ? 0 : stride / pieces, dc = dense ? stride : stride - dr * pieces;
  while (dense ? c < pieces : r < rows) {
    const int64_t at = r * ld + c * E;
    [[maybe_unused]] float* m = nullptr;
    if constexpr (MUON) m = mu.momentum[j] + at;  // (dense: ld == cols)
    if (c * E + E <= width) {
      const typename Piece<T>::type p = *reinterpret_cast<const typename Piece<T>::type*>(g + at);
      typename Piece<float>::type mv = {0.f, 0.f, 0.f, 0.f};
      if constexpr (MUON) mv = *reinterpret_cast<typename Piece<float>::type*>(m);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float t = mv[e & 3];
        add((float)p[e], t);
        mv[e & 3] = t;
      }
      if constexpr (MUON) *reinterpret_cast<typename Piece<float>::type*>(m) = mv;
    } else {
      for (int e = 0; e < E && c * E + e < width; ++e) {
        float t = 0.f;
        if constexpr (MUON) t = m[e];
        add((float)g[at + e], t);
        if constexpr (MUON) m[e] = t;
      }
    }
    c += dc;
    r += dr;
    if (!dense && c >= pieces) { c -= pieces; ++r; }
  }
  __shared__ double lds[4];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<double*>(jobs.ws + job.off + kParts)[part] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// exponent e with bound * 2^e <= 2^13 (entries then stay a factor of 8 below fp16's largest value)
__device__ __forceinline__ int plane_exponent(float bound) { return 12 - ilogbf(bound); }

__device__ __forceinline__ void split8(const float (&v)[8], f16x8& h, f16x8& l) {
  uint32_t hh[4], ll[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) split2(v[2 * q], v[2 * q + 1], hh[q], ll[q]);
  h = __builtin_bit_cast(f16x8, make_uint4(hh[0], hh[1], hh[2], hh[3]));
  l = __builtin_bit_cast(f16x8, make_uint4(ll[0], ll[1], ll[2], ll[3]));
}

// X_0^T as planes, and the exponents of all planes to come
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_split(Jobs jobs, Sources from, Muon<MUON> mu, Bounds bd) {
  const int b = xcd_remap(blockIdx.x, jobs.blocks, jobs.xcds);
  const int j = find_job(jobs, b);
  const Job job = jobs.job[j];
  const bool tall = job.tall;
  const int rows = tall ? job.n : job.k, cols = tall ? job.k : job.n;
  const Layout l = layout_of(job.k, job.n);
  char* base = jobs.ws + job.off;
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int nparts = parts_of(job.k, job.n);
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
  const int local = b - job.first;
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
  const T* g = static_cast<const T*>(from.src[j]);
  const int64_t ld = from.ld[j];
  constexpr int E = Piece<T>::n, ACROSS = 64 / E;
#pragma unroll
  for (int q = 0; q < 64 * ACROSS / 256; ++q) {
    const int i = q * 256 + threadIdx.x, r = i / ACROSS, c = i % ACROSS * E;
    float v[E];
    const bool in = r0 + r < rows;
    if (in && c0 + c + E <= cols) {
      const typename Piece<T>::type p = *reinterpret_cast<const typename Piece<T>::type*>(g + (r0 + r) * ld + c0 + c);
      typename Piece<float>::type m = {0.f, 0.f, 0.f, 0.f};
      if constexpr (MUON) m = *reinterpret_cast<const typename Piece<float>::type*>(mu.momentum[j] + (int64_t)(r0 + r) * cols + c0 + c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = (float)p[e];
        if constexpr (MUON) v[e] = mu.nesterov ? fmaf(mu.mu, m[e & 3], v[e]) : m[e & 3];  // the momentum that k_ns_norm has advanced
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = 0.f;
        if (in && c0 + c + e < cols) {
          v[e] = (float)g[(r0 + r) * ld + c0 + c + e];
          if constexpr (MUON) {
            const float m = mu.momentum[j][(int64_t)(r0 + r) * cols + c0 + c + e];
            v[e] = mu.nesterov ? fmaf(mu.mu, m, v[e]) : m;
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) tile[r][c + e] = v[e] * inv * scale;
  }
  __syncthreads();
  _Float16* d = reinterpret_cast<_Float16*>(base + l.xt0);
  const int dr0 = tall ? r0 : c0, dc0 = tall ? c0 : r0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = q * 256 + threadIdx.x, r = i >> 3, c = (i & 7) * 8;
    if (dr0 + r >= (int)l.rows) continue;  // (rows n .. l.rows: zeros)
    float v[8];
    if (tall) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[c + e][r];
    }
    f16x8 h, lo;
    split8(v, h, lo);
    const int64_t at = (int64_t)(dr0 + r) * l.ldk + dc0 + c;
    *reinterpret_cast<f16x8*>(d + at) = h;
    *reinterpret_cast<f16x8*>(d + l.rows * l.ldk + at) = lo;
  }
}

// tile (ti, tj) of a launch's local index: columns of tiles in bands of kBand, a band row by row, so that the workgroups that run at the
// same time on an XCD (it takes a contiguous range) share kBand rows and columns of tiles in its L2.  symmetric: ti <= tj only
constexpr int kBand = 8;
template <typename T> struct Out8 { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
__device__ __forceinline__ void tile_at(int local, int down, int across, bool symmetric, int& ti, int& tj) {
  if (!symmetric) {
    const int band = local / (down * kBand), rem = local - band * down * kBand, w = min(kBand, across - band * kBand);
    ti = rem / w;
    tj = band * kBand + rem - ti * w;
    return;
  }
  // full bands before band b hold kBand^2 b (b - 1) / 2 + b kBand (kBand + 1) / 2 = 32 b^2 + 4 b tiles
  int band = (int)((sqrtf(16.f + 128.f * (float)local) - 4.f) * (1.f / 64.f));
  while (32 * band * band + 4 * band > local) --band;
  while (32 * (band + 1) * (band + 1) + 4 * (band + 1) <= local) ++band;
  const int rem = local - (32 * band * band + 4 * band), first = band * kBand, w = min(kBand, across - first);
  if (rem < first * w) {
    ti = rem / w;
    tj = first + rem - ti * w;
  } else {  // the triangle on the diagonal, column by column
    int t = rem - first * w;
    tj = first;
    while (t > tj - first) {
      t -= tj - first + 1;
      ++tj;
    }
    ti = first + t;
  }
}

// four blocks of 16 columns x 32 l, both planes, turned on their way out of LDS: at[b] the lane's address of block b, H the distance of
// l + 4, ARR that of the low plane.  One asm block with its own wait: with the builtin hipcc waits for every DMA in flight in front of the
// reads (ten 300 x 600: X X^T 15.7 us instead of 11.0), and a load of inline asm must not leave its block unfinished.
template <int H, int ARR>
__device__ __forceinline__ void read_turned(const uint32_t (&at)[4], f16x8 (&hi)[4], f16x8 (&lo)[4]) {
  uint2 r[4][4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%20\n\tds_read_b64_tr_b16 %2, %16 offset:%21\n\tds_read_b64_tr_b16 %3, %16 offset:%22\n\t"
      "ds_read_b64_tr_b16 %4, %17\n\tds_read_b64_tr_b16 %5, %17 offset:%20\n\tds_read_b64_tr_b16 %6, %17 offset:%21\n\tds_read_b64_tr_b16 %7, %17 offset:%22\n\t"
      "ds_read_b64_tr_b16 %8, %18\n\tds_read_b64_tr_b16 %9, %18 offset:%20\n\tds_read_b64_tr_b16 %10, %18 offset:%21\n\tds_read_b64_tr_b16 %11, %18 offset:%22\n\t"
      "ds_read_b64_tr_b16 %12, %19\n\tds_read_b64_tr_b16 %13, %19 offset:%20\n\tds_read_b64_tr_b16 %14, %19 offset:%21\n\tds_read_b64_tr_b16 %15, %19 offset:%22\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[1][2]), "=&v"(r[1][3]),
        "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[2][2]), "=&v"(r[2][3]), "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[3][2]), "=&v"(r[3][3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(H), "n"(ARR), "n"(ARR + H)
      : "memory");
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    hi[b] = __builtin_bit_cast(f16x8, make_uint4(r[b][0].x, r[b][0].y, r[b][1].x, r[b][1].y));
    lo[b] = __builtin_bit_cast(f16x8, make_uint4(r[b][2].x, r[b][2].y, r[b][3].x, r[b][3].y));
  }
}

// One TT x TT tile of a product on planes, C[i][j] = sum_l P(i, l) Q(j, l).  Four waves of TT/2 x TT/2; wave w fetches operand array w
// (P high, P low, Q high, Q low) by LDS DMA, STAGES - 1 stages ahead.  A stage is 32 deep.
//   A A and B X: l runs along the operands' rows.  A stage holds 64 bytes of TT rows, whose four 16-byte pieces are permuted by
//   (row >> 1) & 3, so that the eight rows of a piece that one LDS cycle reads lie in eight different bank groups.
//   X X^T: l runs down the rows of X^T.  A stage holds 32 rows of 2 TT bytes; a fragment (8 l of one column per lane) is two
//   ds_read_b64_tr_b16, each of which hands a 16-lane group a 4 x 16 block turned.  The 32-byte blocks of a row are permuted by bits of
//   the row, so that the 16 rows that one instruction reads lie evenly over the banks.
template <int TT, int STAGES, int PHASE, typename TO, bool MUON>
__global__ void __launch_bounds__(256) k_ns_product(Jobs jobs, Last<PHASE> to, Muon<MUON> mu, int step, float ca, float cb, float cc) {
  constexpr int MI = TT / 32, ARR = TT * kBK * 2, STAGE = 4 * ARR, NJ = TT / 16;
  constexpr int LDT = TT + 4;  // floats per row of the epilogue's tile: 16-byte rows, neighbours four banks apart
  extern __shared__ __align__(16) char smem[];
  const int b = xcd_remap(blockIdx.x, jobs.blocks, jobs.xcds);
  const int j = find_job(jobs, b);
  const Job job = jobs.job[j];
  const int k = job.k, n = job.n;
  const Layout l = layout_of(k, n);
  char* base = jobs.ws + job.off;
  int ti, tj;
  tile_at(b - job.first, (k + TT - 1) / TT, ((PHASE <= kPoly ? k : n) + TT - 1) / TT, PHASE <= kPoly, ti, tj);
  const int* exps = reinterpret_cast<const int*>(base + kExps);
  const int eX = exps[step], eA = exps[kMaxSteps + 1 + step], eB = exps[2 * (kMaxSteps + 1) + step], eY = exps[step + 1];
  const int64_t xt_in = step & 1 ? l.xt1 : l.xt0, xt_out = step & 1 ? l.xt0 : l.xt1;
  const _Float16* XT = reinterpret_cast<const _Float16*>(base + xt_in);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i0 = ti * TT, j0 = tj * TT, ldk = (int)l.ldk;

  // the wave's DMA pieces: 1 KB each
  const _Float16* src;
  uint32_t offs[NJ];  // in halfs; what lies beyond the matrix re-reads its last row or column (the results are not stored)
  int64_t advance;    // per stage
  int nk;
  if constexpr (PHASE == kGram) {
    constexpr int UNITS = TT / 8, ROWS = 64 / UNITS;  // 16-byte units per row, rows per piece
    src = XT + (wave & 1) * l.rows * ldk;
    nk = (int)l.rows / kBK;
    advance = (int64_t)kBK * ldk;
#pragma unroll
    for (int q = 0; q < NJ; ++q) {
      const int r = q * ROWS + lane / UNITS, u = lane % UNITS;
      const int turn = TT == 64 ? ((r >> 1) & 1) | ((r >> 2) & 2) : (r & 3) | ((r >> 1) & 4);
      const int col = (wave < 2 ? i0 : j0) + (((u >> 1) ^ turn) * 2 + (u & 1)) * 8;
      offs[q] = (uint32_t)r * (uint32_t)ldk + (uint32_t)min(col, ldk - 8);
    }
  } else {
    const _Float16* P = reinterpret_cast<const _Float16*>(base + (PHASE == kPoly ? l.a : l.b));
    const _Float16* Q = PHASE == kPoly ? P : XT;
    const int qrows = PHASE == kPoly ? k : (int)l.rows;
    src = wave < 2 ? P + (int64_t)(wave & 1) * k * ldk : Q + (int64_t)(wave & 1) * qrows * ldk;
    nk = ldk / kBK;
    advance = kBK;
#pragma unroll
    for (int q = 0; q < NJ; ++q) {
      const int r = q * 16 + (lane >> 2);
      const int row = min((wave < 2 ? i0 : j0) + r, (wave < 2 ? k : qrows) - 1);
      offs[q] = (uint32_t)row * (uint32_t)ldk + (uint32_t)(((lane & 3) ^ ((r >> 1) & 3)) * 8);
    }
  }
  auto issue = [&](int t) {
    char* dst = smem + (t % STAGES) * STAGE + wave * ARR;
#pragma unroll
    for (int q = 0; q < NJ; ++q)
      __builtin_amdgcn_global_load_lds(PGNN_GPTR(src + (size_t)offs[q] + (size_t)t * advance), PGNN_LPTR(dst + q * 1024), 16, 0, 0);
  };

  // the epilogue's operand (A behind A A, X^T behind B X) at this thread's pieces of the tile, fetched in front of everything else: its
  // round trip to memory hides behind the product
  constexpr int PIECES = TT / 8, MINE = TT * PIECES / 256;  // 16-byte pieces per row, pieces per thread
  const int out_rows = PHASE <= kPoly ? k : (int)l.rows;
  [[maybe_unused]] f16x8 eh[MINE], el[MINE];
  if constexpr (PHASE != kGram) {
    const _Float16* E = PHASE == kPoly ? reinterpret_cast<const _Float16*>(base + l.a) : XT;
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      const int r = (q * 256 + threadIdx.x) / PIECES, c = (threadIdx.x % PIECES) * 8;
      const int64_t at = (int64_t)min(j0 + r, out_rows - 1) * ldk + min(i0 + c, ldk - 8);
      eh[q] = *reinterpret_cast<const f16x8*>(E + at);
      el[q] = *reinterpret_cast<const f16x8*>(E + (int64_t)out_rows * ldk + at);
    }
  }

  const int wi = (wave >> 1) * (TT / 2), wj = (wave & 1) * (TT / 2);
  const int fr = lane & 15, fc = lane >> 4;
  // byte offsets of the lane's fragments inside a stage: block a of the wave's rows i and of its rows j (X X^T: of its columns)
  uint32_t pat[MI], qat[MI];
#pragma unroll
  for (int a = 0; a < MI; ++a) {
    const int pb = wi / 16 + a, qb = wj / 16 + a;
    if constexpr (PHASE == kGram) {  // rows l = 8 fc + fr / 4; the rows l + 4 have the same permutation
      const int r = 8 * fc + (fr >> 2);
      const int turn = TT == 64 ? ((r >> 1) & 1) | ((r >> 2) & 2) : (r & 3) | ((r >> 1) & 4);
      pat[a] = (uint32_t)(r * TT * 2 + (pb ^ turn) * 32 + (fr & 3) * 8);
      qat[a] = (uint32_t)(r * TT * 2 + (qb ^ turn) * 32 + (fr & 3) * 8 + 2 * ARR);
    } else {
      pat[a] = (uint32_t)((pb * 16 + fr) * 64 + ((fc ^ ((fr >> 1) & 3)) * 16));
      qat[a] = (uint32_t)((qb * 16 + fr) * 64 + ((fc ^ ((fr >> 1) & 3)) * 16) + 2 * ARR);
    }
  }

  f32x4 acc[MI][MI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < MI; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};

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
    if constexpr (PHASE == kGram) {
      const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)st;
      if constexpr (MI == 2) {
        f16x8 h[4], lo[4];
        read_turned<4 * TT * 2, ARR>({at + pat[0], at + pat[1], at + qat[0], at + qat[1]}, h, lo);
#pragma unroll
        for (int a = 0; a < 2; ++a) { ph[a] = h[a]; pl[a] = lo[a]; qh[a] = h[2 + a]; ql[a] = lo[2 + a]; }
      } else {
        static_assert(MI == 2 || MI == 4, "");
        read_turned<4 * TT * 2, ARR>({at + pat[0], at + pat[1], at + pat[2], at + pat[3]}, ph, pl);
        read_turned<4 * TT * 2, ARR>({at + qat[0], at + qat[1], at + qat[2], at + qat[3]}, qh, ql);
      }
    } else {
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        ph[a] = *reinterpret_cast<const f16x8*>(st + pat[a]);
        pl[a] = *reinterpret_cast<const f16x8*>(st + pat[a] + ARR);
        qh[a] = *reinterpret_cast<const f16x8*>(st + qat[a]);
        ql[a] = *reinterpret_cast<const f16x8*>(st + qat[a] + ARR);
      }
    }
#pragma unroll
    for (int c = 0; c < MI; ++c) {  // smallest terms first
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], ql[c], acc[a][c], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a], qh[c], acc[a][c], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], qh[c], acc[a][c], 0, 0, 0);
    }
    asm volatile("" ::: "memory");
  }

  // epilogue: the tile to LDS as fp32 [j][i] (a lane holds four consecutive i of one j), out row by row as the operand lies (rows j),
  // and once more turned (rows i) where the mirror image of a symmetric tile or a wide G wants it
  __syncthreads();
  float* tile = reinterpret_cast<float*>(smem);
  const float f = PHASE == kGram ? ldexpf(1.f, eA - 2 * eX) : PHASE == kPoly ? ldexpf(cc, eB - 2 * eA)
                : PHASE == kApply ? ldexpf(1.f, eY - eX - eB) : ldexpf(1.f, -eX - eB);
  const float fe = PHASE == kPoly ? ldexpf(cb, eB - eA) : PHASE == kApply ? ldexpf(ca, eY - eX) : ldexpf(ca, -eX);
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < MI; ++c)
      *reinterpret_cast<f32x4*>(tile + (wj + c * 16 + fr) * LDT + wi + a * 16 + fc * 4) = acc[a][c] * f;
  __syncthreads();

  auto planes_out = [&](_Float16* d, int rows, int64_t at, const float (&v)[8]) {
    f16x8 h, lo;
    split8(v, h, lo);
    *reinterpret_cast<f16x8*>(d + at) = h;
    *reinterpret_cast<f16x8*>(d + (int64_t)rows * ldk + at) = lo;
  };
  [[maybe_unused]] auto result_out = [&](int64_t at, int m, const float (&v)[8]) {  // m of the 8 values exist
    if constexpr (PHASE == kLast) {
      TO* d = static_cast<TO*>(to.dst[j]) + at;
      if (m >= 8) {
        typename Out8<TO>::type o;
        if constexpr (MUON) o = *reinterpret_cast<typename Out8<TO>::type*>(d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (MUON) o[e] = fmaf(-mu.rate[j], v[e], o[e] * mu.keep);
          else o[e] = (TO)v[e];
        }
        *reinterpret_cast<typename Out8<TO>::type*>(d) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= m) break;
          if constexpr (MUON) d[e] = fmaf(-mu.rate[j], v[e], d[e] * mu.keep);
          else d[e] = (TO)v[e];
        }
      }
    }
  };
  const bool again = PHASE <= kPoly ? ti != tj : PHASE == kLast && !job.tall;
  _Float16* D = reinterpret_cast<_Float16*>(base + (PHASE == kGram ? l.a : PHASE == kPoly ? l.b : xt_out));
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    const int r = (q * 256 + threadIdx.x) / PIECES, c = (threadIdx.x % PIECES) * 8;
    float* p = tile + r * LDT + c;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
    if constexpr (PHASE != kGram) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(fe, (float)eh[q][e] + (float)el[q][e], v[e]);
      if (again) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
      }
    }
    if constexpr (PHASE != kLast) {
      if (j0 + r < out_rows && i0 + c < ldk) {  // zeros beyond the matrix: the next products contract over them
        const bool row_in = j0 + r < (PHASE <= kPoly ? k : n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row_in && i0 + c + e < k ? v[e] : 0.f;
        planes_out(D, out_rows, (int64_t)(j0 + r) * ldk + i0 + c, v);
      }
    } else if (!again && j0 + r < n) {
      result_out((int64_t)(j0 + r) * k + i0 + c, k - (i0 + c), v);
    }
  }
  if (!again) return;
  if constexpr (PHASE != kGram) __syncthreads();
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    const int r = (q * 256 + threadIdx.x) / PIECES, c = (threadIdx.x % PIECES) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(c + e) * LDT + r];
    if constexpr (PHASE <= kPoly) {
      if (i0 + r < k && j0 + c < ldk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = j0 + c + e < k ? v[e] : 0.f;
        planes_out(D, k, (int64_t)(i0 + r) * ldk + j0 + c, v);
      }
    } else {
      if (i0 + r < k) result_out((int64_t)(i0 + r) * n + j0 + c, n - (j0 + c), v);
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
template <typename Count>
void place(Jobs& jobs, Count blocks_of) {
  jobs.blocks = 0;
  for (int j = 0; j < jobs.count; ++j) {
    jobs.job[j].first = jobs.blocks;
    jobs.blocks += blocks_of(jobs.job[j]);
  }
}

template <int TT, int STAGES, int PHASE, typename TO, bool MUON>
void launch_product(Jobs& jobs, const Last<PHASE>& to, const Muon<MUON>& mu, int step, const float* c, hipStream_t st) {
  place(jobs, [](const Job& q) { return tiles_of<TT>(q.k, q.n, PHASE <= kPoly); });
  constexpr size_t lds = std::max<size_t>((size_t)STAGES * 4 * TT * kBK * 2, (size_t)TT * (TT + 4) * 4);
  const void* fn = (const void*)k_ns_product<TT, STAGES, PHASE, TO, MUON>;
  allow_big_lds(fn, lds);
  hipLaunchKernelGGL((k_ns_product<TT, STAGES, PHASE, TO, MUON>), dim3(jobs.blocks), dim3(256), lds, st, jobs, to, mu, step, c[0], c[1], c[2]);
}

template <int TT, int STAGES, typename TO, bool MUON>
void run_steps(Jobs& jobs, const Results& to, const Muon<MUON>& mu, const Bounds& bd, hipStream_t st) {
  const Nothing no{0};
  for (int t = 0; t < bd.steps; ++t) {
    launch_product<TT, STAGES, kGram, float, false>(jobs, no, no, t, bd.coef[t], st);
    launch_product<TT, STAGES, kPoly, float, false>(jobs, no, no, t, bd.coef[t], st);
    if (t + 1 < bd.steps) launch_product<TT, STAGES, kApply, float, false>(jobs, no, no, t, bd.coef[t], st);
    else launch_product<TT, STAGES, kLast, TO, MUON>(jobs, to, mu, t, bd.coef[t], st);
  }
}

template <typename T, bool MUON>
void run_chunk(Jobs& jobs, const Sources& from, const Results& to, const Muon<MUON>& mu, const Bounds& bd, hipStream_t st) {
  place(jobs, [](const Job& q) { return parts_of(q.k, q.n); });
  hipLaunchKernelGGL((k_ns_norm<T, MUON>), dim3(jobs.blocks), dim3(256), 0, st, jobs, from, mu);
  place(jobs, [](const Job& q) { return tiles_of<64>(q.k, q.n, false); });
  hipLaunchKernelGGL((k_ns_split<T, MUON>), dim3(jobs.blocks), dim3(256), 0, st, jobs, from, mu, bd);
  int64_t big = 0;
  for (int j = 0; j < jobs.count; ++j) big += tiles_of<128>(jobs.job[j].k, jobs.job[j].n, true);
  if (big >= num_cu()) run_steps<128, 2, T, MUON>(jobs, to, mu, bd, st);
  else run_steps<64, 4, T, MUON>(jobs, to, mu, bd, st);
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
    Sources src{};
    Results res{};
    MuonArgs mu{};
    jobs.ws = (char*)ws;
    jobs.xcds = num_xcd();
    int64_t off = 0;
    for (int64_t j = from; j < to; ++j) {
      if (rows[j] == 0 || cols[j] == 0) continue;
      const int q = jobs.count++;
      jobs.job[q] = Job{0, (int)std::min(rows[j], cols[j]), (int)std::max(rows[j], cols[j]), rows[j] > cols[j], off};
      off += layout_of(jobs.job[q].k, jobs.job[q].n).bytes;
      fill.set(src, res, mu, q, j);
    }
    if (jobs.count) fill.run(jobs, src, res, mu, bd);
    launched |= jobs.count > 0;
    from = to;
  }
  return launched ? check_launch(what) : PGNN_OK;
}

struct FillPlain {
  const void* const* src; const int64_t* ld; void* const* dst; int type; hipStream_t st;
  bool valid(int64_t j) const { return src[j] && dst[j] && ld[j] >= 0; }
  void set(Sources& s, Results& r, MuonArgs&, int q, int64_t j) const {
    s.src[q] = src[j];
    s.ld[q] = ld[j];
    r.dst[q] = dst[j];
  }
  void run(Jobs& jobs, const Sources& s, const Results& r, const MuonArgs&, const Bounds& bd) const {
    const Nothing no{0};
    if (type == PGNN_F32) run_chunk<float, false>(jobs, s, r, no, bd, st);
    else if (type == PGNN_BF16) run_chunk<__bf16, false>(jobs, s, r, no, bd, st);
    else run_chunk<_Float16, false>(jobs, s, r, no, bd, st);
  }
};
struct FillMuon {
  float* const* params; const float* const* grads; float* const* momentum; const float* rates; const int64_t* cols; float mu, keep; int nesterov;
  hipStream_t st;
  bool valid(int64_t j) const { return params[j] && grads[j] && momentum[j]; }
  void set(Sources& s, Results& r, MuonArgs& m, int q, int64_t j) const {
    s.src[q] = grads[j];
    s.ld[q] = cols[j];
    r.dst[q] = params[j];
    m.momentum[q] = momentum[j];
    m.rate[q] = rates[j];
  }
  void run(Jobs& jobs, const Sources& s, const Results& r, MuonArgs& m, const Bounds& bd) const {
    m.mu = mu;
    m.keep = keep;
    m.nesterov = nesterov;
    run_chunk<float, true>(jobs, s, r, m, bd, st);
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
                 FillPlain{src, ld_src, dst, type, (hipStream_t)stream});
}

int pgnn_muon_step(float* const* params, const float* const* grads, float* const* momentum, const float* rates, const int64_t* rows,
                   const int64_t* cols, int64_t count, float mu, int nesterov, float keep, const float* coefficients, int steps, float eps,
                   void* ws, size_t ws_bytes, pgnn_stream stream) {
  PGNN_REQUIRE(count <= 0 || (params && grads && momentum && rates), "muon_step: bad list of matrices");
  return run_all("muon_step", rows, cols, count, coefficients, steps, eps, ws, ws_bytes,
                 FillMuon{params, grads, momentum, rates, cols, mu, keep, nesterov, (hipStream_t)stream});
}

}  // extern "C"
