// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step that is built on it:
//   X_0 = G / (|G|_F + eps), transposed if it has more rows than columns (X is k x n, k <= n), then per step
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
// which drives the singular values of X towards 1 and leaves its singular vectors alone.  Muon orthogonalises the momentum:
//   M <- mu M + G,  U = G + mu M (nesterov) or M,  p <- p (1 - lr wd) - rate orthogonal(U)
//
// Everything after the first read of G lives as TWO fp16 planes h + l of s X, s a power of two (two_plane.h): three
// v_mfma_f32_16x16x32_f16 per block (h l, l h, h h) with fp32 accumulation, 3/16 of the matrix-core time of v_mfma_f32_16x16x4_f32, and
// two planes take the bytes of one fp32 matrix.  The iteration bounds its own
// entries -- |X_ij| <= |X|_2 <= u_t, with u_0 = |G|_F / (|G|_F + eps) and u_{t+1} the maximum of |a x + b x^3 + c x^5| on [0, u_t] --
// so ONE scale per matrix and step is known before a product runs: no row maxima, and no fp16 overflow for any input.
// What that gives up: planes hold a value to 2^-23 of itself (fp32: 2^-24) only down to 2^-16 u_t, where l becomes subnormal, and to 2^-37
// u_t below.  Sums of hundreds of fp32 terms lose more than 2^-23 of the norm, so in the norm the result is an fp32 iteration's (4096 x 4096:
// 3.0e-6 of the 64-bit one, the library's fp32 products 4.6e-6).  Rows far weaker than the rest are not (200 x 400 graded 1 to 1e-6: the weakest
// are 2.5e-4 of themselves off, 1e-5 with fp32 products; graded 1 to 1e-3: 2e-6 and 9e-6).  An exponent per row would have to scale the
// contraction index of A and B X, whose operands are the same planes; an optimizer's direction asks for the norm.
// X is kept as X^T only: the product B X contracts along rows of B and of X^T (the fragments of an MFMA are 16-byte pieces of rows),
// and X X^T contracts down the rows of X^T, whose fragments ds_read_b64_tr_b16 turns on their way out of LDS (keeping X as well
// doubled what the last product writes and reads: ten 300 x 600 14.0 instead of 12.5 us).  A and B are symmetric: only the tiles on
// and above the diagonal are computed, and written twice.  a X is added behind the product B X, in fp32: as a I inside B it would stand in
// the middle of each long sum and cost the small terms their last bits (4096 x 4096: 6.5e-6 of the 64-bit result instead of 3e-6).
// The matrices of a call share the launches: one if all are tiny (k_ns_tiny), 2 + 2 steps if all are small (kSmall), else 2 + 3 steps, and
// `steps` more where small ones go apart from large ones.  The launches stand in stream order and use nothing of an earlier call's workspace.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "two_plane.h"

using namespace pgnn;

namespace {

constexpr int kMaxJobs = 48;         // matrices per launch (their table travels in the kernel arguments: kArguments)
constexpr int kMaxSteps = 32;
constexpr int kMaxParts = 1024;      // partial sums of squares per matrix (256: one wave per SIMD, 4096 x 4096 40 us)
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
constexpr int kExpRow = kMaxSteps + 1;  // exponents of X_t, A_t, B_t, Z_t: four rows
constexpr int kMaxSplit = 128;          // tiles of a launch that are formed in parts, at most (a ticket each)
constexpr int64_t kExps = 0, kParts = 768, kTickets = kParts + kMaxParts * 8, kPlanes = kTickets + kMaxSplit * 4;
static_assert(4 * kExpRow * 4 <= kParts && kPlanes % 256 == 0, "");
// A matrix on planes lies in blocks of 16 rows x 32 columns, the high plane's 1 KB and then the low one's, down a column of blocks and then
// the next (what a stage of a product takes of an operand is one piece).  Inside a block the lane (fr, fc) of a wave that takes it as an operand -- row fr, columns 8 fc .. 8 fc + 7 -- has the 16
// bytes at unit_of(fr, fc): every fragment and every DMA is 1 KB in one piece (as 64- or 128-byte pieces of 16 rows of a row-major matrix
// a CU took 18 to 27 bytes per clock of them), and LDS holds blocks as memory does.  The xor keeps both ways
// of reading free of bank conflicts: ds_read_b128 takes rows 0-3 and 12-15 of one fc together with rows 4-11 of the next, and
// ds_read_b64_tr_b16 takes rows 0-3 and 8-11 of two neighbours (an xor by 4 does for the second only: A A of 4096 x 4096 268 instead of 264 us).
constexpr int kBlockHalfs = 1024;  // both planes
__host__ __device__ inline int unit_of(int fr, int fc) { return fc * 16 + (fr ^ ((fc & 1) * 12)); }
struct Layout {
  int64_t ldk, rows, xt0, xt1, a, b, bytes;  // ldk: columns, and rows of A and B; rows: of X^T, n of them, then zeros
};
__host__ __device__ inline Layout layout_of(int64_t k, int64_t n) {
  Layout l;
  l.ldk = (k + kPad - 1) & ~(int64_t)(kPad - 1);
  l.rows = (n + kPad - 1) & ~(int64_t)(kPad - 1);
  l.xt0 = kPlanes;
  l.xt1 = l.xt0 + 4 * l.rows * l.ldk;
  l.a = l.xt1 + 4 * l.rows * l.ldk;
  l.b = l.a + 4 * l.ldk * l.ldk;
  l.bytes = l.b + 4 * l.ldk * l.ldk;
  return l;
}
// where the eight columns c .. c + 7 of row r begin (halfs, high plane)
__device__ __forceinline__ int64_t piece_at(int rows, int r, int c) {
  return ((int64_t)(c >> 5) * (rows >> 4) + (r >> 4)) * kBlockHalfs + unit_of(r & 15, (c >> 3) & 3) * 8;
}
// row and first column of piece p of a tile WIDE columns wide, in the order in which the pieces lie in memory
template <int WIDE>
__device__ __forceinline__ void piece_of(int p, int& r, int& c) {
  const int block = p >> 6, fc = (p >> 4) & 3;
  r = block / (WIDE / 32) * 16 + ((p & 15) ^ ((fc & 1) * 12));
  c = block % (WIDE / 32) * 32 + fc * 8;
}

// a matrix of a launch: its first workgroup, its sizes (k <= n), whether G has more rows than columns, which matrix of the call it is, its
// workspace
struct Job {
  int first, k, n, tall;
  int64_t off;
  int64_t slot;
};
struct Jobs {
  int count, blocks, xcds;
  int split, parts;  // of a product: the first `split` tiles are formed in `parts` parts (1: none)
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

// k_ns_tiny takes all of these (3 964 bytes), the other kernels fewer; a launch's arguments are 4 KB at most
constexpr size_t kArguments = sizeof(Jobs) + sizeof(Sources) + sizeof(Results) + sizeof(MuonArgs) + sizeof(Bounds);
static_assert(kArguments <= 4096, "fewer matrices per launch");

// the job of a workgroup: every lane loads one, a ballot finds the last that begins at or before this workgroup, its fields are read from
// that lane.  One round trip to the kernel arguments; a bisection and a load of what it found are five
__device__ __forceinline__ Job find_job(const Jobs& jobs, int b) {
  const int lane = threadIdx.x & 63;
  const Job mine = jobs.job[min(lane, kMaxJobs - 1)];
  const int at = __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(lane < jobs.count && mine.first <= b)) - 1);
  Job f;
  f.slot = __builtin_amdgcn_readlane((int)mine.slot, at);
  f.first = __builtin_amdgcn_readlane(mine.first, at);
  f.k = __builtin_amdgcn_readlane(mine.k, at);
  f.n = __builtin_amdgcn_readlane(mine.n, at);
  f.tall = __builtin_amdgcn_readlane(mine.tall, at);
  f.off = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine.off, at) |
          (int64_t)__builtin_amdgcn_readlane((int)(mine.off >> 32), at) << 32;
  return f;
}
// 16 bytes of G at the element's own alignment
template <typename T> struct Piece { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); static constexpr int n = 16 / sizeof(T); };

// one of 256 threads' share of partial sum `part` of the squares, in float64 (millions of terms, squares of gradients far below 1); Muon:
// the momentum is advanced here
template <typename T, bool MUON>
__device__ __forceinline__ double squares(const Job& job, int part, int thread, const Sources& from, const Muon<MUON>& mu) {
  const int j = (int)job.slot;
  const int rows = job.tall ? job.n : job.k, cols = job.tall ? job.k : job.n;
  const int nparts = parts_of(job.k, job.n);
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
  const int64_t stride = (int64_t)nparts * 256, start = (int64_t)part * 256 + thread;
  int64_t r = 0, c = start;
  if (!dense) { r = start / pieces; c = start - r * pieces; }
  const int64_t dr = dense ? 0 : stride / pieces, dc = dense ? stride : stride - dr * pieces;
  const int64_t nrows = dense ? 1 : rows;
  while (c < pieces && r < nrows) {
    // four pieces on their way at a time; what is no whole piece is added on the spot
    typename Piece<T>::type p[4];
    [[maybe_unused]] typename Piece<float>::type mv[4];
    int64_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      at[q] = -1;
      if (c < pieces && r < nrows) {
        const int64_t a = r * ld + c * E;
        if (c * E + E <= width) {
          at[q] = a;
          p[q] = *reinterpret_cast<const typename Piece<T>::type*>(g + a);
          if constexpr (MUON) mv[q] = *reinterpret_cast<const typename Piece<float>::type*>(mu.momentum[j] + a);
        } else {
          for (int e = 0; e < E && c * E + e < width; ++e) {
            float m = 0.f;
            if constexpr (MUON) m = mu.momentum[j][a + e];  // (Muon: dense, ld == cols)
            add((float)g[a + e], m);
            if constexpr (MUON) mu.momentum[j][a + e] = m;
          }
        }
        c += dc;
        r += dr;
        if (!dense && c >= pieces) { c -= pieces; ++r; }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (at[q] >= 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float m = 0.f;
          if constexpr (MUON) m = mv[q][e & 3];
          add((float)p[q][e], m);
          if constexpr (MUON) mv[q][e & 3] = m;
        }
        if constexpr (MUON) *reinterpret_cast<typename Piece<float>::type*>(mu.momentum[j] + at[q]) = mv[q];
      }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  return s;  // (of the wave)
}

// (HBM: 4096 x 4096 fp32 14.6 us, 4.6 TB/s; Muon's 21 M values with the momentum 46 us, 5.5 TB/s)
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_norm(Jobs jobs, Sources from, Muon<MUON> mu) {
  const Job job = find_job(jobs, blockIdx.x);
  const int part = blockIdx.x - job.first;
  __shared__ double lds[4];
  const double s = squares<T, MUON>(job, part, threadIdx.x, from, mu);
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

// 1 / (norm + eps) as a factor in [0.5, 1) and an exponent: as one fp32 number it would leave the normal range for norms beyond 2^126
__device__ __forceinline__ float inverse(double norm, float eps, int& e) { return (float)frexp(1.0 / (norm + (double)eps), &e); }

// v inv 2^shift.  By the power first: v may be subnormal.  Rounded here in every kernel (not fused with what follows)
__device__ __forceinline__ float scaled(float v, int shift, float inv) {
  float x = ldexpf(v, shift) * inv;
  asm("" : "+v"(x));
  return x;
}

// the bound on X_0 from the norm, and what a step makes of a bound: exponents of A, B, Z and the next X
__device__ __forceinline__ float first_bound(const Bounds& bd, double norm) {
  float u = (float)(norm / (norm + (double)bd.eps)) * 1.001f;
  if (!(u >= 0x1p-60f)) u = 0x1p-60f;  // (also a NaN: everything becomes NaN whatever the scale)
  return u <= bd.cap_x[0] ? u : bd.cap_x[0];
}
struct StepExps { int a, b, z, y; };
__device__ __forceinline__ StepExps step_bounds(const Bounds& bd, int t, float& u) {
  const float a = fabsf(bd.coef[t][0]), b = fabsf(bd.coef[t][1]), c = fabsf(bd.coef[t][2]);
  StepExps e;
  const float al = fmaxf(1.001f * u * u, 0x1p-60f);
  e.a = plane_exponent(al);
  const float be = fmaxf(fminf(1.001f * al * (b + al * c), bd.cap_b[t]), 0x1p-60f);
  e.b = plane_exponent(be);
  e.z = plane_exponent(fmaxf(1.001f * u * (b + al * c), 0x1p-60f));  // Z = b X + c A X
  u = fmaxf(fminf((a + be) * u, bd.cap_x[t + 1]), 0x1p-60f);
  e.y = plane_exponent(u);
  return e;
}

// X_0^T as planes, and the exponents of all planes to come (HBM: 4096 x 4096 fp32 25.3 us, 5.3 TB/s)
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) k_ns_split(Jobs jobs, Sources from, Muon<MUON> mu, Bounds bd) {
  const int b = xcd_remap(blockIdx.x, jobs.blocks, jobs.xcds);
  const Job job = find_job(jobs, b);
  const int j = (int)job.slot;
  const bool tall = job.tall;
  const int rows = tall ? job.n : job.k, cols = tall ? job.k : job.n;
  const Layout l = layout_of(job.k, job.n);
  char* base = jobs.ws + job.off;
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int nparts = parts_of(job.k, job.n);
  double s = 0.0;
  for (int q = threadIdx.x; q < nparts; q += 256) s += reinterpret_cast<const double*>(base + kParts)[q];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  int shift;
  const float inv = inverse(norm, bd.eps, shift);
  float u = first_bound(bd, norm);
  const int e0 = plane_exponent(u);
  shift += e0;
  const int local = b - job.first;
  if (local == 0 && threadIdx.x < kMaxSplit) reinterpret_cast<unsigned*>(base + kTickets)[threadIdx.x] = 0;
  if (local == 0 && threadIdx.x == 0) {
    int* e = reinterpret_cast<int*>(base + kExps);
    e[0] = e0;
    for (int t = 0; t < bd.steps; ++t) {
      const StepExps x = step_bounds(bd, t, u);
      e[kExpRow + t] = x.a;
      e[2 * kExpRow + t] = x.b;
      e[3 * kExpRow + t] = x.z;
      e[t + 1] = x.y;
    }
  }
  const int tc = (int)((cols + 63) / 64), r0 = local / tc * 64, c0 = local % tc * 64;
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
    for (int e = 0; e < E; ++e) tile[r][c + e] = scaled(v[e], shift, inv);
  }
  __syncthreads();
  _Float16* d = reinterpret_cast<_Float16*>(base + l.xt0);
  const int dr0 = tall ? r0 : c0, dc0 = tall ? c0 : r0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    int r, c;
    piece_of<64>(q * 256 + threadIdx.x, r, c);  // (rows n .. l.rows: zeros)
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
    const int64_t at = piece_at((int)l.rows, dr0 + r, dc0 + c);
    *reinterpret_cast<f16x8*>(d + at) = h;
    *reinterpret_cast<f16x8*>(d + at + kBlockHalfs / 2) = lo;
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

// four blocks of 16 columns x 32 l, both planes, turned on their way out of LDS: at[b] the lane's address in block b's high plane, l + 4
// is that xor 64, the low plane 1 KB further.  One asm block with its own wait: with the builtin hipcc waits for every DMA in flight in
// front of the reads (ten 300 x 600: X X^T 15.7 us instead of 11.0), and a load of inline asm must not leave its block unfinished.
__device__ __forceinline__ void read_turned(const uint32_t (&at)[4], f16x8 (&hi)[4], f16x8 (&lo)[4]) {
  uint2 r[4][4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %20\n\tds_read_b64_tr_b16 %2, %16 offset:1024\n\tds_read_b64_tr_b16 %3, %20 offset:1024\n\t"
      "ds_read_b64_tr_b16 %4, %17\n\tds_read_b64_tr_b16 %5, %21\n\tds_read_b64_tr_b16 %6, %17 offset:1024\n\tds_read_b64_tr_b16 %7, %21 offset:1024\n\t"
      "ds_read_b64_tr_b16 %8, %18\n\tds_read_b64_tr_b16 %9, %22\n\tds_read_b64_tr_b16 %10, %18 offset:1024\n\tds_read_b64_tr_b16 %11, %22 offset:1024\n\t"
      "ds_read_b64_tr_b16 %12, %19\n\tds_read_b64_tr_b16 %13, %23\n\tds_read_b64_tr_b16 %14, %19 offset:1024\n\tds_read_b64_tr_b16 %15, %23 offset:1024\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[1][2]), "=&v"(r[1][3]),
        "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[2][2]), "=&v"(r[2][3]), "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[3][2]), "=&v"(r[3][3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[0] ^ 64u), "v"(at[1] ^ 64u), "v"(at[2] ^ 64u), "v"(at[3] ^ 64u)
      : "memory");
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    hi[b] = __builtin_bit_cast(f16x8, make_uint4(r[b][0].x, r[b][0].y, r[b][1].x, r[b][1].y));
    lo[b] = __builtin_bit_cast(f16x8, make_uint4(r[b][2].x, r[b][2].y, r[b][3].x, r[b][3].y));
  }
}

// the same for four neighbouring blocks of P and of Q in one go: block 1 lies 512 bytes behind block 0 (two units of 16), 2 and 3 2 KB
// behind those (p, q: blocks 0, of even number).  Two waits instead of one: 4096 x 4096 3650 us instead of 3617, ten 1024 x 2048 1352, 1335
__device__ __forceinline__ void read_turned8(uint32_t p, uint32_t q, f16x8 (&ph)[4], f16x8 (&pl)[4], f16x8 (&qh)[4], f16x8 (&ql)[4]) {
  uint2 r[2][4][4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %32 offset:0\n\t"
      "ds_read_b64_tr_b16 %1, %33 offset:0\n\t"
      "ds_read_b64_tr_b16 %2, %32 offset:1024\n\t"
      "ds_read_b64_tr_b16 %3, %33 offset:1024\n\t"
      "ds_read_b64_tr_b16 %4, %32 offset:512\n\t"
      "ds_read_b64_tr_b16 %5, %33 offset:512\n\t"
      "ds_read_b64_tr_b16 %6, %32 offset:1536\n\t"
      "ds_read_b64_tr_b16 %7, %33 offset:1536\n\t"
      "ds_read_b64_tr_b16 %8, %32 offset:2048\n\t"
      "ds_read_b64_tr_b16 %9, %33 offset:2048\n\t"
      "ds_read_b64_tr_b16 %10, %32 offset:2048+1024\n\t"
      "ds_read_b64_tr_b16 %11, %33 offset:2048+1024\n\t"
      "ds_read_b64_tr_b16 %12, %32 offset:2560\n\t"
      "ds_read_b64_tr_b16 %13, %33 offset:2560\n\t"
      "ds_read_b64_tr_b16 %14, %32 offset:3584\n\t"
      "ds_read_b64_tr_b16 %15, %33 offset:3584\n\t"
      "ds_read_b64_tr_b16 %16, %34 offset:0\n\t"
      "ds_read_b64_tr_b16 %17, %35 offset:0\n\t"
      "ds_read_b64_tr_b16 %18, %34 offset:1024\n\t"
      "ds_read_b64_tr_b16 %19, %35 offset:1024\n\t"
      "ds_read_b64_tr_b16 %20, %34 offset:512\n\t"
      "ds_read_b64_tr_b16 %21, %35 offset:512\n\t"
      "ds_read_b64_tr_b16 %22, %34 offset:1536\n\t"
      "ds_read_b64_tr_b16 %23, %35 offset:1536\n\t"
      "ds_read_b64_tr_b16 %24, %34 offset:2048\n\t"
      "ds_read_b64_tr_b16 %25, %35 offset:2048\n\t"
      "ds_read_b64_tr_b16 %26, %34 offset:2048+1024\n\t"
      "ds_read_b64_tr_b16 %27, %35 offset:2048+1024\n\t"
      "ds_read_b64_tr_b16 %28, %34 offset:2560\n\t"
      "ds_read_b64_tr_b16 %29, %35 offset:2560\n\t"
      "ds_read_b64_tr_b16 %30, %34 offset:3584\n\t"
      "ds_read_b64_tr_b16 %31, %35 offset:3584\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0][0][0]), "=&v"(r[0][0][1]), "=&v"(r[0][0][2]), "=&v"(r[0][0][3]), "=&v"(r[0][1][0]), "=&v"(r[0][1][1]), "=&v"(r[0][1][2]), "=&v"(r[0][1][3]), "=&v"(r[0][2][0]), "=&v"(r[0][2][1]), "=&v"(r[0][2][2]), "=&v"(r[0][2][3]), "=&v"(r[0][3][0]), "=&v"(r[0][3][1]), "=&v"(r[0][3][2]), "=&v"(r[0][3][3]), "=&v"(r[1][0][0]), "=&v"(r[1][0][1]), "=&v"(r[1][0][2]), "=&v"(r[1][0][3]), "=&v"(r[1][1][0]), "=&v"(r[1][1][1]), "=&v"(r[1][1][2]), "=&v"(r[1][1][3]), "=&v"(r[1][2][0]), "=&v"(r[1][2][1]), "=&v"(r[1][2][2]), "=&v"(r[1][2][3]), "=&v"(r[1][3][0]), "=&v"(r[1][3][1]), "=&v"(r[1][3][2]), "=&v"(r[1][3][3])
      : "v"(p), "v"(p ^ 64u), "v"(q), "v"(q ^ 64u)
      : "memory");
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    ph[b] = __builtin_bit_cast(f16x8, make_uint4(r[0][b][0].x, r[0][b][0].y, r[0][b][1].x, r[0][b][1].y));
    pl[b] = __builtin_bit_cast(f16x8, make_uint4(r[0][b][2].x, r[0][b][2].y, r[0][b][3].x, r[0][b][3].y));
    qh[b] = __builtin_bit_cast(f16x8, make_uint4(r[1][b][0].x, r[1][b][0].y, r[1][b][1].x, r[1][b][1].y));
    ql[b] = __builtin_bit_cast(f16x8, make_uint4(r[1][b][2].x, r[1][b][2].y, r[1][b][3].x, r[1][b][3].y));
  }
}

// One TT x TT tile of a product on planes, C[i][j] = sum_l P(i, l) Q(j, l).  G groups, each with every G-th stage, of four waves of TT/2 x
// TT/2; two fetch P and two fetch Q by LDS DMA, STAGES - 1 of the group's stages ahead.  A stage is 32 deep: of A A and B X, where l runs
// along the operands' rows, a column of TT/16 blocks of each; of X X^T, where l runs down the rows of X^T, two rows of TT/32 blocks, whose
// fragments (8 l of one column per lane) are two ds_read_b64_tr_b16 each: a 16-lane group hands over 4 rows x 16 columns turned.
// Bound by the matrix pipes and what keeps them waiting at the barriers (busy 0.65-0.72 of the time): 4096 x 4096 A 194 us, 1 100 TFLOP/s on
// planes (diagonal tiles whole); A A 200, 1 060; B X 329, 1 250, the last one 344, 1 200; the library's fp16 product of 8192 1 330 beside it.
template <int TT, int STAGES, int G, int PHASE, typename TO, bool MUON>
__global__ void __launch_bounds__(256 * G) k_ns_product(Jobs jobs, Last<PHASE> to, Muon<MUON> mu, int step, float ca, float cb, float cc) {
  constexpr int MI = TT / 32, OPER = TT * kBK * 4, STAGE = 2 * OPER, NJ = TT / 16;
  constexpr int LDT = TT + 4;  // floats per row of the epilogue's tile: 16-byte rows, neighbours four banks apart
  extern __shared__ __align__(16) char smem[];
  const int in_parts = jobs.split * jobs.parts;  // workgroups of them, in front
  const bool split = (int)blockIdx.x < in_parts;
  const int b = split ? (int)blockIdx.x / jobs.parts : jobs.split + xcd_remap(blockIdx.x - in_parts, jobs.blocks - in_parts, jobs.xcds);
  const Job job = find_job(jobs, b);
  const int j = (int)job.slot;
  const int k = job.k, n = job.n;
  const Layout l = layout_of(k, n);
  char* base = jobs.ws + job.off;
  int ti, tj;
  tile_at(b - job.first, (k + TT - 1) / TT, ((PHASE <= kPoly ? k : n) + TT - 1) / TT, PHASE <= kPoly, ti, tj);
  const int* exps = reinterpret_cast<const int*>(base + kExps);
  const int eX = exps[step], eA = exps[kExpRow + step], eB = exps[2 * kExpRow + step], eY = exps[step + 1];
  const int64_t xt_in = step & 1 ? l.xt1 : l.xt0, xt_out = step & 1 ? l.xt0 : l.xt1;
  const _Float16* XT = reinterpret_cast<const _Float16*>(base + xt_in);
  const int group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), wave = (threadIdx.x >> 6) & 3, lane = threadIdx.x & 63;
  const int i0 = ti * TT, j0 = tj * TT, ldk = (int)l.ldk;

  // the wave's DMA pieces: 1 KB each, NJ of its half of P (waves 0, 1) or Q (waves 2, 3)
  const _Float16* src;
  uint32_t offs[NJ];  // in halfs; blocks beyond the matrix's last are that one again (the results are not stored)
  int64_t advance;    // per stage
  int nk;
  const int from = wave < 2 ? i0 : j0;
  if constexpr (PHASE == kGram) {
    src = XT;
    nk = (n + kBK - 1) / kBK;  // (k_ns_apply leaves rows behind the last strip as they are)
    advance = 2 * kBlockHalfs;
#pragma unroll
    for (int q = 0; q < NJ; ++q)  // wave 0 / 2: the first row of blocks, 1 / 3: the second
      offs[q] = (uint32_t)(min(from / 32 + (q >> 1), ldk / 32 - 1) * ((int)l.rows / 16) + (wave & 1)) * kBlockHalfs + (q & 1) * (kBlockHalfs / 2) + lane * 8;
  } else {
    const _Float16* P = reinterpret_cast<const _Float16*>(base + (PHASE == kPoly ? l.a : l.b));
    src = wave < 2 || PHASE == kPoly ? P : XT;
    const int down = (wave < 2 || PHASE == kPoly ? ldk : (int)l.rows) / 16;
    nk = ldk / kBK;
    advance = (int64_t)down * kBlockHalfs;
#pragma unroll
    for (int q = 0; q < NJ; ++q) {
      const int x = (wave & 1) * NJ + q;
      offs[q] = (uint32_t)(min(from / 16 + (x >> 1), down - 1) * kBlockHalfs + (x & 1) * (kBlockHalfs / 2) + lane * 8);
    }
  }
  auto issue = [&](int t) {
    if (t * G + group >= nk) return;
    char* dst = smem + (t % STAGES * G + group) * STAGE + wave * (OPER / 2);
#pragma unroll
    for (int q = 0; q < NJ; ++q)
      __builtin_amdgcn_global_load_lds(PGNN_GPTR(src + (size_t)offs[q] + (size_t)(t * G + group) * advance), PGNN_LPTR(dst + q * 1024), 16, 0, 0);
  };

  // the epilogue's operand (A behind A A, X^T behind B X) at this thread's pieces of the tile, fetched in front of everything else: its
  // round trip to memory hides behind the product
  constexpr int MINE = TT * TT / 8 / (256 * G);  // pieces of eight columns per thread
  const int out_rows = PHASE <= kPoly ? ldk : (int)l.rows;
  [[maybe_unused]] f16x8 eh[MINE], el[MINE];
  [[maybe_unused]] auto fetch_operand = [&]() {
    const _Float16* E = PHASE == kPoly ? reinterpret_cast<const _Float16*>(base + l.a) : XT;
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      int r, c;
      piece_of<TT>(q * 256 * G + threadIdx.x, r, c);
      const int64_t at = piece_at(out_rows, min(j0 + r, out_rows - 1), min(i0 + c, ldk - 8));
      eh[q] = *reinterpret_cast<const f16x8*>(E + at);
      el[q] = *reinterpret_cast<const f16x8*>(E + at + kBlockHalfs / 2);
    }
  };
  if constexpr (PHASE != kGram) {
    if (!split) fetch_operand();
  }
  if (split) {  // this workgroup's share of the contraction
    const int part = blockIdx.x % jobs.parts, k0 = (int)((int64_t)nk * part / jobs.parts);
    nk = (int)((int64_t)nk * (part + 1) / jobs.parts) - k0;
    src += k0 * advance;
  }

  const int wi = (wave >> 1) * (TT / 2), wj = (wave & 1) * (TT / 2);
  const int fr = lane & 15, fc = lane >> 4;
  // byte offsets of the lane's fragments inside a stage: block a of the wave's rows i and of its rows j (X X^T: of its columns)
  uint32_t pat[MI], qat[MI];
#pragma unroll
  for (int a = 0; a < MI; ++a) {
    const int pb = wi / 16 + a, qb = wj / 16 + a;
    if constexpr (PHASE == kGram) {  // row l = 8 fc + fr / 4, columns 4 (fr & 3) .. of the 16: unit 2 (block & 1) + (fr & 3) / 2 of that row
      auto at = [&](int block) {
        const int u = 2 * (block & 1) + ((fr & 3) >> 1);
        return (uint32_t)(((fc >> 1) * (TT / 16) + (block >> 1) * 2) * 1024 + unit_of(8 * (fc & 1) + (fr >> 2), u) * 16 + (fr & 1) * 8);
      };
      pat[a] = at(pb);
      qat[a] = at(qb) + OPER;
    } else {
      pat[a] = (uint32_t)(pb * 2048 + unit_of(fr, fc) * 16);
      qat[a] = (uint32_t)(qb * 2048 + unit_of(fr, fc) * 16 + OPER);
    }
  }

  f32x4 acc[MI][MI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < MI; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) issue(t);
  for (int t = 0; t * G < nk; ++t) {
    // stage t has landed; behind the barrier every wave's part of it has, and every wave is done with the buffer refilled below
    if ((t + STAGES - 2) * G + group < nk) gemm_wait_vmcnt_imm<(STAGES - 2) * NJ>();
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (G > 1 && t * G + group >= nk) break;  // (an odd number of stages: the last round is the first group's; no barrier follows in the loop)
    const char* st = smem + (t % STAGES * G + group) * STAGE;
    f16x8 ph[MI], pl[MI], qh[MI], ql[MI];
    if constexpr (PHASE == kGram) {
      const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)st;
      if constexpr (MI == 2) {
        f16x8 h[4], lo[4];
        read_turned({at + pat[0], at + pat[1], at + qat[0], at + qat[1]}, h, lo);
#pragma unroll
        for (int a = 0; a < 2; ++a) { ph[a] = h[a]; pl[a] = lo[a]; qh[a] = h[2 + a]; ql[a] = lo[2 + a]; }
      } else {
        static_assert(MI == 2 || MI == 4, "");
        read_turned8(at + pat[0], at + qat[0], ph, pl, qh, ql);
      }
    } else {
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        ph[a] = *reinterpret_cast<const f16x8*>(st + pat[a]);
        pl[a] = *reinterpret_cast<const f16x8*>(st + pat[a] + 1024);
      }
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        ql[a] = *reinterpret_cast<const f16x8*>(st + qat[a] + 1024);
        qh[a] = *reinterpret_cast<const f16x8*>(st + qat[a]);
      }
    }
    // The stage that follows is asked for behind the fragments' reads, which would wait in the same queue, and the wave at its products goes
    // before the one beside it that waits for LDS (4096 x 4096 3830 -> 3680 -> 3650 us, 2301 x 1111 346 -> 313 -> 315)
    issue(t + STAGES - 1);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int c = 0; c < MI; ++c) {  // smallest terms first
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], ql[c], acc[a][c], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a], qh[c], acc[a][c], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < MI; ++a) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], qh[c], acc[a][c], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    asm volatile("" ::: "memory");
  }

  // the second group's sums to the first, through LDS
  if constexpr (G > 1) {
    __syncthreads();
    f32x4* hand = reinterpret_cast<f32x4*>(smem) + (threadIdx.x & 255);
    if (group) {
#pragma unroll
      for (int e = 0; e < MI * MI; ++e) hand[e * 256] = acc[e / MI][e % MI];
    }
    __syncthreads();
    if (!group) {
#pragma unroll
      for (int e = 0; e < MI * MI; ++e) acc[e / MI][e % MI] += hand[e * 256];
    }
  }

  // a tile in parts: each part's sums go to memory that the launch does not use otherwise (the X^T to come, behind B X what was A), and
  // the part that arrives last adds all of them up in their own order and goes on as if it had formed the whole tile
  if (split) {
    uint64_t* mem = reinterpret_cast<uint64_t*>(base + (PHASE <= kPoly ? xt_out : l.a)) + (int64_t)(b - job.first) * jobs.parts * (TT * TT / 2) + (threadIdx.x & 255);
    uint64_t* mine = mem + (int64_t)(blockIdx.x % jobs.parts) * (TT * TT / 2);
    if (!group) {
#pragma unroll
      for (int e = 0; e < MI * MI; ++e) {
        const uint4 w = __builtin_bit_cast(uint4, acc[e / MI][e % MI]);
        publish(mine + e * 512, (uint64_t)w.y << 32 | w.x);
        publish(mine + e * 512 + 256, (uint64_t)w.w << 32 | w.z);
      }
      publish_commit();
    }
    __syncthreads();
    unsigned* ticket = reinterpret_cast<unsigned*>(base + kTickets) + (b - job.first);
    if (threadIdx.x == 0) {
      const bool last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)jobs.parts - 1u;
      if (last) publish(ticket, 0u);
      *reinterpret_cast<int*>(smem) = last;
    }
    __syncthreads();
    if (!*reinterpret_cast<int*>(smem)) return;
    asm volatile("" ::: "memory");
    for (int part = 0; part < jobs.parts && !group; ++part) {
      const uint64_t* from_part = mem + (int64_t)part * (TT * TT / 2);
      uint64_t w[MI * MI][2];
#pragma unroll
      for (int e = 0; e < MI * MI; ++e) {
        w[e][0] = fetch_published(from_part + e * 512);
        w[e][1] = fetch_published(from_part + e * 512 + 256);
      }
#pragma unroll
      for (int e = 0; e < MI * MI; ++e) {
        const f32x4 v = __builtin_bit_cast(f32x4, make_uint4((uint32_t)w[e][0], (uint32_t)(w[e][0] >> 32), (uint32_t)w[e][1], (uint32_t)(w[e][1] >> 32)));
        f32x4& sum = acc[e / MI][e % MI];
        sum = part == 0 ? v : sum + v;
      }
    }
    if constexpr (PHASE != kGram) fetch_operand();
  }

  // epilogue: the tile to LDS as fp32 [j][i] (a lane holds four consecutive i of one j), out row by row as the operand lies (rows j),
  // and once more turned (rows i) where the mirror image of a symmetric tile or a wide G wants it
  __syncthreads();
  float* tile = reinterpret_cast<float*>(smem);
  const float f = PHASE == kGram ? ldexpf(1.f, eA - 2 * eX) : PHASE == kPoly ? ldexpf(cc, eB - 2 * eA)
                : PHASE == kApply ? ldexpf(1.f, eY - eX - eB) : ldexpf(1.f, -eX - eB);
  const float fe = PHASE == kPoly ? ldexpf(cb, eB - eA) : PHASE == kApply ? ldexpf(ca, eY - eX) : ldexpf(ca, -eX);
  if (!group) {
#pragma unroll
    for (int a = 0; a < MI; ++a)
#pragma unroll
      for (int c = 0; c < MI; ++c)
        *reinterpret_cast<f32x4*>(tile + (wj + c * 16 + fr) * LDT + wi + a * 16 + fc * 4) = acc[a][c] * f;
  }
  __syncthreads();

  auto planes_out = [&](_Float16* d, int r, int c, const float (&v)[8]) {
    f16x8 h, lo;
    split8(v, h, lo);
    const int64_t at = piece_at(out_rows, r, c);
    *reinterpret_cast<f16x8*>(d + at) = h;
    *reinterpret_cast<f16x8*>(d + at + kBlockHalfs / 2) = lo;
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
        for (int e = 0; e < 8; ++e)
          if (e < m) {
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
    int r, c;
    piece_of<TT>(q * 256 * G + threadIdx.x, r, c);
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
        planes_out(D, j0 + r, i0 + c, v);
      }
    } else if (!again && j0 + r < n) {
      result_out((int64_t)(j0 + r) * k + i0 + c, k - (i0 + c), v);
    }
  }
  if (!again) return;
  if constexpr (PHASE != kGram) __syncthreads();
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    int r, c;
    piece_of<TT>(q * 256 * G + threadIdx.x, r, c);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(c + e) * LDT + r];
    if constexpr (PHASE <= kPoly) {
      if (i0 + r < k && j0 + c < ldk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = j0 + c + e < k ? v[e] : 0.f;
        planes_out(D, i0 + r, j0 + c, v);
      }
    } else {
      if (i0 + r < k) result_out((int64_t)(i0 + r) * n + j0 + c, n - (j0 + c), v);
    }
  }
}

// The second half of a step for small k in one launch: X <- a X + A Z, Z = b X + c A X, a strip of 32 rows of X^T per workgroup (one row of
// X^T knows nothing of another, so the two products need no exchange between workgroups; B = b A + c A A would, and one more launch).  It
// costs 4 k^2 n instead of 2 k^3 + 2 k^2 n operations, which a small matrix has to spare: its launches are bound by their latency.  k <=
// kSmall takes it (against B and B X; us for the whole iteration: 100 x 200 73 and 87, sixteen 128 x 2048 158 and 164, 200 x
// 200 94 and 99, four 256 x 512 111 and 120, 300 x 600 124 and 122, ten of them 136 and 137, the Muon step of a 5-layer network of such weights
// 144.5 and 145.5; 384 x 384 130 and 118).
// The strip and Z lie in LDS, A streams from L2 straight into registers -- every wave
// takes whole 16-row blocks of A, so nothing of A is read twice by a workgroup -- RING pairs of 32-deep steps ahead; the strip's
// fragments of a pair are read from LDS while the pair before it multiplies.  A lane's four results
// are four consecutive columns of one row of X^T: they go to LDS as they are, and the strip leaves in whole rows.
// Ten 300 x 600: 17.8 us, 0.33 of the matrix pipes: A's way from L2 into each CU (410 KB, twice) and the chain of loads in front.
constexpr int kStrip = 32, kSmall = 320;

template <int RING, bool LAST, typename TO, bool MUON>
__global__ void __launch_bounds__(512) k_ns_apply(Jobs jobs, Last<LAST ? kLast : kApply> to, Muon<MUON> mu, int step, float ca, float cb, float cc) {
  extern __shared__ __align__(16) char smem[];
  const int b = xcd_remap(blockIdx.x, jobs.blocks, jobs.xcds);
  const Job job = find_job(jobs, b);
  const int k = job.k, n = job.n;
  const Layout l = layout_of(k, n);
  char* base = jobs.ws + job.off;
  const int j0 = (b - job.first) * kStrip, ldk = (int)l.ldk, down = (int)l.rows / 16;
  const int* exps = reinterpret_cast<const int*>(base + kExps);
  const int eX = exps[step], eA = exps[kExpRow + step], eZ = exps[3 * kExpRow + step], eY = exps[step + 1];
  const _Float16* XT = reinterpret_cast<const _Float16*>(base + (step & 1 ? l.xt1 : l.xt0));
  const _Float16* A = reinterpret_cast<const _Float16*>(base + l.a);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, nwaves = blockDim.x >> 6;
  char* const strip = smem;
  char* const zed = smem + kStrip * ldk * 4;

  // the strip by DMA: 4 KB of each column of blocks
  const _Float16* from = XT + (int64_t)(j0 / 16) * kBlockHalfs + lane * 8;
  for (int q = wave; q < ldk / 8; q += nwaves)
    __builtin_amdgcn_global_load_lds(PGNN_GPTR(from + (int64_t)(q >> 2) * down * kBlockHalfs + (q & 3) * 512), PGNN_LPTR(strip + q * 1024), 16, 0, 0);
  const int fr = lane & 15, fc = lane >> 4;
  const int pairs = ldk / 64;                                              // of 32-deep steps
  const int blocks = wave < ldk / 16 ? (ldk / 16 - wave + nwaves - 1) / nwaves : 0;  // 16-row blocks of A for this wave
  const int total = blocks * pairs;
  f16x8 ring[RING][4];  // high and low plane of two steps
  int fblk = 0, fpr = 0;  // the next pair to fetch.  Past the end it stays on the last one: a load that is always issued leaves hipcc its count
  auto fetch = [&](f16x8 (&d)[4]) {
    const _Float16* s = A + ((int64_t)fpr * 2 * (ldk / 16) + min(wave + fblk * nwaves, ldk / 16 - 1)) * kBlockHalfs + unit_of(fr, fc) * 8;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = *reinterpret_cast<const f16x8*>(s + (int64_t)(e >> 1) * (ldk / 16) * kBlockHalfs + 512 * (e & 1));
    if (fpr + 1 < pairs) {
      ++fpr;
    } else if (fblk + 1 < blocks) {
      ++fblk;
      fpr = 0;
    }
  };
  auto prime = [&]() {
    fblk = fpr = 0;
#pragma unroll
    for (int q = 0; q < RING; ++q) fetch(ring[q]);
  };
  // C[i][j] = sum_l A[i][l] op[j][l] for the wave's blocks of rows i; done(i0, acc) per block
  auto product = [&](const char* op, auto done) {
    f32x4 big[2], cross[2];  // high x high, and the two small terms: twice as many chains of dependent MFMAs
#pragma unroll
    for (int c = 0; c < 2; ++c) big[c] = cross[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    f16x8 of[2][8];  // fragments of the strip for a pair: [step][block of 16][plane]
    auto read = [&](int pr, f16x8 (&d)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = *reinterpret_cast<const f16x8*>(op + (pr * 4 + (e >> 1)) * 2048 + (e & 1) * 1024 + unit_of(fr, fc) * 16);
    };
    int blk = 0, pr = 0;
    read(0, of[0]);
    for (int at0 = 0; at0 < total; at0 += RING) {
#pragma unroll
      for (int q = 0; q < RING; ++q) {
        const int next = pr + 1 == pairs ? 0 : pr + 1;
        read(next, of[(q + 1) & 1]);
        const f16x8 (&f)[8] = of[q & 1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 2; ++c) cross[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[q][2 * h], f[4 * h + 2 * c + 1], cross[c], 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 2; ++c) big[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[q][2 * h], f[4 * h + 2 * c], big[c], 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 2; ++c) cross[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[q][2 * h + 1], f[4 * h + 2 * c], cross[c], 0, 0, 0);
        }
        fetch(ring[q]);
        // (a whole ring is always run, the last one's surplus into nothing: with a way out between the slots hipcc waits for every load
        // in flight at the head of the loop)
        if (next == 0) {
          big[0] += cross[0];
          big[1] += cross[1];
          if (blk < blocks) done((wave + blk * nwaves) * 16, big);
#pragma unroll
          for (int c = 0; c < 2; ++c) big[c] = cross[c] = f32x4{0.f, 0.f, 0.f, 0.f};
          ++blk;
        }
        pr = next;
      }
    }
  };
  // the lane's four columns i .. i + 3 of row r of an LDS operand
  auto quad = [&](char* op, int r, int i, int low) {
    return op + ((i >> 5) * 2 + (r >> 4)) * 2048 + low * 1024 + unit_of(r & 15, (i >> 3) & 3) * 16 + (i & 7) * 2;
  };
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  auto x_at = [&](int r, int i, float (&x)[4]) {
    const f16x4 h = *reinterpret_cast<const f16x4*>(quad(strip, r, i, 0)), lo = *reinterpret_cast<const f16x4*>(quad(strip, r, i, 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float)h[e] + (float)lo[e];
  };
  auto put = [&](char* op, int r, int i, const float (&v)[4]) {
    uint32_t h[2], lo[2];
    split2(i < k ? v[0] : 0.f, i + 1 < k ? v[1] : 0.f, h[0], lo[0]);
    split2(i + 2 < k ? v[2] : 0.f, i + 3 < k ? v[3] : 0.f, h[1], lo[1]);
    *reinterpret_cast<uint2*>(quad(op, r, i, 0)) = make_uint2(h[0], h[1]);
    *reinterpret_cast<uint2*>(quad(op, r, i, 1)) = make_uint2(lo[0], lo[1]);
  };

  prime();
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the strip (and the first of A); the builtin, which hipcc counts along with
  __syncthreads();
  {
    const float fy = ldexpf(cc, eZ - eA - eX), fx = ldexpf(cb, eZ - eX);
    product(strip, [&](int i0, const f32x4 (&acc)[2]) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = c * 16 + fr, i = i0 + 4 * fc;
        float x[4], z[4];
        x_at(r, i, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = fmaf(fx, x[e], acc[c][e] * fy);
        put(zed, r, i, z);
      }
    });
  }
  prime();
  __syncthreads();
  const float fy = ldexpf(1.f, (LAST ? 0 : eY) - eA - eZ), fx = ldexpf(ca, (LAST ? 0 : eY) - eX);
  product(zed, [&](int i0, const f32x4 (&acc)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = c * 16 + fr, i = i0 + 4 * fc;
      float x[4], v[4];
      x_at(r, i, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(fx, x[e], acc[c][e] * fy);
      if constexpr (!LAST) {
        put(strip, r, i, v);  // nobody else reads these four any more
      } else if (j0 + r < n) {
        const int64_t at = job.tall ? (int64_t)(j0 + r) * k + i : (int64_t)i * n + j0 + r, next = job.tall ? 1 : n;
        TO* d = static_cast<TO*>(to.dst[job.slot]) + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i + e >= k) break;
          if constexpr (MUON) d[e * next] = fmaf(-mu.rate[job.slot], v[e], d[e * next] * mu.keep);
          else d[e * next] = (TO)v[e];
        }
      }
    }
  });
  if constexpr (!LAST) {
    __syncthreads();
    _Float16* out = reinterpret_cast<_Float16*>(base + (step & 1 ? l.xt0 : l.xt1));
    f16x8* d = reinterpret_cast<f16x8*>(out + (int64_t)(j0 / 16) * kBlockHalfs);
    for (int q = threadIdx.x; q < kStrip * ldk / 4; q += blockDim.x)
      d[(int64_t)(q >> 8) * down * (kBlockHalfs / 8) + (q & 255)] = reinterpret_cast<const f16x8*>(strip)[q];
  }
}

// The whole iteration of one small matrix (k <= kTinyK, n <= kTinyN) in one workgroup, X^T, A and Z in LDS: no launch but this one.  Gram:
// waves 0-3 and 4-7 each form A's 64 x 64 over every other 32 rows of X^T, the second four hand theirs over through LDS.  Then a wave takes
// whole 16-row blocks of X^T, whose new rows depend on nothing but themselves and A: Z = b X + c A X into scratch of its own, X <- a X + A Z
// back in place, no barrier between.  Every sum is taken in the order of the kernels above where a launch of theirs is small.
// Latency throughout: a call of 16 x 16 takes 18 us (the launches above 55), 64 x 64 20 (52), 384 x 64 63 (69).
constexpr int kTinyK = 64, kTinyN = 384;

template <typename T, bool MUON>
__global__ void __launch_bounds__(512) k_ns_tiny(Jobs jobs, Sources from, Results to, Muon<MUON> mu, Bounds bd) {
  extern __shared__ __align__(16) char smem[];  // (alone: read_turned flips bit 6 of its addresses, so LDS begins with the blocks)
  const Job job = jobs.job[blockIdx.x];
  const int j = (int)job.slot;
  const int k = job.k, n = job.n, np = (n + 31) & ~31, down = np / 16;
  const bool tall = job.tall;
  const int rows = tall ? n : k, cols = tall ? k : n;
  char* const xt = smem;                  // blocks [2][down][planes]
  char* const am = smem + np * 256;       // blocks [2][4][planes]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, fr = lane & 15, fc = lane >> 4;
  char* const zed = am + 16384 + wave * 4096;  // blocks [2][planes], of this wave alone
  double* const red = reinterpret_cast<double*>(am);
  const T* g = static_cast<const T*>(from.src[j]);
  const int64_t ld = from.ld[j];

  // eight elements of the thread on their way at a time; row of element e by a multiplication (e cols < 2^32 / cols: exact)
  const uint32_t magic = (uint32_t)((0xffffffffull + cols) / cols);
  const int total = rows * cols;
  auto row_of = [&](int e) { return cols == 1 ? e : (int)__umulhi((uint32_t)e, magic); };
  auto load8 = [&](int e0, float (&v)[8], float (&m)[8]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int e = min(e0 + 512 * q, total - 1), r = row_of(e);
      v[q] = (float)g[r * ld + (e - r * cols)];
      if constexpr (MUON) m[q] = mu.momentum[j][e];
    }
  };
  // the norm by the same sums as k_ns_norm and k_ns_split: waves 0-3 and 4-7 take a part each
  const int nparts = parts_of(k, n);
  for (int part = wave >> 2; part < nparts; part += 2) {
    const double s = squares<T, MUON>(job, part, threadIdx.x & 255, from, mu);
    if (lane == 0) red[part * 4 + (wave & 3)] = s;
  }
  for (int e = threadIdx.x; e < np * 16; e += 512) reinterpret_cast<uint4*>(xt)[e] = make_uint4(0, 0, 0, 0);  // rows n .., columns k ..
  __syncthreads();
  double s = lane < nparts ? (red[lane * 4] + red[lane * 4 + 1]) + (red[lane * 4 + 2] + red[lane * 4 + 3]) : 0.0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  const double norm = sqrt(s);
  int shift;
  const float inv = inverse(norm, bd.eps, shift);
  float u = first_bound(bd, norm);
  int eX = plane_exponent(u);
  shift += eX;
  for (int e0 = threadIdx.x; e0 < total; e0 += 8 * 512) {
    float v[8], m[8];  // (the momentum: what the workgroup has just written, behind a barrier)
    load8(e0, v, m);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int e = e0 + 512 * q, r = row_of(e), c = e - r * cols;
      if (e >= total) continue;
      if constexpr (MUON) v[q] = mu.nesterov ? fmaf(mu.mu, m[q], v[q]) : m[q];
      const float x = scaled(v[q], shift, inv);
      const _Float16 h = (_Float16)x;
      _Float16* d = reinterpret_cast<_Float16*>(xt) + piece_at(np, tall ? r : c, (tall ? c : r) & ~7) + ((tall ? c : r) & 7);
      d[0] = h;
      d[kBlockHalfs / 2] = (_Float16)low_part(x, h);
    }
  }
  __syncthreads();

  const uint32_t xt_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)xt;
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  auto frag = [&](const char* block) { return *reinterpret_cast<const f16x8*>(block + unit_of(fr, fc) * 16); };
  // four columns i .. i + 3 of row r inside a column of blocks of `d` blocks each
  auto quad = [&](char* m, int d, int r, int i) { return m + ((i >> 5) * d + (r >> 4)) * 2048 + unit_of(r & 15, (i >> 3) & 3) * 16 + (i & 7) * 2; };
  auto put = [&](char* at, const float (&v)[4]) {
    uint32_t h[2], lo[2];
    split2(v[0], v[1], h[0], lo[0]);
    split2(v[2], v[3], h[1], lo[1]);
    *reinterpret_cast<uint2*>(at) = make_uint2(h[0], h[1]);
    *reinterpret_cast<uint2*>(at + 1024) = make_uint2(lo[0], lo[1]);
  };
  // acc[a] = (rows 16 a .. of A) . (16 rows of op)^T; op's blocks: column of blocks h at op + h * stride
  auto by_a = [&](const char* op, int stride, f32x4 (&acc)[4]) {
    f32x4 cross[4];  // (the terms in the order of k_ns_apply)
#pragma unroll
    for (int a = 0; a < 4; ++a) acc[a] = cross[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f16x8 oh = frag(op + h * stride), ol = frag(op + h * stride + 1024);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f16x8 ah = frag(am + (h * 4 + a) * 2048), alow = frag(am + (h * 4 + a) * 2048 + 1024);
        cross[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, ol, cross[a], 0, 0, 0);
        acc[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, oh, acc[a], 0, 0, 0);
        cross[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(alow, oh, cross[a], 0, 0, 0);
      }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) acc[a] += cross[a];
  };
  for (int t = 0; t < bd.steps; ++t) {
    const StepExps ex = step_bounds(bd, t, u);
    const float ca = bd.coef[t][0], cb = bd.coef[t][1], cc = bd.coef[t][2];
    {  // A = X X^T
      const int pb = (wave >> 1 & 1) * 2, qb = (wave & 1) * 2, half = wave >> 2;
      f32x4 acc[2][2];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto at = [&](int block) {  // row l = 8 fc + fr / 4, columns 4 (fr & 3) .. of block's 16
        const int unit = 2 * (block & 1) + ((fr & 3) >> 1);
        return xt_at + (uint32_t)(((block >> 1) * down + (fc >> 1)) * 2048 + unit_of(8 * (fc & 1) + (fr >> 2), unit) * 16 + (fr & 1) * 8);
      };
      for (int st = half; st < np / 32; st += 2) {
        f16x8 h[4], lo[4];
        const uint32_t o = (uint32_t)st * 4096;
        read_turned({at(pb) + o, at(pb + 1) + o, at(qb) + o, at(qb + 1) + o}, h, lo);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[a], lo[2 + c], acc[a][c], 0, 0, 0);
            acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[a], h[2 + c], acc[a][c], 0, 0, 0);
            acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[a], h[2 + c], acc[a][c], 0, 0, 0);
          }
      }
      f32x4* other = reinterpret_cast<f32x4*>(am + 16384 + (wave & 3) * 4096) + lane;  // (the first four waves' scratch: idle here)
      if (half) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int c = 0; c < 2; ++c) other[(a * 2 + c) * 64] = acc[a][c];
      }
      __syncthreads();
      if (!half) {
        const float f = ldexpf(1.f, ex.a - 2 * eX);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const f32x4 v = (acc[a][c] + other[(a * 2 + c) * 64]) * f;
            put(quad(am, 4, (qb + c) * 16 + fr, (pb + a) * 16 + 4 * fc), {v[0], v[1], v[2], v[3]});
          }
      }
      __syncthreads();
    }
    const bool last = t + 1 == bd.steps;
    const float fz = ldexpf(cc, ex.z - ex.a - eX), fzx = ldexpf(cb, ex.z - eX);
    const int ey = last ? 0 : ex.y;
    const float fy = ldexpf(1.f, ey - ex.a - ex.z), fyx = ldexpf(ca, ey - eX);
    for (int blk = wave; blk < down; blk += 8) {
      float x[4][4];
      f32x4 acc[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const char* q = quad(xt, down, blk * 16 + fr, a * 16 + 4 * fc);
        const f16x4 h = *reinterpret_cast<const f16x4*>(q), lo = *reinterpret_cast<const f16x4*>(q + 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[a][e] = (float)h[e] + (float)lo[e];
      }
      by_a(xt + blk * 2048, down * 2048, acc);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = fmaf(fzx, x[a][e], acc[a][e] * fz);
        put(quad(zed, 1, fr, a * 16 + 4 * fc), z);
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): Z is whole before any lane of the wave reads it
      asm volatile("" ::: "memory");
      by_a(zed, 2048, acc);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(fyx, x[a][e], acc[a][e] * fy);
        const int r = blk * 16 + fr, i = a * 16 + 4 * fc;
        if (!last) {
          put(quad(xt, down, r, i), v);
        } else if (r < n) {
          const int64_t at = tall ? (int64_t)r * k + i : (int64_t)i * n + r, next = tall ? 1 : n;
          T* d = static_cast<T*>(to.dst[j]) + at;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < k) {
              if constexpr (MUON) d[e * next] = fmaf(-mu.rate[j], v[e], d[e * next] * mu.keep);
              else d[e * next] = (T)v[e];
            }
        }
      }
    }
    eX = ex.y;
    __syncthreads();
  }
}

constexpr int kPartStages = 8, kMaxTileParts = 16;  // a part is at least 8 stages deep (16: 1500 x 1500 452 instead of 425 us, two 2048 x 2048 1138 instead of 1153; 4: 2048 x 2048 742 instead of 713)

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

// A CU's matrix cores are busy with one tile, so a launch takes the time of ceil(tiles / CUs) tiles one after the other: what is left over a
// multiple of the CUs' number is formed in as many parts as give every CU one.  They stand in front of the launch, so that their sums meet
// while the CUs work on whole tiles.  4096 x 4096 (528 tiles of A, 16 left over on 256 CUs, in 16 parts) 4255 -> 3692 us; with two or three
// parts to a tile the way through memory costs more than it saves beside whole tiles (ten 1024 x 2048, 104 left over: 1261 -> 1321).
template <int TT, int PHASE>
void split_rest(Jobs& jobs) {
  const int rest = jobs.blocks % num_cu();
  jobs.split = 0;
  jobs.parts = 1;
  if (rest == 0 || rest > kMaxSplit) return;
  int64_t parts = std::min(num_cu() / rest, kMaxTileParts);
  for (int j = 0; j < jobs.count && jobs.job[j].first < rest; ++j) {
    const Job& q = jobs.job[j];
    const Layout l = layout_of(q.k, q.n);
    const int tiles = std::min(rest, j + 1 < jobs.count ? jobs.job[j + 1].first : jobs.blocks) - q.first;
    if (tiles == 0) continue;
    const int64_t room = 4 * l.ldk * (PHASE <= kPoly ? l.rows : l.ldk), stages = (PHASE == kGram ? q.n : q.k) / kBK;
    parts = std::min(std::min(parts, room / ((int64_t)tiles * TT * TT * 4)), stages / kPartStages);
  }
  if (parts < (rest == jobs.blocks ? 2 : 4)) return;
  jobs.split = rest;
  jobs.parts = (int)parts;
  jobs.blocks += rest * (jobs.parts - 1);
}

template <int TT, int STAGES, int G, int PHASE, typename TO, bool MUON>
void launch_product(Jobs& jobs, const Last<PHASE>& to, const Muon<MUON>& mu, int step, const float* c, hipStream_t st) {
  place(jobs, [](const Job& q) { return tiles_of<TT>(q.k, q.n, PHASE <= kPoly); });
  split_rest<TT, PHASE>(jobs);
  constexpr size_t lds = std::max<size_t>((size_t)STAGES * G * 2 * TT * kBK * 4, (size_t)TT * (TT + 4) * 4);
  const void* fn = (const void*)k_ns_product<TT, STAGES, G, PHASE, TO, MUON>;
  allow_big_lds(fn, lds);
  hipLaunchKernelGGL((k_ns_product<TT, STAGES, G, PHASE, TO, MUON>), dim3(jobs.blocks), dim3(256 * G), lds, st, jobs, to, mu, step, c[0], c[1], c[2]);
}

template <int RING, bool LAST, typename TO, bool MUON>
void launch_apply(Jobs& jobs, const Last<LAST ? kLast : kApply>& to, const Muon<MUON>& mu, int step, const float* c, int most, hipStream_t st) {
  place(jobs, [](const Job& q) { return (int)ceil_div(q.n, kStrip); });
  const int blocks = (int)layout_of(most, most).ldk / 16, each = (int)ceil_div(blocks, 8), waves = (int)ceil_div(blocks, each);
  const size_t lds = (size_t)layout_of(most, most).ldk * kStrip * 8;
  allow_big_lds((const void*)k_ns_apply<RING, LAST, TO, MUON>, lds);
  hipLaunchKernelGGL((k_ns_apply<RING, LAST, TO, MUON>), dim3(jobs.blocks), dim3(64 * waves), lds, st, jobs, to, mu, step, c[0], c[1], c[2]);
}
template <bool LAST, typename TO, bool MUON>
void apply(Jobs& jobs, const Last<LAST ? kLast : kApply>& to, const Muon<MUON>& mu, int step, const float* c, hipStream_t st) {
  int most = 0;
  for (int j = 0; j < jobs.count; ++j) most = std::max(most, jobs.job[j].k);
  if (most <= 128) launch_apply<2, LAST, TO, MUON>(jobs, to, mu, step, c, most, st);  // a wave has two pairs of steps in all
  else launch_apply<4, LAST, TO, MUON>(jobs, to, mu, step, c, most, st);
}

// Tiles of 64 while three of them per CU take them all at once, else of 128: launches of 640, 648 and 675 tiles of 64 take 15.7, 28.2 and
// 38.4 us, with tiles of 128 17.2, 31.1 and 41.9; launches of 870 and 1024 33.0 and 65.7, with tiles of 128 29.1 and 53.6.
// A wave that is alone on its SIMD waits for the barrier, LDS and the matrix cores one after the other, so a CU wants several:
// - no more tiles than CUs: a tile's stages go to two groups of four waves in turn (tiles of 64: 300 x 600 11.6 -> 10.4 us a launch, 1000 x
//   4096 46 -> 36; of 128: 2048 x 2048 69.7 -> 60.9).  Eight stages in flight for one group changed nothing.
// - up to two tiles of 64 per CU: two groups each, and LDS for two tiles, i.e. two stages per group (four 700 x 800 16.0 -> 14.1, 1300 x 1300
//   22.1 -> 21.2 against one group with four stages).
// - more: LDS for three tiles of one group and three stages (572 and 768 tiles 21.6 -> 18.2 and 36.4 -> 31.7 against four stages, which are
//   two tiles; 441 tiles 22.8, with two groups 21.2; two stages for five tiles: 35.0 for 768, and 32 for 476 instead of 27).
// - tiles of 128: two of one group (ten 1024 x 2048 134 us, with two groups and thus one tile 154).
template <int PHASE, typename TO, bool MUON>
void product(Jobs& jobs, const Last<PHASE>& to, const Muon<MUON>& mu, int step, const float* c, hipStream_t st) {
  int64_t big = 0, small = 0;
  for (int j = 0; j < jobs.count; ++j) {
    big += tiles_of<128>(jobs.job[j].k, jobs.job[j].n, PHASE <= kPoly);
    small += tiles_of<64>(jobs.job[j].k, jobs.job[j].n, PHASE <= kPoly);
  }
  if (small > 3 * num_cu()) {
    if (big > num_cu()) launch_product<128, 2, 1, PHASE, TO, MUON>(jobs, to, mu, step, c, st);
    else launch_product<128, 2, 2, PHASE, TO, MUON>(jobs, to, mu, step, c, st);
  }
  else if (small > 2 * num_cu()) launch_product<64, 3, 1, PHASE, TO, MUON>(jobs, to, mu, step, c, st);
  else if (small > num_cu()) launch_product<64, 2, 2, PHASE, TO, MUON>(jobs, to, mu, step, c, st);
  else launch_product<64, 4, 2, PHASE, TO, MUON>(jobs, to, mu, step, c, st);
}

template <typename T, bool MUON>
void run_chunk(Jobs& jobs, const Sources& from, const Results& to, const Muon<MUON>& mu, const Bounds& bd, hipStream_t st) {
  const Nothing no{0};
  // k_ns_tiny where every matrix of the chunk fits it: beside others in the list its launch would only stand in their way (the list of a
  // 5-layer network, with 3 x 300 among 300 x 600: 153 us without it, 194 with it), and there the small ones cost next to nothing
  int tiny_n = 0;
  for (int j = 0; j < jobs.count && tiny_n >= 0; ++j)
    tiny_n = jobs.job[j].k <= kTinyK && jobs.job[j].n <= kTinyN ? std::max(tiny_n, jobs.job[j].n) : -1;
  if (tiny_n > 0) {
    const size_t lds = (size_t)((tiny_n + 31) & ~31) * 256 + 16384 + 8 * 4096;
    allow_big_lds((const void*)k_ns_tiny<T, MUON>, lds);
    hipLaunchKernelGGL((k_ns_tiny<T, MUON>), dim3(jobs.count), dim3(512), lds, st, jobs, from, to, mu, bd);
    return;
  }
  // few: by k_ns_apply.  Beside larger ones whose tiles leave CUs idle the small ones ride along in their launches instead (five 300 x 300
  // and five 400 x 400 224 -> 153 us); a launch that is full already is better off without them (2048 x 2048 and 119 x 2048 708, together 873)
  int64_t larger = 0;
  for (int j = 0; j < jobs.count; ++j)
    if (jobs.job[j].k > kSmall) larger += tiles_of<128>(jobs.job[j].k, jobs.job[j].n, false);
  const bool together = larger > 0 && larger < num_cu();
  Jobs few{}, many{};
  few.ws = many.ws = jobs.ws;
  few.xcds = many.xcds = jobs.xcds;
  for (int j = 0; j < jobs.count; ++j) {
    Jobs& half = jobs.job[j].k <= kSmall && !together ? few : many;
    half.job[half.count++] = jobs.job[j];
  }
  place(jobs, [](const Job& q) { return parts_of(q.k, q.n); });
  hipLaunchKernelGGL((k_ns_norm<T, MUON>), dim3(jobs.blocks), dim3(256), 0, st, jobs, from, mu);
  place(jobs, [](const Job& q) { return tiles_of<64>(q.k, q.n, false); });
  hipLaunchKernelGGL((k_ns_split<T, MUON>), dim3(jobs.blocks), dim3(256), 0, st, jobs, from, mu, bd);
  for (int t = 0; t < bd.steps; ++t) {
    const bool last = t + 1 == bd.steps;
    const float* c = bd.coef[t];
    product<kGram, float, false>(jobs, no, no, t, c, st);
    if (few.count) {
      if (last) apply<true, T, MUON>(few, to, mu, t, c, st);
      else apply<false, float, false>(few, no, no, t, c, st);
    }
    if (many.count) {
      product<kPoly, float, false>(many, no, no, t, c, st);
      if (last) product<kLast, T, MUON>(many, to, mu, t, c, st);
      else product<kApply, float, false>(many, no, no, t, c, st);
    }
  }
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
      jobs.job[q] = Job{0, (int)std::min(rows[j], cols[j]), (int)std::max(rows[j], cols[j]), rows[j] > cols[j], off, q};
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
