// The Muon step: the update of a matrix is its momentum, orthogonalised by Newton-Schulz products; and the orthogonalisation alone.
//
//   m <- m + (1 - b)(g - m),  u = g + b (m - g) (Nesterov) or m,  X = u / max(|u|_F, eps)
//   per step, on the smaller side:  A = X X^T,  X <- a X + (b A + c A^2) X          (the polynomial a s + b s^3 + c s^5 of each singular value s)
//   p <- p (1 - lr wd) - lr r X
//
// Two forms, by the smaller side n of a matrix.
//
// n <= 64 (factors, adapters): with P = a I + b A + c A^2, X goes to P X and A to P A P, and all of these are polynomials of the first A.  So the steps
// are taken on n x n matrices, and X is touched twice: for A, and for the product of all P with it.  A has the squares of the singular values, and
// noise in its small ones grows by a^2 a step, so this half is in 64 bits (half the rate of 32 on this GPU, and next to nothing beside the memory).  Three
// launches for all such matrices of a call together.  Not for any number of steps: what is noise in A (1e-16, of either sign) must stay small, since a negative square of
// a singular value grows without end, and Q, the product of the P, is applied in fp32.  So X is formed anew, and A from it, before Q could pass 2^10 (kMostGrowth): after
// five steps of a = 3.4445.  (64 x 64 at random, 8 steps: 3e-5 off in one run of steps, 3e-6 in two, fp32 products 4e-6; 16 x 64 of rank one, 20 steps: not a number in one
// run.)  Runs take three launches each.
//
// n > 64: X, A and B = b A + c A^2 are products on the tcgen05 tensor cores.  What is rounded: a value is held as two fp16 numbers (hi + rest, 22 bits)
// times a power of two that the bound on the singular values gives, so that none overflows, and a product is hi hi + hi lo + lo hi; its sums are fp32, at
// most 256 terms in an accumulator (the tensor core cuts sums off: over 4096 terms it loses 3e-5, where fp32 rounding loses 3e-7) and the rest in registers
// (4096 x 4096 against 64 bits: 5.5e-7 with 64 terms, 6.3e-7 with 128, 1.1e-6 with 256, in 3.85 ms with 128 and 3.66 with 256 in turn, 3.7 to 4.0 in others under
// the power cap; fp32 products of a library: 3.6e-6 in 34 ms).  a X is added in fp32 (as part of the product, with a I in B, 5 % faster and two to three times as far off).
// Results of 16 bits are computed the same way and rounded once.  (Products of the hi parts alone are a third of the work, 4096 x 10240 in bfloat16 2.7 ms where these take
// 7.6, but leave X 1e-3 off: a rounding that no caller has asked for, and more than that of fp16 itself.)
// A and B are symmetric: blocks below the diagonal are not computed, the others stored twice.  Either operand is taken in either order, so nothing is
// transposed; where the rows are the longer side A = X^T X and X <- a X + X B.  Matrices of all shapes share their launches.
// Every wait is bounded: one that runs out sets a status word and the CTA leaves through its normal exit.
#include <algorithm>
#include <cmath>
#include <exception>
#include <map>
#include <utility>
#include <vector>

#include <cooperative_groups.h>

#include "common.cuh"
#include "tc_common.cuh"
#include "tc_pair.cuh"
#include "vec_io.cuh"

namespace b200cp {

__device__ int g_muon_status = 0;   // 0 ok; otherwise (code << 16) | (linear block index & 0xffff)

namespace {

namespace cg = cooperative_groups;
using namespace tc;

struct Pointers {   // of one matrix
  void* p;          // what is updated, or receives X
  const void* g;
  float *m, *w;     // momentum (null: u = g), float32 copy (or null)
};
struct Rates {
  float keep, blend;        // b, 1 - b
  int nesterov, update;     // update 0: p receives X itself
  float lr, decay;          // lr, wd
  const float* device_lr;   // or null
  double eps;
};
template <typename G>
__device__ __forceinline__ float momentum_of(const Rates& r, float g, float m) { return fmaf(r.blend, g - m, m); }
__device__ __forceinline__ float direction_of(const Rates& r, float g, float m) { return r.nesterov ? fmaf(r.keep, m - g, g) : m; }
__device__ __forceinline__ float rate_of(const Rates& r) { return r.device_lr ? *r.device_lr : r.lr; }
__device__ __forceinline__ float updated(float w, float x, float shrink, float rate) { return fmaf(-rate, x, w * shrink); }

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ======== matrices with a side of at most 64 =====================================================================================
constexpr int kSmall = 64;
// Tensors of a launch: a table's bytes are written for each launch, so there are two sizes of it.
constexpr int kFewSmall = 24, kTableSmall = 224;
struct SmallEntry {
  Pointers at;
  int rows, cols;
  int stack;
  int chunks, length;        // of a matrix: parts of its longer side, and how much of it each has (a multiple of Side::sub)
  int first;                 // CTA of the launch over parts
  int matrix;                // matrices before
  int vec;                   // four values of every array lie on its boundary, and rows are multiples of four
  float scale;               // of the rate
  size_t gram, q;            // in doubles, in floats: of its first matrix
};
struct SmallHead {
  Rates r;
  int count, first_step, steps, coefficients;   // steps of this run, from first_step on
  int normed;                // X is an earlier run's, not to be divided by its norm
  double *gram, *inverse;
  float* q;
};
template <int CAP>
struct SmallTable : SmallHead {
  SmallEntry e[CAP];
};
struct Coefficients {
  double v[3 * 100];
};
__device__ __forceinline__ int side_of(const SmallEntry& e) { return min(e.rows, e.cols); }
template <int CAP, typename F>
__device__ __forceinline__ int entry_of(const SmallTable<CAP>& t, int block, F first) {
  int a = 0, b = t.count;
  while (b - a > 1) {
    const int c = (a + b) / 2;
    if (first(t.e[c]) <= block) a = c; else b = c;
  }
  return a;
}
// Sides are padded to N = 16 TS with TS = 1, 2, 4.  A symmetric result has 2 TS x 2 TS tiles of 8 x 8; those on and above the diagonal are taken in TS groups
// of 2 TS + 1: rows g and 2 TS - 1 - g of tiles.
template <int TS>
struct Side {
  static constexpr int N = 16 * TS, LD = N + 4, rows = 2 * TS, slots = 2 * TS + 1, tiles = TS * slots;   // (LD: fragments without bank conflicts)
  static constexpr int sub = 2048 / N;                  // of the longer side that a CTA holds: 2048 values
  static constexpr int slices = 8 / TS;                 // warps that share a group, each with 16 of sub
  static constexpr int part = tiles * 64;               // doubles of a part of A, [group][slot][lane][2]
  __device__ static __forceinline__ void tile(int group, int slot, int& ti, int& tj) {
    const int first = rows - group;
    ti = slot < first ? group : rows - 1 - group;
    tj = slot < first ? group + slot : ti + slot - first;
  }
};
constexpr int kPart[5] = {0, Side<1>::part, Side<2>::part, 0, Side<4>::part};
// c += a b of 8 x 4 by 4 x 8 in 64 bits: a is of row lane / 4 and k lane % 4, b of column lane / 4, c of row lane / 4 and columns 2 (lane % 4) and one on.
// (The same rate as fma, a fourth of the loads from shared memory: a symmetric product of 64 x 64 x 64 in 1.3 us, with tiles of 4 x 2 in fma 4.8.)
__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// The 2048 values of a matrix that a CTA of 256 threads takes at a time: eight per thread, VEC neighbours in memory together, all on their way at once.
template <int TS, int VEC>
struct Values {
  static constexpr int each = 8 / VEC, SUB = Side<TS>::sub;
  int n, len;                // sizes of the smaller side and of the longer one
  bool wide;
  unsigned inverse;          // 2^32 / (n / VEC), rounded up: exact quotients for numbers below 2^16
  size_t pitch;
  __device__ Values(const SmallEntry& e) : n(side_of(e)), len(max(e.rows, e.cols)), wide(e.rows <= e.cols), inverse(0xffffffffu / (unsigned)max(1, n / VEC) + 1), pitch(e.cols) {}
  // group j of this thread: its place, and whether it is among the first ks of the longer side
  __device__ __forceinline__ bool place(int j, int ks, int& row, int& k) const {
    const int i = threadIdx.x + j * 256;
    if (wide) {
      row = i / (SUB / VEC);
      k = i % (SUB / VEC) * VEC;
      return row < n && k < ks;
    }
    const int per = n / VEC;
    k = per == 1 ? i : (int)__umulhi((unsigned)i, inverse);
    row = (i - k * per) * VEC;
    return k < ks;
  }
  __device__ __forceinline__ size_t at(int row, int k) const { return wide ? (size_t)row * pitch + k : (size_t)k * n + row; }
  template <typename T>
  __device__ __forceinline__ void load(const T* from, int k0, float (&x)[8]) const {
    const int ks = min(SUB, len - k0);
    Group<T, VEC> v[each];
#pragma unroll
    for (int j = 0; j < each; ++j) {
      int row, k;
      if (place(j, ks, row, k)) v[j] = load_group<T, VEC>(from + at(row, k0 + k));
      else
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j].v[i] = from_float<T>(0.f);
    }
#pragma unroll
    for (int j = 0; j < each; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[j * VEC + i] = to_float(v[j].v[i]);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* to, int k0, const float (&x)[8]) const {
    const int ks = min(SUB, len - k0);
#pragma unroll
    for (int j = 0; j < each; ++j) {
      int row, k;
      if (!place(j, ks, row, k)) continue;
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = x[j * VEC + i];
      store_group(to + at(row, k0 + k), pack<T>(v));
    }
  }
  // f(row, k, value) of what has a place in N x SUB (zeros where nothing is)
  template <typename F>
  __device__ __forceinline__ void each_of(int k0, float (&x)[8], F f) const {
    const int ks = min(SUB, len - k0);
#pragma unroll
    for (int j = 0; j < each; ++j) {
      int row, k;
      const bool in = place(j, ks, row, k);
      if (!in && (wide ? row >= Side<TS>::N : k >= SUB)) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) f(wide ? row : row + i, wide ? k + i : k, x[j * VEC + i]);
    }
  }
};

// A part of A, in 64 bits, from a part of the longer side; the momentum is brought up to date on the way.
template <typename G, int TS, int VEC>
__device__ __forceinline__ void gram_part(const SmallHead& t, const SmallEntry& e, int matrix, int chunk, double* u) {
  using S = Side<TS>;
  constexpr int LD = S::LD;
  Values<TS, VEC> values(e);
  const int n = values.n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t base = (size_t)matrix * e.rows * e.cols;
  const G* g = static_cast<const G*>(e.at.g) + base;
  float* m = e.at.m ? e.at.m + base : nullptr;
  const int group = warp % TS, slice = warp / TS;
  double acc[S::slots][2] = {};
  const int l0 = chunk * e.length, l1 = min(values.len, l0 + e.length);
  if (n < S::N)
    for (int i = tid; i < S::sub * LD; i += 256) u[i] = 0.0;   // (rows past n stay zero)
  float x[8], b[8];   // (the next values are on their way while these are multiplied)
  values.load(g, l0, x);
  if (m) values.load(m, l0, b);
  for (int k0 = l0; k0 < l1; k0 += S::sub) {
    if (m) {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = momentum_of<G>(t.r, x[i], b[i]);
      values.store(m, k0, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = direction_of(t.r, x[i], b[i]);
    }
    __syncthreads();
    values.each_of(k0, x, [&](int row, int k, float v) {
      if (row < n) u[k * LD + row] = (double)v;
    });
    __syncthreads();
    if (k0 + S::sub < l1) {
      values.load(g, k0 + S::sub, x);
      if (m) values.load(m, k0 + S::sub, b);
    }
    const double* from = u + (slice * 16 + (lane & 3)) * LD + (lane >> 2);
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      const double a0 = from[k * LD + group * 8], a1 = from[k * LD + (S::rows - 1 - group) * 8];
#pragma unroll
      for (int s = 0; s < S::slots; ++s) {
        int ti, tj;
        S::tile(group, s, ti, tj);
        mma_f64(acc[s], s < S::rows - group ? a0 : a1, from[k * LD + tj * 8]);
      }
    }
  }
  // the slices' sums, in their order
  __syncthreads();
#pragma unroll
  for (int s = 0; s < S::slots; ++s) {
    double* to = u + ((slice * TS + group) * S::slots + s) * 64 + lane * 2;
    to[0] = acc[s][0];
    to[1] = acc[s][1];
  }
  __syncthreads();
  double* to = t.gram + e.gram + ((size_t)matrix * e.chunks + chunk) * S::part;
  for (int i = tid; i < S::part; i += 256) {
    double s = u[i];
#pragma unroll
    for (int q = 1; q < S::slices; ++q) s += u[q * S::part + i];
    to[i] = s;
  }
}
constexpr int gram_doubles(int ts) {   // of shared memory: the values, or the slices' sums
  return ts == 1 ? std::max(Side<1>::sub * Side<1>::LD, 8 * Side<1>::part) : ts == 2 ? std::max(Side<2>::sub * Side<2>::LD, 4 * Side<2>::part)
                                                                               : std::max(Side<4>::sub * Side<4>::LD, 2 * Side<4>::part);
}
// W: what the widest matrix of the launch takes.  Sides of at most 16 alone (factors of adapters) leave registers for more CTAs an SM, and those are bound by what is
// on its way: 32 matrices of 4096 x 16 and 32 of 16 x 4096, in bfloat16 with copies, 57 us with three of them.
constexpr int per_sm(int w) { return w == 1 ? 5 : 3; }
template <typename G, int W, int CAP>
__global__ void __launch_bounds__(256, per_sm(W)) muon_gram_kernel(const __grid_constant__ SmallTable<CAP> t) {
  extern __shared__ __align__(16) double work[];
  grid_dependency_wait();
  const SmallEntry& e = t.e[entry_of(t, blockIdx.x, [](const SmallEntry& s) { return s.first; })];
  const int at = (int)blockIdx.x - e.first, matrix = at / e.chunks, chunk = at - matrix * e.chunks, n = side_of(e);
#define B200CP_GRAM(TS) (e.vec ? gram_part<G, TS, 4>(t, e, matrix, chunk, work) : gram_part<G, TS, 1>(t, e, matrix, chunk, work))
  if constexpr (W == 1) {
    B200CP_GRAM(1);
  } else {
    if (n <= 16) B200CP_GRAM(1);
    else if (n <= 32) B200CP_GRAM(2);
    else B200CP_GRAM(4);
  }
#undef B200CP_GRAM
}

// out = put(x y), all symmetric and commuting, rows of LD doubles: only tiles on and above the diagonal are there, up to three are formed by each of twelve warps (those below are read
// from above, transposed).  CL CTAs of a cluster share the tiles, and each writes its own into the memory of all.  LAST: of those
// between two barriers (A p and Q p of a step share them: 37.6 us for 74 factors, 36.2 so).
constexpr int kIterateThreads = 384, kShare = 4;
template <int CL>
__device__ __forceinline__ int rank_in_cluster() {
  if constexpr (CL == 1) return 0;
  else return (int)cg::this_cluster().block_rank();
}
template <int CL>
__device__ __forceinline__ void sync_all() {
  if constexpr (CL == 1) __syncthreads();
  else cg::this_cluster().sync();
}
// f(what lies at p in each of the CTAs)
template <int CL, typename F>
__device__ __forceinline__ void for_all(double* p, F f) {
  if constexpr (CL == 1) {
    f(p);
  } else {
#pragma unroll
    for (int q = 0; q < CL; ++q) f(cg::this_cluster().map_shared_rank(p, q));
  }
}
template <int TS, int CL, bool LAST, typename Put>
__device__ __forceinline__ void symmetric_product(const double* x, const double* y, double* out, Put put) {
  using S = Side<TS>;
  constexpr int LD = S::LD, share = (S::tiles + CL - 1) / CL, C = (share + 11) / 12;
  static_assert(share % C == 0 && (CL == 1 || S::tiles % CL == 0));
  const int lane = threadIdx.x & 31, mine = (threadIdx.x >> 5) * C, first = rank_in_cluster<CL>() * share + mine;
  if (mine < share) {
    double acc[C][2] = {};
    int ti[C], tj[C];
#pragma unroll
    for (int c = 0; c < C; ++c) S::tile((first + c) / S::slots, (first + c) % S::slots, ti[c], tj[c]);
    const int direct = (lane & 3) * LD + (lane >> 2), crossed = (lane >> 2) * LD + (lane & 3);
    const auto fragment = [&](const double* z, int k, int tile) { return z[k / 8 <= tile ? direct + k * LD + tile * 8 : crossed + tile * 8 * LD + k]; };
#pragma unroll
    for (int k = 0; k < S::N; k += 4)
#pragma unroll
      for (int c = 0; c < C; ++c) mma_f64(acc[c], fragment(x, k, ti[c]), fragment(y, k, tj[c]));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int row = ti[c] * 8 + (lane >> 2), col = tj[c] * 8 + (lane & 3) * 2;
      const double2 v = make_double2(put(acc[c][0], row, col), put(acc[c][1], row, col + 1));
      for_all<CL>(out, [&](double* to) { *reinterpret_cast<double2*>(to + row * LD + col) = v; });
    }
  }
  if constexpr (LAST) sync_all<CL>();
}
template <int TS, int CL>
__device__ __forceinline__ void iterate(const SmallHead& t, const Coefficients& co, const SmallEntry& e, int matrix, double* work) {
  using S = Side<TS>;
  constexpr int N = S::N, LD = S::LD, NN = N * LD, share = S::part / CL, kOwn = (share + kIterateThreads - 1) / kIterateThreads;
  const int tid = threadIdx.x, rank = rank_in_cluster<CL>(), n = side_of(e);
  double *A = work, *Q = A + NN, *F = Q + NN, *P = F + NN, *R = P + NN;
  __shared__ double trace_sum;
  // the parts of A, in their order
  const double* from = t.gram + e.gram + (size_t)matrix * e.chunks * S::part + rank * share;
  double own[kOwn] = {};
#pragma unroll (CL == 1 ? 2 : 8)
  for (int c = 0; c < e.chunks; ++c)
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (tid + j * kIterateThreads < share) own[j] += from[(size_t)c * S::part + tid + j * kIterateThreads];
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    if (tid + j * kIterateThreads >= share) break;
    const int i = rank * share + tid + j * kIterateThreads;
    int ti, tj;
    S::tile(i / 64 / S::slots, i / 64 % S::slots, ti, tj);
    const int r = ti * 8 + i % 64 / 8, c = tj * 8 + i % 8;
    for_all<CL>(A, [&](double* to) { to[r * LD + c] = own[j]; });
  }
  sync_all<CL>();
  if (tid < 32) {
    double s = 0.0;
    for (int i = tid; i < n; i += 32) s += A[i * LD + i];
    s = warp_sum(s);
    if (tid == 0) trace_sum = s;
  }
  __syncthreads();
  const double root = sqrt(trace_sum), inverse = t.normed ? 1.0 : 1.0 / (root > t.r.eps || root != root ? root : t.r.eps);
  for (int i = tid; i < NN; i += kIterateThreads) {
    A[i] = A[i] * inverse * inverse;   // (one after the other: the square of 1 / eps may be infinite, and A zero)
    if (t.steps == 0) Q[i] = i / LD == i % LD ? 1.0 : 0.0;
  }
  __syncthreads();
  const auto as_is = [](double v, int, int) { return v; };
  for (int step = 0; step < t.steps; ++step) {
    const double *v = co.v + (t.coefficients > 1 ? 3 * (t.first_step + step) : 0), v0 = v[0], v1 = v[1], v2 = v[2];
    double* p = step == 0 ? Q : P;
    symmetric_product<TS, CL, true>(A, A, p, [&](double s, int r, int c) { return fma(v2, s, fma(v1, A[r * LD + c], r == c ? v0 : 0.0)); });
    const bool last = step + 1 == t.steps;
    if (!last) symmetric_product<TS, CL, false>(A, p, F, as_is);
    if (step > 0) {
      symmetric_product<TS, CL, false>(Q, p, R, as_is);
      double* q = Q;
      Q = R;
      R = q;
    }
    sync_all<CL>();
    if (!last) symmetric_product<TS, CL, true>(F, p, A, as_is);
  }
  float* to = t.q + e.q + (size_t)matrix * (n * n);
  for (int i = rank * kIterateThreads + tid; i < n * n; i += CL * kIterateThreads) {
    const int r = i / n, c = i % n;
    to[i] = (float)Q[r / 8 <= c / 8 ? r * LD + c : c * LD + r];
  }
  if (tid == 0 && rank == 0) t.inverse[e.matrix + matrix] = inverse;
}
template <int CAP>
__device__ __forceinline__ const SmallEntry& entry_with(const SmallTable<CAP>& t, int matrix) {
  return t.e[entry_of(t, matrix, [](const SmallEntry& s) { return s.matrix; })];
}
// WIDEST: of the launch's matrices, as Side's TS.  Sides up to 32 leave room for three CTAs an SM (3000 of 16 x 64 86 us, with
// one 122), 64 takes 174 KB of shared memory.
template <int WIDEST, int CAP>
__global__ void __launch_bounds__(kIterateThreads, WIDEST == 4 ? 1 : 3) muon_iterate_kernel(const __grid_constant__ SmallTable<CAP> t, const __grid_constant__ Coefficients co) {
  extern __shared__ __align__(16) double work[];
  grid_dependency_wait();
  const SmallEntry& e = entry_with(t, blockIdx.x);
  const int matrix = (int)blockIdx.x - e.matrix, n = side_of(e);
  if constexpr (WIDEST == 4)
    if (n > 32) return iterate<4, 1>(t, co, e, matrix, work);
  if constexpr (WIDEST >= 2)
    if (n > 16) return iterate<2, 1>(t, co, e, matrix, work);
  iterate<1, 1>(t, co, e, matrix, work);
}
// The same with a cluster for each of the first `wide` matrices, whose sides are above 32, and a CTA for each of the others: where all of them have an SM.  A product of
// 64 x 64 takes 3100 cycles of one SM (2300 of its 64-bit tensor instructions), 2250 of four: 1150 for the tiles, 800 until they are in all memories, 300 for the barrier.  (One
// matrix of 64 x 64 42 us in all when one CTA took its steps, 33 so.)  Where they do not all have an SM, clusters would wait for the SMs of other ones.
template <int CAP>
__global__ void __cluster_dims__(kShare, 1, 1) __launch_bounds__(kIterateThreads)
    muon_iterate_shared_kernel(const __grid_constant__ SmallTable<CAP> t, const __grid_constant__ Coefficients co, int wide, int matrices) {
  extern __shared__ __align__(16) double work[];
  const bool shared = (int)blockIdx.x < kShare * wide;
  const int at = shared ? (int)blockIdx.x / kShare : (int)blockIdx.x - (kShare - 1) * wide;
  if (shared) sync_all<kShare>();   // (all CTAs of the cluster are there before one writes into another)
  grid_dependency_wait();
  if (at >= matrices) return;
  const SmallEntry& e = entry_with(t, at);
  const int matrix = at - e.matrix, n = side_of(e);
  if (shared) iterate<4, kShare>(t, co, e, matrix, work);
  else if (n <= 16) iterate<1, 1>(t, co, e, matrix, work);
  else iterate<2, 1>(t, co, e, matrix, work);
}

// X = Q u / |u| for a part of the longer side, and the update.
constexpr int small_apply_floats(int ts) {   // Q [j][i], X [j][k] and what becomes of it
  const int N = 16 * ts;
  return N * N + 2 * N * (2048 / N + 1);
}
template <typename P, typename G, int TS, int VEC>
__device__ __forceinline__ void apply_part(const SmallHead& t, const SmallEntry& e, int matrix, int chunk, float* low) {
  using S = Side<TS>;
  constexpr int LD = S::sub + 1, N = S::N;
  Values<TS, VEC> values(e);
  const int n = values.n, tid = threadIdx.x;
  float *q = low, *x = q + N * N, *o = x + N * LD;
  const size_t base = (size_t)matrix * e.rows * e.cols;
  const G* g = static_cast<const G*>(e.at.g) + base;
  const float* m = e.at.m ? e.at.m + base : nullptr;
  float* w = e.at.w ? e.at.w + base : nullptr;
  P* p = static_cast<P*>(e.at.p) + base;
  const float* from = t.q + e.q + (size_t)matrix * (n * n);
  const double inverse = t.inverse[e.matrix + matrix];
  const float lr = rate_of(t.r), rate = lr * e.scale, shrink = 1.f - lr * t.r.decay;
#pragma unroll 4
  for (int i = tid; i < N * N; i += 256) q[i] = i / N < n && i % N < n ? from[i / N * n + i % N] : 0.f;
  const int l0 = chunk * e.length, l1 = min(values.len, l0 + e.length);
  float v[8], b[8], next[8];   // (the next values are on their way while these are multiplied)
  const auto fetch = [&](int k0) {
    values.load(g, k0, v);
    if (m) values.load(m, k0, b);
    if (t.r.update) {
      if (w) values.load(w, k0, next);
      else values.load(p, k0, next);
    }
  };
  fetch(l0);
  for (int k0 = l0; k0 < l1; k0 += S::sub) {
    const int ks = min(S::sub, values.len - k0);
    float old[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      old[i] = next[i];
      v[i] = (float)((double)(m ? direction_of(t.r, v[i], b[i]) : v[i]) * inverse);
    }
    __syncthreads();
    values.each_of(k0, v, [&](int row, int k, float a) {
      if (row < n) x[row * LD + k] = a;
    });
    __syncthreads();
    if (k0 + S::sub < l1) fetch(k0 + S::sub);
    // eight rows of a k per thread
    const int k = tid % S::sub, i0 = tid / S::sub * 8;
    if (i0 < n) {
      float acc[8] = {};
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float a = x[j * LD + k];
        const float4 c = *reinterpret_cast<const float4*>(q + j * N + i0), d = *reinterpret_cast<const float4*>(q + j * N + i0 + 4);
        acc[0] = fmaf(c.x, a, acc[0]); acc[1] = fmaf(c.y, a, acc[1]); acc[2] = fmaf(c.z, a, acc[2]); acc[3] = fmaf(c.w, a, acc[3]);
        acc[4] = fmaf(d.x, a, acc[4]); acc[5] = fmaf(d.y, a, acc[5]); acc[6] = fmaf(d.z, a, acc[6]); acc[7] = fmaf(d.w, a, acc[7]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[(i0 + i) * LD + k] = acc[i];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j) {
      int row, c;
      if (!values.place(j, ks, row, c)) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float a = o[(values.wide ? row : row + i) * LD + (values.wide ? c + i : c)];
        old[j * VEC + i] = t.r.update ? updated(old[j * VEC + i], a, shrink, rate) : a;
      }
    }
    if (w && t.r.update) values.store(w, k0, old);
    values.store(p, k0, old);
  }
}
template <typename P, typename G, int W, int CAP>
__global__ void __launch_bounds__(256, per_sm(W)) muon_small_apply_kernel(const __grid_constant__ SmallTable<CAP> t) {
  extern __shared__ __align__(16) float low[];
  grid_dependency_wait();
  const SmallEntry& e = t.e[entry_of(t, blockIdx.x, [](const SmallEntry& s) { return s.first; })];
  const int at = (int)blockIdx.x - e.first, matrix = at / e.chunks, chunk = at - matrix * e.chunks, n = side_of(e);
#define B200CP_APPLY(TS) (e.vec ? apply_part<P, G, TS, 4>(t, e, matrix, chunk, low) : apply_part<P, G, TS, 1>(t, e, matrix, chunk, low))
  if constexpr (W == 1) {
    B200CP_APPLY(1);
  } else {
    if (n <= 16) B200CP_APPLY(1);
    else if (n <= 32) B200CP_APPLY(2);
    else B200CP_APPLY(4);
  }
#undef B200CP_APPLY
}

// ======== larger matrices ===========================================================================================================
// All of them go together, up to kItems matrices of kProblems shapes and a gigabyte or two of planes: a launch takes all their tiles.
constexpr int kFlight = 8;                                     // loads of a thread that are on their way together
constexpr int kFewItems = 16, kItems = 256, kFewProblems = 4, kProblems = 48, kNormParts = 1024;   // (tables of two sizes, as above; kNormParts: parts of a norm)
constexpr int kTurn = 256 * 8 * 4;                             // values of a CTA
struct Item {
  Pointers at;
  int rows, cols, ld;             // ld: of the planes
  int vec;                        // eight values of every array lie on its boundary, and rows are multiples of eight
  size_t plane;                   // halves from one plane to the next
  __half* x;
  int first, chunk, parts, norm;  // of the launch over the values: its first CTA, values of a CTA, CTAs; its first part of a norm
  int first8;                     // of the launches over the planes
  float rate;                     // factor of the rate
};
struct ItemsHead {
  Rates r;
  int count;
  float scale;                    // planes hold scale X
  double* norms;
};
template <int CAP>
struct Items : ItemsHead {
  Item e[CAP];
};
template <int CAP, typename F>
__device__ __forceinline__ const Item& item_of(const Items<CAP>& t, int block, F first) {
  int a = 0, b = t.count;
  while (b - a > 1) {
    const int c = (a + b) / 2;
    if (first(t.e[c]) <= block) a = c; else b = c;
  }
  return t.e[a];
}
template <typename T>
__device__ __forceinline__ void load8(const T* from, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 8; h += kPerLoad<T>) {
    float y[kPerLoad<T>];
    unpack(load_group<T, kPerLoad<T>>(from + h), y);
#pragma unroll
    for (int k = 0; k < kPerLoad<T>; ++k) x[h + k] = y[k];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 8; h += kPerLoad<T>) {
    float y[kPerLoad<T>];
#pragma unroll
    for (int k = 0; k < kPerLoad<T>; ++k) y[k] = x[h + k];
    store_group(to + h, pack<T>(y));
  }
}

// Momentum, and a part of |u|^2 in 64 bits.
template <typename G, int CAP>
__global__ void __launch_bounds__(256) muon_momentum_kernel(const __grid_constant__ Items<CAP> t) {
  grid_dependency_wait();
  const Item& e = item_of(t, blockIdx.x, [](const Item& i) { return i.first; });
  const int part = (int)blockIdx.x - e.first;
  const G* g = static_cast<const G*>(e.at.g);
  float* m = e.at.m;
  const long long i0 = (long long)part * e.chunk, n = min((long long)e.rows * e.cols, i0 + e.chunk);
  double s = 0.0;
  if (e.vec) {
#pragma unroll 2
    for (long long i = i0 + threadIdx.x * 8; i < n; i += 256 * 8) {
      float x[8], b[8];
      load8(g + i, x);
      if (m) {
        load8(m + i, b);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          b[k] = momentum_of<G>(t.r, x[k], b[k]);
          x[k] = direction_of(t.r, x[k], b[k]);
        }
        store8(m + i, b);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fma((double)x[k], (double)x[k], s);
    }
  } else {
    for (long long i = i0 + threadIdx.x; i < n; i += 256 * kFlight) {
      float x[kFlight], b[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const long long at = i + j * 256;
        x[j] = at < n ? to_float(g[at]) : 0.f;
        b[j] = m && at < n ? m[at] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const long long at = i + j * 256;
        if (at >= n) break;
        if (m) {
          b[j] = momentum_of<G>(t.r, x[j], b[j]);
          m[at] = b[j];
          x[j] = direction_of(t.r, x[j], b[j]);
        }
        s = fma((double)x[j], (double)x[j], s);
      }
    }
  }
  __shared__ double red[8];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i];
    t.norms[e.norm + part] = s;
  }
}
__device__ __forceinline__ void split8(const float (&v)[8], Group<__half, 8>& hi, Group<__half, 8>& lo) {
  float r[8];
  hi = pack<__half>(v);
  unpack(hi, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i] - r[i];
  lo = pack<__half>(r);
}
// The planes of X.  Eight columns per thread and turn, four turns.
template <typename G, int CAP>
__global__ void __launch_bounds__(256) muon_planes_kernel(const __grid_constant__ Items<CAP> t) {
  __shared__ double red[8];
  grid_dependency_wait();
  const Item& e = item_of(t, blockIdx.x, [](const Item& i) { return i.first8; });
  double s = 0.0;
  for (int i = threadIdx.x; i < e.parts; i += 256) s += t.norms[e.norm + i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += red[i];
  s = sqrt(s);
  const double inv = (double)t.scale / (s > t.r.eps || s != s ? s : t.r.eps);
  const G* g = static_cast<const G*>(e.at.g);
  const float* m = e.at.m;
  const unsigned per = (unsigned)(e.cols + 7) / 8;
  const unsigned long long n = (unsigned long long)e.rows * per, first = (unsigned long long)((int)blockIdx.x - e.first8) * 1024 + threadIdx.x;
#pragma unroll 2
  for (int j = 0; j < 4; ++j) {
    const unsigned long long i = first + j * 256;
    if (i >= n) break;
    const size_t row = n <= 0xffffffffu ? (size_t)((unsigned)i / per) : (size_t)(i / per);
    const int c = (int)(i - row * per) * 8;
    const size_t src = row * e.cols + c;
    float x[8], b[8];
    if (e.vec) {
      load8(g + src, x);
      if (m) load8(m + src, b);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = c + k < e.cols ? to_float(g[src + k]) : 0.f;
        b[k] = m && c + k < e.cols ? m[src + k] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (m) x[k] = direction_of(t.r, x[k], b[k]);
      x[k] = (float)((double)x[k] * inv);
    }
    Group<__half, 8> hi, lo;
    split8(x, hi, lo);
    store_group(e.x + row * e.ld + c, hi);
    store_group(e.x + e.plane + row * e.ld + c, lo);
  }
}
// The update from the planes of the last X.
template <typename P, int CAP>
__global__ void __launch_bounds__(256) muon_apply_kernel(const __grid_constant__ Items<CAP> t) {
  grid_dependency_wait();
  const Item& e = item_of(t, blockIdx.x, [](const Item& i) { return i.first8; });
  P* p = static_cast<P*>(e.at.p);
  float* master = e.at.w;
  const float lr = rate_of(t.r), rate = lr * e.rate, shrink = 1.f - lr * t.r.decay, unit = 1.f / t.scale;
  const unsigned per = (unsigned)(e.cols + 7) / 8;
  const unsigned long long n = (unsigned long long)e.rows * per, first = (unsigned long long)((int)blockIdx.x - e.first8) * 1024 + threadIdx.x;
#pragma unroll 2
  for (int j = 0; j < 4; ++j) {
    const unsigned long long i = first + j * 256;
    if (i >= n) break;
    const size_t row = n <= 0xffffffffu ? (size_t)((unsigned)i / per) : (size_t)(i / per);
    const int c = (int)(i - row * per) * 8;
    const size_t dst = row * e.cols + c;
    float x[8], l[8], w[8];
    unpack(load_group<__half, 8>(e.x + row * e.ld + c), x);
    unpack(load_group<__half, 8>(e.x + e.plane + row * e.ld + c), l);
    if (t.r.update) {
      if (e.vec) {
        if (master) load8(master + dst, w);
        else load8(p + dst, w);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = c + k < e.cols ? (master ? master[dst + k] : to_float(p[dst + k])) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = (x[k] + l[k]) * unit;
      if (t.r.update) x[k] = updated(w[k], x[k], shrink, rate);
    }
    if (e.vec) {
      if (master && t.r.update) store8(master + dst, x);
      store8(p + dst, x);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (c + k >= e.cols) break;
        if (master && t.r.update) master[dst + k] = x[k];
        p[dst + k] = from_float<P>(x[k]);
      }
    }
  }
}

// ---- the products ------------------------------------------------------------------------------------------------------------------
// out = alpha sum_k L[m][k] R[n][k] + beta add, of planes, for batches of matrices of several shapes (problems).  A pair of CTAs has a tile of
// 256 x BN; one thread issues, accumulators in turn.  A stage has both planes of 64 k, products are hi hi + hi lo + lo hi; an accumulator holds kGroupSteps stages and is then
// added to totals in registers.
constexpr int kStep = 64, kBand = 16, kGroupSteps = 4;
constexpr int kPatch = 32 * 64;   // bytes of a warp's block of 32 x 32 halves on its way in or out
template <int BN>
struct Tile {
  static constexpr int planes = 2;
  static constexpr int aplane = 128 * kStep * 2, bplane = BN / 2 * kStep * 2;
  static constexpr int abytes = planes * aplane, stage = abytes + planes * bplane;                   // 64 or 48 KB
  static constexpr int stages = 192 * 1024 / stage, depth = BN == 256 ? 2 : 4;                       // of the ring; accumulators
  static constexpr int readers = 4 * BN / 64, threads = 64 + 32 * readers;
  static constexpr size_t smem = (size_t)stages * stage + readers * kPatch + 1024 + 256;
  static_assert(smem <= 227 * 1024 && depth * BN == 512 && (2 * stages + 2 * depth) * 8 + 8 <= 256, "");
};
struct alignas(64) Problem {
  CUtensorMap L, R;
  int M, N, steps;               // of a result; of a sum, in stages
  int tiles_m, tiles_n, per, first;   // tiles of a matrix; the problem's first one in the launch
  int symmetric, l_mn, r_mn;     // an operand lies as [k][row] (boxes of 64 rows x 64 k), else as [row][k]
  float alpha, beta;
  const __half* add;             // as out, or null
  __half* out;
  int ld;
  size_t plane, matrix;          // halves from one plane to the next, and from one matrix
};
template <int CAP>
struct Problems {
  int count, units;
  int early;                     // few tiles: the next launch takes its place on the other SMs meanwhile (66 x 70 in a graph: 131 us a step, 119 so)
  Problem p[CAP];
};
struct UnitAt {
  int problem, matrix, m0, n0;
  bool mirror;
};
template <int BN, int CAP>
__device__ __forceinline__ UnitAt unit_at(const Problems<CAP>& all, int unit) {
  int k = 0;
  while (k + 1 < all.count && all.p[k + 1].first <= unit) ++k;
  const Problem& g = all.p[k];
  const int i = (unit - g.first) / g.per;
  int t = unit - g.first - i * g.per;
  if (g.symmetric) {             // rows of blocks, each from its diagonal on
    constexpr int q = 256 / BN;
    int row = 0, left = g.tiles_n;
    while (t >= left) {
      t -= left;
      left -= q;
      ++row;
    }
    const int n0 = (row * q + t) * BN;
    return UnitAt{k, i, row * 256, n0, n0 >= (row + 1) * 256};
  }
  const int band = t / (kBand * g.tiles_n), m1 = band * kBand, height = min(kBand, g.tiles_m - m1), q = t - m1 * g.tiles_n;
  return UnitAt{k, i, (m1 + q % height) * 256, (q / height) * BN, false};
}
__device__ __forceinline__ void tma_load_planes(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int matrix) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(0), "r"(matrix)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"f"(v[0]),
      "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "r"(taddr)
      : "memory");
}

// A warp's block of 32 rows of 32 halves, a row to a lane in registers, but 64 bytes of each of eight rows at a time in memory: through shared memory (rows of 64 bytes,
// their 16-byte pieces swizzled).  Straight from the registers every access is of 32 rows and 16 bytes of each; the read-out of a tile then took 16 000 cycles, more than
// the accumulators that wait meanwhile last.
struct Block {
  int M, N, ld, m0, n;
  // (rows are longer than N where that is no multiple of eight: nobody reads what is behind)
  __device__ __forceinline__ bool in(int i, int& row, int& col) const {
    const int lane = threadIdx.x & 31;
    row = m0 + i * 8 + (lane >> 2);
    col = n + (lane & 3) * 8;
    return row < M && col < N;
  }
  __device__ __forceinline__ static uint4* place(uint8_t* patch, int row, int piece) {
    return reinterpret_cast<uint4*>(patch + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
  }
  __device__ __forceinline__ void load(const __half* from, uint4 (&q)[4]) const {   // as it lies in memory
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int row, col;
      q[i] = in(i, row, col) ? *reinterpret_cast<const uint4*>(from + (size_t)row * ld + col) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void turn(uint8_t* patch, uint4 (&q)[4]) const {       // to a row per lane
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) *place(patch, i * 8 + (lane >> 2), lane & 3) = q[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *place(patch, lane, i);
  }
  __device__ __forceinline__ void store(uint8_t* patch, __half* to, const uint4 (&q)[4]) const {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) *place(patch, lane, i) = q[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int row, col;
      if (in(i, row, col)) *reinterpret_cast<uint4*>(to + (size_t)row * ld + col) = *place(patch, i * 8 + (lane >> 2), lane & 3);
    }
  }
};
__device__ __forceinline__ void unpack_times(const uint4& q, float by, float* v, bool more) {
  float x[8];
  unpack(*reinterpret_cast<const Group<__half, 8>*>(&q), x);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = more ? fmaf(by, x[i], v[i]) : by * x[i];
}

template <int BN, int CAP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Tile<BN>::threads, 1) newton_kernel(const __grid_constant__ Problems<CAP> all) {
  using T = Tile<BN>;
  constexpr int kStages = T::stages, kBox = T::planes * kStep * 128;   // kBox: bytes of 64 rows, MN-major
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = sm + kStages * T::stage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(patches + T::readers * kPatch);
  uint64_t* full = bars;                 // [kStages] the leader's: the stage of both CTAs has landed  (tx bytes)
  uint64_t* empty = full + kStages;      // [kStages] the products that read the stage are done         (commit, both CTAs)
  uint64_t* accfull = empty + kStages;   // [depth] the accumulator is complete                         (commit, both CTAs)
  uint64_t* accfree = accfull + T::depth;   // [depth] the leader's: read out by the warps of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accfree + T::depth);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < T::depth; ++i) {
      mbar_init(&accfull[i], 1);
      mbar_init(&accfree[i], 2 * T::readers);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t fullb = smem_u32(full), emptyb = smem_u32(empty), accfullb = smem_u32(accfull), accfreeb = smem_u32(accfree),
                 abortb = smem_u32(const_cast<int*>(abort_flag));
  grid_dependency_wait();
  if (all.early) grid_launch_dependents();

  if (warp == 0) {
    // ================= TMA: this CTA's rows of L and its half of the rows of R ==============================================
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int unit = pair; unit < all.units && ok; unit += npairs) {
        const UnitAt t = unit_at<BN>(all, unit);
        const Problem& g = all.p[t.problem];
        const int m = t.m0 + rank * 128, n = t.n0 + rank * (BN / 2);
        for (int s = 0; s < g.steps; ++s, ++it) {
          const int slot = it % kStages;
          if (it >= kStages && !(ok = wait_or_abort(emptyb + slot * 8, ((it / kStages) - 1) & 1, abortb))) break;
          if (rank == 0) mbar_expect_tx(&full[slot], 2 * T::stage);
          const uint32_t bar = leader_addr(fullb + slot * 8), a = smem_u32(sm) + slot * T::stage, b = a + T::abytes;
          const int k = s * kStep;
          if (g.l_mn) {
#pragma unroll
            for (int q = 0; q < 2; ++q) tma_load_planes(a + q * kBox, &g.L, bar, m + q * 64, k, t.matrix);
          } else {
            tma_load_planes(a, &g.L, bar, k, m, t.matrix);
          }
          if (g.r_mn) {
#pragma unroll
            for (int q = 0; q < BN / 128; ++q) tma_load_planes(b + q * kBox, &g.R, bar, n + q * 64, k, t.matrix);
          } else {
            tma_load_planes(b, &g.R, bar, k, n, t.matrix);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ================= products: one thread of the pair ======================================================================
    if (rank == 0 && elect_one()) {
      int it = 0, gi = 0;   // stages, accumulators
      bool ok = true;
      for (int unit = pair; unit < all.units && ok; unit += npairs) {
        const Problem& g = all.p[unit_at<BN>(all, unit).problem];
        const uint32_t idesc = (1u << 4) | ((uint32_t)g.l_mn << 15) | ((uint32_t)g.r_mn << 16) | (((uint32_t)BN >> 3) << 17) | ((256u >> 4) << 24);
        // K-major: rows of 128 bytes, eight rows per swizzle atom (1024 bytes); 16 k = 32 bytes on; the second plane all rows on.
        // MN-major: 64 rows (128 bytes) per k, eight k per atom, the next 64 rows a box on; 16 k = 2048 bytes on; the second plane 64 k on.
        const uint64_t dl = make_smem_desc(0, g.l_mn ? kBox : 16, 1024, kSwizzle128B), dr = make_smem_desc(0, g.r_mn ? kBox : 16, 1024, kSwizzle128B);
        const uint64_t sl = (g.l_mn ? 2048 : 32) >> 4, sr = (g.r_mn ? 2048 : 32) >> 4;
        const uint64_t pl = (g.l_mn ? kStep * 128 : T::aplane) >> 4, pr = (g.r_mn ? kStep * 128 : T::bplane) >> 4;
        const int steps = g.steps;
        for (int s = 0; s < steps; ++s, ++it) {
          const int slot = it % kStages, buf = gi % T::depth;
          const bool first = s % kGroupSteps == 0, last = s + 1 == steps || s % kGroupSteps == kGroupSteps - 1;
          if (!(ok = wait_or_abort(fullb + slot * 8, (it / kStages) & 1, abortb))) break;
          if (first && gi >= T::depth && !(ok = wait_or_abort(accfreeb + buf * 8, (gi / T::depth - 1) & 1, abortb))) break;
          tc_fence_after_sync();
          const uint32_t a = smem_u32(sm) + slot * T::stage, d = tmem_base + buf * BN;
          const uint64_t l = dl + (a >> 4), r = dr + ((a + T::abytes) >> 4);
#pragma unroll
          for (int i = 0; i < kStep / 16; ++i) {   // the small products first
            mma_f16_pair(d, l + pl + i * sl, r + i * sr, idesc, !first || i > 0);
            mma_f16_pair(d, l + i * sl, r + pr + i * sr, idesc, true);
          }
#pragma unroll
          for (int i = 0; i < kStep / 16; ++i) mma_f16_pair(d, l + i * sl, r + i * sr, idesc, true);
          if (last) {
            commit_pair(accfullb + buf * 8);
            ++gi;
          }
          commit_pair(emptyb + slot * 8);
        }
      }
    }
  } else {
    // ================= read-out: accumulators -> totals -> planes =============================================================
    const int qd = warp & 3, c0 = ((warp - 2) >> 2) * 64;   // the lane quarter that this warp may read, and its columns
    const uint32_t taddr = tmem_base + ((uint32_t)(qd * 32) << 16) + c0;
    int gi = 0;
    bool ok = true;
    for (int unit = pair; unit < all.units && ok; unit += npairs) {
      int buf = 0;
      float tot[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) tot[j] = 0.f;
      const int groups = (all.p[unit_at<BN>(all, unit).problem].steps + kGroupSteps - 1) / kGroupSteps;
      for (int s = 0; s < groups; ++s, ++gi) {
        buf = gi % T::depth;
        if (!(ok = __all_sync(0xffffffffu, wait_or_abort(accfullb + buf * 8, (gi / T::depth) & 1, abortb)))) break;
        tc_fence_after_sync();
#pragma unroll
        for (int j0 = 0; j0 < 64; j0 += 16) {
          float v[16];
          tmem_ld16(taddr + buf * BN + j0, v);
          if (j0 == 48 && s + 1 < groups) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_cluster(leader_addr(accfreeb + buf * 8));
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) tot[j0 + j] += v[j];
        }
      }
      if (!ok) break;
      // through the accumulator just read, so that a short loop stores them (unrolled over registers it is code that every tile fetches anew)
#pragma unroll
      for (int j0 = 0; j0 < 64; j0 += 16) tmem_st16(taddr + buf * BN + j0, tot + j0);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      const UnitAt t = unit_at<BN>(all, unit);
      const Problem& g = all.p[t.problem];
      const int m0 = t.m0 + rank * 128 + qd * 32, m = m0 + lane;
      uint8_t* patch = patches + (warp - 2) * kPatch;
      const size_t base = t.matrix * g.matrix;
#pragma unroll 1
      for (int j0 = 0; j0 < 64; j0 += 32) {
        const int n = t.n0 + c0 + j0;
        if (m0 >= g.M || n >= g.N) continue;   // (all lanes)
        __syncwarp();
        const Block at{g.M, g.N, g.ld, m0, n};
        // (g.plane is never 0: the branches on it keep the second plane's values out of the registers until the first one's are done.  Without them more is
        // spilled, and five steps take 1.5 to 3.5 % longer: 3 of 1100 x 1111 522 us, so 502)
        float v[32];
        if (g.add) {
          uint4 in[4], more[4];
          at.load(g.add + base, in);
          if (g.plane) at.load(g.add + base + g.plane, more);
          at.turn(patch, in);
#pragma unroll
          for (int j = 0; j < 32; j += 8) unpack_times(in[j / 8], g.beta, v + j, false);
          if (g.plane) {
            at.turn(patch, more);
#pragma unroll
            for (int j = 0; j < 32; j += 8) unpack_times(more[j / 8], g.beta, v + j, true);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float x[8];
          tmem_ld8(taddr + buf * BN + j0 + j, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j + i] = fmaf(g.alpha, x[i], v[j + i]);
        }
        __half* out = g.out + base;
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {   // hi, then what is left
          if (plane && !g.plane) break;
          uint4 q[4];
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            Group<__half, 8> h;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = v[j + i];
            h = pack<__half>(x);
            unpack(h, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j + i] -= x[i];
            q[j / 8] = *reinterpret_cast<const uint4*>(&h);
          }
          __half* to = out + plane * g.plane;
          if (t.mirror && m < g.M) {   // neighbouring lanes have neighbouring columns of these
            const __half* h = reinterpret_cast<const __half*>(q);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (n + j < g.N) to[(size_t)(n + j) * g.ld + m] = h[j];
          }
          at.store(patch, to, q);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_cluster(leader_addr(accfreeb + buf * 8));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    atomicCAS(&g_muon_status, 0, (1 << 16) | (blockIdx.x & 0xffff));
    const long long t0 = clock64();   // copies in flight land before the shared memory is given back
    while (clock64() - t0 < 40000000ll) {
    }
  }
  cluster_sync();   // the peer's products read this CTA's shared memory, and its commits arrive on its barriers
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ======== host ======================================================================================================================
// (A slot per kernel, not per caller: callers of several types share some, and each would set its own, smaller size.)
template <auto KERNEL>
cudaError_t allow_smem(int bytes) {
  static std::atomic<int> set[64];
  return ensure_dynamic_smem(reinterpret_cast<const void*>(KERNEL), set, bytes);
}
struct Planes {   // of a batch of matrices
  __half* p;
  int rows, cols, ld, count;
  size_t plane() const { return (size_t)rows * ld; }
  size_t matrix() const { return 2 * plane(); }
};
// Rows of planes start on 128-byte lines, so that what a tile takes of one is one line (1030 x 2051 in rows of 2056: 32.8 us for X X^T, now 28.7).
int pitch_of(int n) { return (n + 63) / 64 * 64; }
int encode(CUtensorMap* map, const Planes& m, int box_rows) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B200CP_ERR_NO_DEVICE, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dim[4] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, 2, (cuuint64_t)m.count},
                   stride[3] = {(cuuint64_t)m.ld * 2, (cuuint64_t)m.plane() * 2, (cuuint64_t)m.matrix() * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 2, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, m.p, dim, stride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (cr != CUDA_SUCCESS) return fail(B200CP_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)cr);
  return B200CP_OK;
}
long long tiles_of(int M, int N, int BN, bool symmetric) {   // of one matrix
  const long long tm = ceil_div(M, 256), tn = ceil_div(N, BN), q = 256 / BN;
  return symmetric ? tm * tn - q * tm * (tm - 1) / 2 : tm * tn;
}
// The tensor maps of a call, each encoded once: by the planes' address and the rows of a box.
struct Maps {
  std::map<std::pair<const void*, int>, CUtensorMap> all;
  int get(CUtensorMap* to, const Planes& m, int box_rows) {
    const auto [at, is_new] = all.try_emplace({m.p, box_rows});
    if (is_new)
      if (int rc = encode(&at->second, m, box_rows)) return rc;
    *to = at->second;
    return B200CP_OK;
  }
};
// out = alpha L R^T + beta add
struct Product {
  Planes L, R, out;
  bool l_mn, r_mn, symmetric;
  int K;
  double alpha, beta;
  const Planes* add;
};
template <int BN, int CAP>
int launch_table(const std::vector<Product>& ps, Maps& maps, int pairs, cudaStream_t st) {
  using T = Tile<BN>;
  Problems<CAP> all;
  all.count = 0;
  long long units = 0;
  for (const Product& q : ps) {
    Problem& p = all.p[all.count++];
    if (int rc = maps.get(&p.L, q.L, q.l_mn ? kStep : 128)) return rc;
    if (int rc = maps.get(&p.R, q.R, q.r_mn ? kStep : BN / 2)) return rc;
    p.M = q.out.rows;
    p.N = q.out.cols;
    p.steps = ceil_div(q.K, kStep);
    p.tiles_m = ceil_div(p.M, 256);
    p.tiles_n = ceil_div(p.N, BN);
    p.per = (int)tiles_of(p.M, p.N, BN, q.symmetric);
    p.first = (int)units;
    p.symmetric = q.symmetric;
    p.l_mn = q.l_mn;
    p.r_mn = q.r_mn;
    p.alpha = (float)q.alpha;
    p.beta = (float)q.beta;
    p.add = q.add ? q.add->p : nullptr;
    p.out = q.out.p;
    p.ld = q.out.ld;
    p.plane = q.out.plane();
    p.matrix = q.out.matrix();
    units += (long long)p.per * q.out.count;
  }
  if (units > 0x3fffffff) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_step: the matrices are too large");
  all.units = (int)units;
  all.early = 2 * units <= pairs;
  const auto kern = newton_kernel<BN, CAP>;
  B200CP_CUDA_OK((allow_smem<newton_kernel<BN, CAP>>((int)T::smem)));
  B200CP_CUDA_OK(launch_kernel(kern, dim3((unsigned)(2 * std::min<long long>(units, pairs))), dim3(T::threads), T::smem, st, true, all));
  B200CP_LAUNCH_OK("newton_kernel");
  return B200CP_OK;
}
template <int BN>
int launch_products(const std::vector<Product>& ps, Maps& maps, int pairs, cudaStream_t st) {
  return ps.size() <= kFewProblems ? launch_table<BN, kFewProblems>(ps, maps, pairs, st) : launch_table<BN, kProblems>(ps, maps, pairs, st);
}
// One launch for all, the longest sums first.  Tiles of 256 columns, or of 128 where those fill the pairs of CTAs better: a narrow tile takes 0.55 of a wide
// one, so 4096 x 4096 goes in seven rounds of narrow ones, not in four of wide ones (279 us a product, and 350); 4096 x 10240 in nine of wide
// ones, not in 18.
int products(std::vector<Product> ps, Maps& maps, const DeviceInfo& di, cudaStream_t st) {
  const int pairs = di.sm_count / 2;
  std::stable_sort(ps.begin(), ps.end(), [](const Product& a, const Product& b) { return a.K > b.K; });
  long long tiles[2] = {};
  for (const Product& p : ps)
    for (int i = 0; i < 2; ++i) tiles[i] += tiles_of(p.out.rows, p.out.cols, 128 << i, p.symmetric) * p.out.count;
  const auto rounds = [&](long long n) { return (double)((n + pairs - 1) / pairs); };
  return rounds(tiles[1]) <= 0.55 * rounds(tiles[0]) ? launch_products<256>(ps, maps, pairs, st) : launch_products<128>(ps, maps, pairs, st);
}

// ---- bounds on the singular values, and the scales of the planes that follow ----------------------------------------------------------
double grown(double bound, const double* v) {   // the largest |a s + b s^3 + c s^5| for s up to bound
  const auto at = [&](double y) { return std::fabs(std::sqrt(y) * (v[0] + y * (v[1] + y * v[2]))); };
  double most = at(bound * bound);
  const double A = 5 * v[2], B = 3 * v[1], C = v[0], D = B * B - 4 * A * C;   // of the derivative in y = s^2
  const auto look = [&](double y) {
    if (y > 0 && y < bound * bound) most = std::max(most, at(y));
  };
  if (A == 0) {
    if (B != 0) look(-C / B);
  } else if (D >= 0) {
    look((-B + std::sqrt(D)) / (2 * A));
    look((-B - std::sqrt(D)) / (2 * A));
  }
  return most;
}
double room_for(double bound) { return std::ldexp(1.0, 15 - (int)std::ceil(std::log2(bound))); }   // bound times it is at most 2^15
constexpr double kMostGrowth = 1024;   // of a direction with a small singular value, in a run of steps on A
struct Plan {
  int steps, coefficients;
  const double* v;
  double bound[101];
  int runs, run[101];        // of the small matrices: where each begins, and the end
};
int plan_of(const char* who, const b200cp_muon* h, Plan* p) {
  if (h->steps < 0 || h->steps > 100 || (h->steps && !h->coefficients) || (h->coefficient_count != 1 && h->coefficient_count != h->steps))
    return fail(B200CP_ERR_INVALID_ARG, "%s: %d steps (0 to 100) with %d triples of coefficients (1, or one for each step)", who, h->steps, h->coefficient_count);
  if (!(h->momentum >= 0 && h->momentum <= 1 && h->eps > 0)) return fail(B200CP_ERR_INVALID_ARG, "%s: momentum %g or eps %g out of range", who, h->momentum, h->eps);
  p->steps = h->steps;
  p->coefficients = h->coefficient_count;
  p->v = h->coefficients;
  p->bound[0] = 1.01;   // (a hundredth for what is rounded)
  for (int s = 0; s < p->steps; ++s) {
    const double b = grown(p->bound[s], p->v + (p->coefficients > 1 ? 3 * s : 0)) * 1.01;
    if (!(b <= 100.0)) return fail(B200CP_ERR_UNSUPPORTED, "%s: these coefficients may raise a singular value above 100 in step %d", who, s + 1);
    p->bound[s + 1] = std::max(b, 1e-3);
  }
  p->runs = 0;
  p->run[0] = 0;
  double growth = 1;
  for (int s = 0; s < p->steps; ++s) {
    const double a = std::max(1.0, std::fabs(p->v[p->coefficients > 1 ? 3 * s : 0]));
    if (s > p->run[p->runs] && growth * a > kMostGrowth) {
      p->run[++p->runs] = s;
      growth = 1;
    }
    growth *= a;
  }
  p->run[++p->runs] = p->steps;
  return B200CP_OK;
}

// ---- which matrices go together --------------------------------------------------------------------------------------------------------
bool small(const b200cp_muon_matrix& a) { return std::min(a.rows, a.cols) <= kSmall; }
int tile_side(int n) { return n <= 16 ? 1 : n <= 32 ? 2 : 4; }
struct SmallSizes {
  size_t doubles = 0, floats = 0, values = 0;   // of parts of A; of Q; of X between two runs of steps
  int matrices = 0, ctas = 0;
};
// What a CTA takes at a time of a matrix's longer side, and how many such turns there are.
int turn_of(const b200cp_muon_matrix& a) { return 2048 / (16 * tile_side(std::min(a.rows, a.cols))); }
int turns_of(const b200cp_muon_matrix& a) { return ceil_div(std::max(a.rows, a.cols), turn_of(a)); }
// Parts of a matrix: its share, by its turns, of the CTAs that the SMs hold (slots), so that the call is one round of CTAs that all have about as many turns; and no more than are
// added (one after another, by the CTAs that take the matrix's steps) in the time that they save: 64 x 8192 takes 50 us in 64 parts, 45 in 128, 49 in 256.
void cut_small(const b200cp_muon_matrix& a, long long all, int slots, SmallEntry* e, SmallSizes* s) {
  const int n = std::min(a.rows, a.cols), len = std::max(a.rows, a.cols), ts = tile_side(n), sub = turn_of(a), turns = turns_of(a);
  const int most = (int)std::ceil(8 * std::sqrt((double)turns));
  const int parts = (int)std::min<long long>({turns, most, std::max<long long>(1, (long long)slots * turns / all)});
  e->rows = a.rows; e->cols = a.cols; e->stack = a.stack;
  e->length = ceil_div(turns, parts) * sub;
  e->chunks = ceil_div(len, e->length);
  e->first = s->ctas;
  e->matrix = s->matrices;
  e->gram = s->doubles;
  e->q = s->floats;
  s->ctas += e->chunks * a.stack;
  s->matrices += a.stack;
  s->doubles += (size_t)a.stack * e->chunks * kPart[ts];
  s->floats += (size_t)a.stack * n * n;
  s->values += align_up((size_t)a.stack * a.rows * a.cols, 64);
}
size_t small_bytes(const SmallSizes& s, bool several_runs) {
  return align_up(s.doubles * 8, 256) + align_up((size_t)s.matrices * 8, 256) + align_up(s.floats * 4, 256) + (several_runs ? s.values * 4 : 0);
}
// Small matrices of a launch: tensors (of stacks, at most kMostStack matrices) from `at` on, up to a table's size, 2^20 CTAs and 256 MB of parts.
int next_small(const std::vector<b200cp_muon_matrix>& ms, size_t at, long long all, int slots, SmallTable<kTableSmall>* t, SmallSizes* s) {
  int count = 0;
  while (at + count < ms.size() && count < kTableSmall && s->ctas < (1 << 20) && s->doubles < (size_t)1 << 25) {
    SmallEntry e{};
    cut_small(ms[at + count], all, slots, &e, s);
    const b200cp_muon_matrix& a = ms[at + count];
    e.at = Pointers{a.param, a.grad, a.momentum, a.master};
    const auto off = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; };
    e.vec = a.cols % 4 == 0 && !(off(a.param) | off(a.grad) | off(a.momentum) | off(a.master));
    if (t) t->e[count] = e;
    ++count;
  }
  return count;
}
struct Shape {
  int rows, cols;
  std::vector<Pointers> at;
};
size_t type_size(int type) { return type == B200CP_FLOAT32 ? 4 : 2; }
constexpr int kMostStack = 4096;
struct Work {
  std::vector<b200cp_muon_matrix> little;   // those with sides above 32 first
  long long turns = 0;      // of small ones
  int widest = 1;           // 1: all of them have a side of at most 16; or 4
  std::vector<Shape> large;
  Work(const b200cp_muon_matrix* ms, int count, int ptype, int gtype) {
    for (int i = 0; i < count; ++i) {
      const b200cp_muon_matrix& a = ms[i];
      if (a.stack < 1 || a.rows < 1 || a.cols < 1) continue;
      const size_t n = (size_t)a.rows * a.cols;
      const auto part = [&](int k, int stack) {   // of a stack, from matrix k on
        const auto on = [&](auto* p, size_t size) { return p ? (decltype(p))((char*)p + k * n * size) : p; };
        return b200cp_muon_matrix{on(a.param, type_size(ptype)), on(a.grad, type_size(gtype)), on(a.momentum, 4), on(a.master, 4), stack, a.rows, a.cols};
      };
      if (small(a)) {
        for (int k = 0; k < a.stack; k += kMostStack) little.push_back(part(k, std::min(kMostStack, a.stack - k)));
        turns += (long long)a.stack * turns_of(a);
        if (tile_side(std::min(a.rows, a.cols)) > 1) widest = 4;
        continue;
      }
      auto s = std::find_if(large.begin(), large.end(), [&](const Shape& q) { return q.rows == a.rows && q.cols == a.cols; });
      if (s == large.end()) {
        large.push_back(Shape{a.rows, a.cols, {}});
        s = large.end() - 1;
      }
      for (int k = 0; k < a.stack; ++k) {
        const b200cp_muon_matrix q = part(k, 1);
        s->at.push_back(Pointers{q.param, q.grad, q.momentum, q.master});
      }
    }
    std::stable_partition(little.begin(), little.end(), [](const b200cp_muon_matrix& a) { return tile_side(std::min(a.rows, a.cols)) == 4; });
  }
};
// Larger matrices that share launches: parts of shapes, as the tables and some memory hold them.
struct Share {
  const Shape* s;
  int first, count;
};
struct ShareSizes {
  size_t x, a;   // bytes of the planes of X, of a square matrix
};
ShareSizes share_sizes(const Shape& s, int count) {
  const size_t n = std::min(s.rows, s.cols);
  return ShareSizes{align_up((size_t)count * 4 * s.rows * pitch_of(s.cols), 256), align_up((size_t)count * 4 * n * pitch_of((int)n), 256)};
}
size_t share_bytes(const Share& s) {
  const ShareSizes z = share_sizes(*s.s, s.count);
  return 2 * z.x + 2 * z.a;
}
std::vector<std::vector<Share>> rounds_of(const Work& w) {
  constexpr size_t kRoom = (size_t)3 << 29;   // 1.5 GB, or one matrix
  std::vector<std::vector<Share>> out(1);
  size_t used = 0;
  int items = 0;
  for (const Shape& s : w.large) {
    const size_t each = share_bytes(Share{&s, 0, 1});
    for (int first = 0; first < (int)s.at.size();) {
      if (items == kItems || (int)out.back().size() == kProblems || (items && used + each > kRoom)) {
        out.emplace_back();
        used = 0;
        items = 0;
      }
      const size_t room = used < kRoom ? (kRoom - used) / each : 0;
      const int count = (int)std::min<size_t>({s.at.size() - first, (size_t)(kItems - items), std::max<size_t>(1, room)});
      out.back().push_back(Share{&s, first, count});
      used += each * count;
      items += count;
      first += count;
    }
  }
  if (out.back().empty()) out.pop_back();
  return out;
}
size_t round_bytes(const std::vector<Share>& round) {
  size_t n = align_up((size_t)kItems * kNormParts * 8, 256);
  for (const Share& s : round) n += share_bytes(s);
  return n;
}
size_t workspace_of(const Work& w, int sm_count, bool several_runs) {
  size_t most = 0;
  for (size_t at = 0; at < w.little.size();) {
    SmallSizes s;
    at += next_small(w.little, at, w.turns, per_sm(w.widest) * sm_count, nullptr, &s);
    most = std::max(most, small_bytes(s, several_runs));
  }
  for (const std::vector<Share>& r : rounds_of(w)) most = std::max(most, round_bytes(r));
  return most;
}
float factor_of(int adjust, int rows, int cols) {
  if (adjust == B200CP_MUON_ORIGINAL) return (float)std::sqrt(std::max(1.0, (double)rows / cols));
  if (adjust == B200CP_MUON_MATCH_RMS_ADAMW) return (float)(0.2 * std::sqrt((double)std::max(rows, cols)));
  return 1.f;
}

template <typename G, int W, int CAP>
int launch_gram(const SmallTable<CAP>& t, const SmallSizes& s, int ts, cudaStream_t st) {
  // (each as much as the widest matrix of the launch needs; the others need less)
  const int gram = std::max({gram_doubles(1), ts > 1 ? gram_doubles(2) : 0, ts > 2 ? gram_doubles(4) : 0}) * 8;
  B200CP_CUDA_OK((allow_smem<muon_gram_kernel<G, W, CAP>>(gram)));
  B200CP_CUDA_OK(launch_kernel(muon_gram_kernel<G, W, CAP>, dim3(s.ctas), dim3(256), gram, st, true, t));
  B200CP_LAUNCH_OK("muon_gram_kernel");
  return B200CP_OK;
}
template <int CAP>
int launch_iterate(const SmallTable<CAP>& t, const Coefficients& co, const SmallSizes& s, int ts, int sm_count, cudaStream_t st) {
  const int five = 5 * 16 * ts * (16 * ts + 4) * 8;
  int wide = 0;   // (they are the first ones)
  for (int i = 0; i < t.count; ++i) wide += tile_side(std::min(t.e[i].rows, t.e[i].cols)) == 4 ? t.e[i].stack : 0;
  const int shared = ceil_div(s.matrices + (kShare - 1) * wide, kShare) * kShare;
  if (wide && shared <= sm_count) {
    B200CP_CUDA_OK(allow_smem<muon_iterate_shared_kernel<CAP>>(five));
    B200CP_CUDA_OK(launch_kernel(muon_iterate_shared_kernel<CAP>, dim3(shared), dim3(kIterateThreads), five, st, true, t, co, wide, s.matrices));
  } else {
    const auto steps = [&](auto kernel, auto allow) {
      B200CP_CUDA_OK(allow(five));
      B200CP_CUDA_OK(launch_kernel(kernel, dim3(s.matrices), dim3(kIterateThreads), five, st, true, t, co));
      return (int)B200CP_OK;
    };
    const int rc = ts == 1   ? steps(muon_iterate_kernel<1, CAP>, allow_smem<muon_iterate_kernel<1, CAP>>)
                   : ts == 2 ? steps(muon_iterate_kernel<2, CAP>, allow_smem<muon_iterate_kernel<2, CAP>>)
                             : steps(muon_iterate_kernel<4, CAP>, allow_smem<muon_iterate_kernel<4, CAP>>);
    if (rc) return rc;
  }
  B200CP_LAUNCH_OK("muon_iterate_kernel");
  return B200CP_OK;
}
template <typename P, typename G, int W, int CAP>
int launch_apply(const SmallTable<CAP>& t, const SmallSizes& s, int ts, cudaStream_t st) {
  const int low = std::max({small_apply_floats(1), ts > 1 ? small_apply_floats(2) : 0, ts > 2 ? small_apply_floats(4) : 0}) * 4;
  B200CP_CUDA_OK((allow_smem<muon_small_apply_kernel<P, G, W, CAP>>(low)));
  B200CP_CUDA_OK(launch_kernel(muon_small_apply_kernel<P, G, W, CAP>, dim3(s.ctas), dim3(256), low, st, true, t));
  B200CP_LAUNCH_OK("muon_small_apply_kernel");
  return B200CP_OK;
}
// x: where X lies between two runs of steps.
template <typename P, typename G, int W, int CAP>
int launch_small(const SmallHead& head, const SmallEntry* e, const Plan& plan, const Coefficients& co, const SmallSizes& s, float* x, int sm_count, cudaStream_t st) {
  SmallTable<CAP> t;
  static_cast<SmallHead&>(t) = head;
  std::copy(e, e + head.count, t.e);
  int ts = 1;
  for (int i = 0; i < t.count; ++i) ts = std::max(ts, tile_side(std::min(t.e[i].rows, t.e[i].cols)));
  for (int run = 0; run < plan.runs; ++run) {
    const bool first = run == 0, last = run + 1 == plan.runs;
    t.first_step = plan.run[run];
    t.steps = plan.run[run + 1] - t.first_step;
    t.normed = !first;
    t.r.update = last && head.r.update;
    float* at = x;
    for (int i = 0; i < t.count; ++i) {   // (X is replaced in place: a CTA stores the values that it has read)
      Pointers& to = t.e[i].at;
      to = e[i].at;
      if (!first) {
        to.g = at;
        to.m = nullptr;
      }
      if (!last) to.p = at;
      at += align_up((size_t)e[i].stack * e[i].rows * e[i].cols, 64);
    }
    if (int rc = first ? launch_gram<G, W, CAP>(t, s, ts, st) : launch_gram<float, W, CAP>(t, s, ts, st)) return rc;
    if (int rc = launch_iterate<CAP>(t, co, s, ts, sm_count, st)) return rc;
    if (int rc = first ? (last ? launch_apply<P, G, W, CAP>(t, s, ts, st) : launch_apply<float, G, W, CAP>(t, s, ts, st))
                       : (last ? launch_apply<P, float, W, CAP>(t, s, ts, st) : launch_apply<float, float, W, CAP>(t, s, ts, st)))
      return rc;
  }
  return B200CP_OK;
}
template <typename P, typename G>
int run_small(const Work& w, const Rates& r, const Plan& plan, int adjust, char* ws, const DeviceInfo& di, cudaStream_t st) {
  Coefficients co;
  if (plan.steps) std::copy(plan.v, plan.v + 3 * plan.coefficients, co.v);
  SmallTable<kTableSmall> t;
  for (size_t at = 0; at < w.little.size();) {
    SmallSizes s;
    t.count = next_small(w.little, at, w.turns, per_sm(w.widest) * di.sm_count, &t, &s);
    at += t.count;
    t.r = r;
    t.coefficients = plan.coefficients;
    char* to = ws;
    t.gram = reinterpret_cast<double*>(to);
    t.inverse = reinterpret_cast<double*>(to += align_up(s.doubles * 8, 256));
    t.q = reinterpret_cast<float*>(to += align_up((size_t)s.matrices * 8, 256));
    float* x = reinterpret_cast<float*>(to += align_up(s.floats * 4, 256));
    for (int i = 0; i < t.count; ++i) t.e[i].scale = factor_of(adjust, t.e[i].rows, t.e[i].cols);
    const bool few = t.count <= kFewSmall;
    const int rc = w.widest == 1 ? (few ? launch_small<P, G, 1, kFewSmall>(t, t.e, plan, co, s, x, di.sm_count, st) : launch_small<P, G, 1, kTableSmall>(t, t.e, plan, co, s, x, di.sm_count, st))
                                 : (few ? launch_small<P, G, 4, kFewSmall>(t, t.e, plan, co, s, x, di.sm_count, st) : launch_small<P, G, 4, kTableSmall>(t, t.e, plan, co, s, x, di.sm_count, st));
    if (rc) return rc;
  }
  return B200CP_OK;
}

// (Taking the last steps on A, as the small matrices do, is 20 % less work for sides of 1 to 2.5, but Q then raises what X lacks by 41 while it leaves what X has:
// sums that cancel, where the tensor core's cut sums show.  A gradient of rank one came out 1e-3 off, of these forms 3e-5.)
struct Large {
  Planes X, Y, A, B;
  bool wide;
  int n, len;
};
template <typename P, typename G, int CAP>
int run_large(const std::vector<Share>& round, const Rates& r, const Plan& plan, int adjust, char* ws, const DeviceInfo& di, cudaStream_t st) {
  Items<CAP> t;
  t.r = r;
  t.count = 0;
  t.norms = reinterpret_cast<double*>(ws);
  ws += align_up((size_t)kItems * kNormParts * 8, 256);
  double sx = room_for(plan.bound[0]);
  t.scale = (float)sx;
  std::vector<Large> ms;
  long long ctas = 0, ctas8 = 0;
  int norm = 0;
  for (const Share& q : round) {
    const Shape& s = *q.s;
    const ShareSizes z = share_sizes(s, q.count);
    Large m;
    m.n = std::min(s.rows, s.cols);
    m.len = std::max(s.rows, s.cols);
    m.wide = s.rows <= s.cols;
    const auto half = [&](size_t at) { return reinterpret_cast<__half*>(ws + at); };
    m.X = Planes{half(0), s.rows, s.cols, pitch_of(s.cols), q.count};
    m.Y = m.X;
    m.Y.p = half(z.x);
    m.A = Planes{half(2 * z.x), m.n, m.n, pitch_of(m.n), q.count};
    m.B = m.A;
    m.B.p = half(2 * z.x + z.a);
    ws += share_bytes(q);
    const long long values = (long long)s.rows * s.cols, groups = (long long)s.rows * ((s.cols + 7) / 8);
    const long long chunk = std::max<long long>(kTurn, (values + kNormParts * 2048LL - 1) / (kNormParts * 2048LL) * 2048);
    if (chunk > 0x7fffffff) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_step: a matrix of %d x %d", s.rows, s.cols);
    for (int i = 0; i < q.count; ++i) {
      Item& e = t.e[t.count++];
      e.at = s.at[q.first + i];
      e.rows = s.rows;
      e.cols = s.cols;
      e.ld = m.X.ld;
      e.plane = m.X.plane();
      e.x = m.X.p + i * m.X.matrix();
      e.vec = s.cols % 8 == 0 && !((reinterpret_cast<uintptr_t>(e.at.p) | reinterpret_cast<uintptr_t>(e.at.g) | reinterpret_cast<uintptr_t>(e.at.m) |
                                    reinterpret_cast<uintptr_t>(e.at.w)) & 15);
      e.first = (int)ctas;
      e.chunk = (int)chunk;
      e.parts = (int)((values + chunk - 1) / chunk);
      e.norm = norm;
      e.first8 = (int)ctas8;
      e.rate = factor_of(adjust, s.rows, s.cols);
      ctas += e.parts;
      ctas8 += (groups + 1023) / 1024;
      norm += e.parts;
    }
    ms.push_back(m);
  }
  if (ctas8 > 0x7fffffff) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_step: the matrices are too large");
  B200CP_CUDA_OK(launch_kernel(muon_momentum_kernel<G, CAP>, dim3((unsigned)ctas), dim3(256), 0, st, true, t));
  B200CP_LAUNCH_OK("muon_momentum_kernel");
  B200CP_CUDA_OK(launch_kernel(muon_planes_kernel<G, CAP>, dim3((unsigned)ctas8), dim3(256), 0, st, true, t));
  B200CP_LAUNCH_OK("muon_planes_kernel");
  Maps maps;
  for (int step = 0; step < plan.steps; ++step) {
    const double* v = plan.v + (plan.coefficients > 1 ? 3 * step : 0);
    const double y = plan.bound[step] * plan.bound[step], sa = room_for(y),
                 sb = room_for(std::max(1e-3, std::fabs(v[1]) * y + std::fabs(v[2]) * y * y)), sn = room_for(plan.bound[step + 1]);
    std::vector<Product> ps;
    for (Large& m : ms) ps.push_back(Product{m.X, m.X, m.A, !m.wide, !m.wide, true, m.len, sa / (sx * sx), 0, nullptr});
    if (int rc = products(ps, maps, di, st)) return rc;
    ps.clear();
    for (Large& m : ms) ps.push_back(Product{m.A, m.A, m.B, false, false, true, m.n, v[2] * sb / (sa * sa), v[1] * sb / sa, &m.A});
    if (int rc = products(ps, maps, di, st)) return rc;
    ps.clear();
    for (Large& m : ms)
      ps.push_back(m.wide ? Product{m.B, m.X, m.Y, false, true, false, m.n, sn / (sb * sx), v[0] * sn / sx, &m.X}
                          : Product{m.X, m.B, m.Y, false, false, false, m.n, sn / (sb * sx), v[0] * sn / sx, &m.X});
    if (int rc = products(ps, maps, di, st)) return rc;
    for (Large& m : ms) std::swap(m.X, m.Y);
    sx = sn;
  }
  t.scale = (float)sx;
  int at = 0;
  for (const Large& m : ms)
    for (int i = 0; i < m.X.count; ++i) t.e[at++].x = m.X.p + i * m.X.matrix();
  B200CP_CUDA_OK(launch_kernel(muon_apply_kernel<P, CAP>, dim3((unsigned)ctas8), dim3(256), 0, st, true, t));
  B200CP_LAUNCH_OK("muon_apply_kernel");
  return B200CP_OK;
}

template <typename P, typename G>
int run(const Work& w, const Rates& r, const Plan& plan, int adjust, char* ws, cudaStream_t st) {
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  if (int rc = run_small<P, G>(w, r, plan, adjust, ws, di, st)) return rc;
  for (const std::vector<Share>& round : rounds_of(w)) {
    int items = 0;
    for (const Share& s : round) items += s.count;
    if (int rc = items <= kFewItems ? run_large<P, G, kFewItems>(round, r, plan, adjust, ws, di, st) : run_large<P, G, kItems>(round, r, plan, adjust, ws, di, st))
      return rc;
  }
  return B200CP_OK;
}

int check_muon(const char* who, const b200cp_muon_matrix* ms, int count, int ptype, int gtype) {
  if (count < 0 || (count && !ms)) return fail(B200CP_ERR_INVALID_ARG, "%s: null argument or negative count", who);
  if (ptype < B200CP_FLOAT32 || ptype > B200CP_FLOAT16 || (gtype != ptype && gtype != B200CP_FLOAT32))
    return fail(B200CP_ERR_UNSUPPORTED, "%s: parameters of type %d with gradients of type %d", who, ptype, gtype);
  for (int i = 0; i < count; ++i) {
    const b200cp_muon_matrix& a = ms[i];
    if (a.stack < 0 || a.rows < 0 || a.cols < 0) return fail(B200CP_ERR_INVALID_ARG, "%s: matrix %d is %d x %d x %d", who, i, a.stack, a.rows, a.cols);
    if (a.rows > (1 << 24) || a.cols > (1 << 24) || (long long)std::min(a.rows, a.cols) > (1 << 17))
      return fail(B200CP_ERR_UNSUPPORTED, "%s: matrix %d is %d x %d (sides up to 2^24, the smaller one up to 2^17)", who, i, a.rows, a.cols);
  }
  return B200CP_OK;
}
int muon(const char* who, const b200cp_muon_matrix* ms, int count, int ptype, int gtype, const b200cp_muon* h, bool update, void* workspace, size_t bytes,
         void* stream) {
  if (!h) return fail(B200CP_ERR_INVALID_ARG, "%s: null argument", who);
  if (int rc = check_muon(who, ms, count, ptype, gtype)) return rc;
  Plan plan;
  if (int rc = plan_of(who, h, &plan)) return rc;
  for (int i = 0; i < count; ++i) {
    const b200cp_muon_matrix& a = ms[i];
    if (a.stack && a.rows && a.cols && (!a.param || !a.grad || (update && !a.momentum))) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer in matrix %d", who, i);
    if (a.master && ptype == B200CP_FLOAT32) return fail(B200CP_ERR_INVALID_ARG, "%s: a float32 parameter has no float32 copy (matrix %d)", who, i);
  }
  const Work w(ms, count, ptype, gtype);
  if (w.little.empty() && w.large.empty()) return B200CP_OK;
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  const size_t need = workspace_of(w, di.sm_count, plan.runs > 1);
  if (need && (!workspace || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, %zu given", who, need, bytes);
  Rates r{};
  r.keep = (float)h->momentum; r.blend = (float)(1 - h->momentum);
  r.nesterov = h->nesterov != 0; r.update = update;
  r.lr = (float)h->lr; r.decay = (float)h->weight_decay;
  r.device_lr = h->device_lr;
  r.eps = h->eps;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
#define TYPES(P, G) return run<P, G>(w, r, plan, h->adjust, ws, st)
  if (ptype == B200CP_FLOAT32) TYPES(float, float);
  if (ptype == B200CP_BFLOAT16 && gtype == B200CP_BFLOAT16) TYPES(__nv_bfloat16, __nv_bfloat16);
  if (ptype == B200CP_FLOAT16 && gtype == B200CP_FLOAT16) TYPES(__half, __half);
  if (ptype == B200CP_BFLOAT16) TYPES(__nv_bfloat16, float);
  TYPES(__half, float);
#undef TYPES
}

}  // namespace

int muon_device_status(int* out) {
  int v = 0, zero = 0;
  B200CP_CUDA_OK(cudaMemcpyFromSymbol(&v, g_muon_status, sizeof(int)));
  if (v) B200CP_CUDA_OK(cudaMemcpyToSymbol(g_muon_status, &zero, sizeof(int)));
  *out = v;
  return B200CP_OK;
}

}  // namespace b200cp

using namespace b200cp;

extern "C" {

// (A list of matrices takes host memory: what that throws does not leave the library.)
size_t b200cp_muon_step_workspace_bytes(const b200cp_muon_matrix* matrices, int count, int param_type, int grad_type) try {
  if (check_muon("b200cp_muon_step_workspace_bytes", matrices, count, param_type, grad_type)) return 0;
  DeviceInfo di;
  if (device_info(&di)) return 0;
  return workspace_of(Work(matrices, count, param_type, grad_type), di.sm_count, true);
} catch (const std::exception& e) {
  fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_step_workspace_bytes: %s", e.what());
  return 0;
}

size_t b200cp_muon_workspace_bytes(const b200cp_muon_matrix* matrices, int count, int param_type, int grad_type, const b200cp_muon* hyper) try {
  const char* who = "b200cp_muon_workspace_bytes";
  Plan plan;
  DeviceInfo di;
  if (!hyper || check_muon(who, matrices, count, param_type, grad_type) || plan_of(who, hyper, &plan) || device_info(&di)) return 0;
  return workspace_of(Work(matrices, count, param_type, grad_type), di.sm_count, plan.runs > 1);
} catch (const std::exception& e) {
  fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_workspace_bytes: %s", e.what());
  return 0;
}

int b200cp_muon_step(const b200cp_muon_matrix* matrices, int count, int param_type, int grad_type, const b200cp_muon* hyper, void* workspace,
                     size_t workspace_bytes, void* stream) try {
  const char* who = "b200cp_muon_step";
  if (hyper && (hyper->adjust < B200CP_MUON_PLAIN || hyper->adjust > B200CP_MUON_MATCH_RMS_ADAMW))
    return fail(B200CP_ERR_INVALID_ARG, "%s: adjust %d", who, hyper->adjust);
  return muon(who, matrices, count, param_type, grad_type, hyper, true, workspace, workspace_bytes, stream);
} catch (const std::exception& e) {
  return fail(B200CP_ERR_UNSUPPORTED, "b200cp_muon_step: %s", e.what());
}

int b200cp_orthogonalise(int stack, int rows, int cols, int type, const void* X, void* out, const double* coefficients, int coefficient_count, int steps,
                         double eps, void* workspace, size_t workspace_bytes, void* stream) try {
  const b200cp_muon_matrix m{out, X, nullptr, nullptr, stack, rows, cols};
  b200cp_muon h{};
  h.eps = eps;
  h.steps = steps;
  h.coefficients = coefficients;
  h.coefficient_count = coefficient_count;
  return muon("b200cp_orthogonalise", &m, 1, type, type, &h, false, workspace, workspace_bytes, stream);
} catch (const std::exception& e) {
  return fail(B200CP_ERR_UNSUPPORTED, "b200cp_orthogonalise: %s", e.what());
}

}  // extern "C"
