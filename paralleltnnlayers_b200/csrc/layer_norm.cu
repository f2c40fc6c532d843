// Layer norm of rows, with the residual that is added first, and its gradients.
//
//   h = x (+ r, rounded to the type), mu = mean(h), v = mean((h - mu)^2), y = (h - mu) / sqrt(v + eps) w + b
//   n = (h - mu) rstd, g = dy w:  dh = rstd (g - mean(g) - n mean(g n)) (+ what came to h itself), dw = sum over rows of dy n, db = sum of dy
//
// Bound by HBM.  A row stays in registers from its load to its store, and its variance is that of the deviations from the mean, corrected for
// the mean's own rounding: no second pass over memory and no difference of large sums.  Rows of up to 256 features belong to a warp, others to a CTA,
// 8 to 32 features a thread.
//
// The gradients are one kernel too: a CTA walks over its rows with the sums of dw and db of its threads' features in registers (16 features a
// thread, rows of up to 8192); the next rows come by bulk copies into a ring in shared memory meanwhile (rows that do not lie on 16-byte boundaries, up to 4096, and those of
// up to 256 features, into registers, one ahead, 8 features a thread).  The CTAs' sums are added by a second launch in their order, so that a result has the same bits each
// time.  Longer rows are read twice: for dh and for the sums over rows.  Every wait is bounded: one that runs out sets a status word, and leaves what comes behind it unwritten.
#include <algorithm>

#include "common.cuh"
#include "tc_common.cuh"
#include "vec_io.cuh"

namespace b200cp {

__device__ int g_layer_norm_status = 0;   // 0 ok; otherwise (code << 16) | (block index & 0xffff)

namespace {

constexpr int kWarpRow = 256;        // features of a row that a warp takes
constexpr int kRows = 8;             // rows, and warps, of a CTA then
constexpr int kGradRow = 8192;       // of a row whose gradients are one pass
constexpr int kGradEach = 16;        // of them to a thread (8 where they do not lie on 16-byte boundaries, and in short rows: those keep a row ahead in registers)
constexpr int kGradThreads = kGradRow / kGradEach;   // of a CTA at most, and of an SM at 128 registers each

// Sums of two values over a warp: of the first one in lanes 0 to 15, of the second in the others.
__device__ __forceinline__ float half_sums(float a, float b) {
  const bool up = threadIdx.x & 16;
  float s = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
  for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ float2 both(float s) { return make_float2(__shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, s, 16)); }
// Sums over the CTA of two values: `red` holds 2 x 2 x 32 of the warps', used in turn (`turn` changes between calls), so that one barrier is enough.
constexpr int kRed = 128;
__device__ __forceinline__ float2 block_sum(float a, float b, float* red, int turn) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, i = lane & 15;
  float* r = red + turn * 64 + (lane & 16) * 2;   // (this half's)
  const float s = half_sums(a, b);
  if (i == 0) r[threadIdx.x >> 5] = s;
  __syncthreads();
  float v = i < warps ? r[i] : 0.f;
  if (warps > 16 && i + 16 < warps) v += r[i + 16];
#pragma unroll
  for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return both(v);
}
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float a, float b, float* red, int turn) {
  if constexpr (WARP) return both(half_sums(a, b));
  return block_sum(a, b, red, turn);
}

// (rounding may leave a variance below 0; one that is not a number stays that)
__device__ __forceinline__ float rstd_of(float variance, float eps) { return 1.f / sqrtf((variance < 0.f ? 0.f : variance) + eps); }

struct Forward {
  int rows, D;
  float eps;
  const void *x, *r, *w, *b;
  void *y, *h;
  float *mean, *rstd;
};
template <typename T, typename W, int VEC, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kRows : 1024) norm_kernel(const __grid_constant__ Forward g) {
  __shared__ float red[kRed];
  const int row = WARP ? blockIdx.x * kRows + (threadIdx.x >> 5) : blockIdx.x, t = WARP ? threadIdx.x & 31 : threadIdx.x, n = WARP ? 32 : blockDim.x;
  grid_dependency_wait();
  if (WARP && row >= g.rows) return;
  const size_t at = (size_t)row * g.D;
  const T* x = static_cast<const T*>(g.x) + at;
  Group<T, VEC> p[K];
  float v[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
    if (c < g.D) p[k] = load_group<T, VEC>(x + c);
  }
  if (g.r) {
    const T* r = static_cast<const T*>(g.r) + at;
    T* h = static_cast<T*>(g.h) + at;
    Group<T, VEC> q[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c < g.D) q[k] = load_group<T, VEC>(r + c);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c >= g.D) continue;
      float a[VEC], b[VEC];
      unpack(p[k], a);
      unpack(q[k], b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] += b[i];
      p[k] = pack<T>(a);
      store_group(h + c, p[k]);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool in = (k * n + t) * VEC < g.D;
    if (in) unpack(p[k], v[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (!in) v[k][i] = 0.f;
      s += v[k][i];
    }
  }
  const float inv = 1.f / (float)g.D, mean = row_sum<WARP>(s, 0.f, red, 0).x * inv;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((k * n + t) * VEC >= g.D) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[k][i] -= mean;
      s1 += v[k][i];
      s2 = fmaf(v[k][i], v[k][i], s2);
    }
  }
  const float2 q = row_sum<WARP>(s1, s2, red, 1);
  const float off = q.x * inv, rstd = rstd_of(fmaf(-off, off, q.y * inv), g.eps);
  if (g.mean && t == 0) {
    g.mean[row] = mean + off;
    g.rstd[row] = rstd;
  }
  const W *w = static_cast<const W*>(g.w), *b = static_cast<const W*>(g.b);
  T* y = static_cast<T*>(g.y) + at;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
    if (c >= g.D) continue;
    float m[VEC], a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      m[i] = 1.f;
      a[i] = 0.f;
    }
    if (w) unpack(load_group<W, VEC>(w + c), m);
    if (b) unpack(load_group<W, VEC>(b + c), a);
#pragma unroll
    for (int i = 0; i < VEC; ++i) a[i] = fmaf(fmaf(v[k][i], rstd, -off * rstd), m[i], a[i]);
    store_group(y + c, pack<T>(a));
  }
}

// Rows that a CTA does not hold: three passes, the second and third from the caches.
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(1024) norm_wide_kernel(const __grid_constant__ Forward g) {
  __shared__ float red[kRed];
  grid_dependency_wait();
  const size_t at = (size_t)blockIdx.x * g.D;
  const T *x = static_cast<const T*>(g.x) + at, *src = x;
  float s = 0.f;
  if (g.r) {   // (a thread reads back what it has stored itself)
    const T* r = static_cast<const T*>(g.r) + at;
    T* h = static_cast<T*>(g.h) + at;
    for (long long c = threadIdx.x * VEC; c < g.D; c += 1024 * VEC) {
      float a[VEC], b[VEC];
      unpack(load_group<T, VEC>(x + c), a);
      unpack(load_group<T, VEC>(r + c), b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] += b[i];
      const Group<T, VEC> p = pack<T>(a);
      store_group(h + c, p);
      unpack(p, a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += a[i];
    }
    src = h;
  } else {
    for (long long c = threadIdx.x * VEC; c < g.D; c += 1024 * VEC) {
      float a[VEC];
      unpack(load_group<T, VEC>(x + c), a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += a[i];
    }
  }
  const float inv = 1.f / (float)g.D, mean = block_sum(s, 0.f, red, 0).x * inv;
  float s1 = 0.f, s2 = 0.f;
  for (long long c = threadIdx.x * VEC; c < g.D; c += 1024 * VEC) {
    float a[VEC];
    unpack(load_group<T, VEC>(src + c), a);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = a[i] - mean;
      s1 += d;
      s2 = fmaf(d, d, s2);
    }
  }
  const float2 q = block_sum(s1, s2, red, 1);
  const float off = q.x * inv, rstd = rstd_of(fmaf(-off, off, q.y * inv), g.eps);
  if (g.mean && threadIdx.x == 0) {
    g.mean[blockIdx.x] = mean + off;
    g.rstd[blockIdx.x] = rstd;
  }
  const W *w = static_cast<const W*>(g.w), *b = static_cast<const W*>(g.b);
  T* y = static_cast<T*>(g.y) + at;
  for (long long c = threadIdx.x * VEC; c < g.D; c += 1024 * VEC) {
    float v[VEC], m[VEC], a[VEC];
    unpack(load_group<T, VEC>(src + c), v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      m[i] = 1.f;
      a[i] = 0.f;
    }
    if (w) unpack(load_group<W, VEC>(w + c), m);
    if (b) unpack(load_group<W, VEC>(b + c), a);
#pragma unroll
    for (int i = 0; i < VEC; ++i) a[i] = fmaf((v[i] - mean - off) * rstd, m[i], a[i]);
    store_group(y + c, pack<T>(a));
  }
}

// ---- gradients ----------------------------------------------------------------------------------------------------------------
struct Backward {
  int rows, D;
  const void *dy, *dh, *h, *w;
  const float *mean, *rstd;
  void* dx;          // or null
  float* partial;    // [CTA][dw, db][D], or null
};
// What a row adds to a thread's sums, and its dh.  n = (h - mean) rstd in two operations (h rstd - mean rstd, in one, rounds mean rstd: rows of one value, whose n is 0, gave
// what that rounding is, 2 at a value of 12345), dh = rstd g - rstd mean(g) - n rstd mean(g n) in two.  Instructions count
// here: 8192 x 4096 in bfloat16 with dH (HBM: 41 us) took 69 us with eight features a thread and 350 instructions a row and warp, 63 with these forms and
// sums of two values at once, and takes 53 to 55 with 16 features a thread, which halves what a row costs beside its values (115 with a row ahead in registers).
template <typename T, int VEC>
__device__ __forceinline__ void add_group(const Group<T, VEC>& h, const Group<T, VEC>& dy, const float (&w)[VEC], float mean, float rstd, float (&n)[VEC],
                                          float (&e)[VEC], float& s1, float& s2, float (&dw)[VEC], float (&db)[VEC]) {
  float x[VEC], d[VEC];
  unpack(h, x);
  unpack(dy, d);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    n[i] = (x[i] - mean) * rstd;
    e[i] = d[i] * w[i];
    s1 += e[i];
    s2 = fmaf(e[i], n[i], s2);
    dw[i] = fmaf(d[i], n[i], dw[i]);
    db[i] += d[i];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ Group<T, VEC> dx_group(const float (&n)[VEC], const float (&e)[VEC], const Group<T, VEC>* dh, float rstd, float c1, float c2) {
  float a[VEC] = {};
  if (dh) unpack(*dh, a);
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = fmaf(-n[i], c2, fmaf(e[i], rstd, a[i] - c1));
  return pack<T>(a);
}
template <typename T, int VEC, int K>
struct RowOf {   // what a thread has of a row, as it lies in memory
  Group<T, VEC> h[K], dy[K], dh[K];
  float mean, rstd;
};
template <typename T, int VEC, int K>
__device__ __forceinline__ void load_row(const Backward& g, int row, int t, int n, RowOf<T, VEC, K>& to) {
  const size_t at = (size_t)row * g.D;
  to.mean = g.mean[row];
  to.rstd = g.rstd[row];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
    if (c >= g.D) continue;
    to.h[k] = load_group<T, VEC>(static_cast<const T*>(g.h) + at + c);
    to.dy[k] = load_group<T, VEC>(static_cast<const T*>(g.dy) + at + c);
    if (g.dh && g.dx) to.dh[k] = load_group<T, VEC>(static_cast<const T*>(g.dh) + at + c);
  }
}
template <typename T, typename W, int VEC, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kRows : kGradThreads, 1) norm_grads_kernel(const __grid_constant__ Backward g) {
  __shared__ float red[kRed];
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, n = WARP ? 32 : blockDim.x;
  const int first = WARP ? blockIdx.x * kRows + (threadIdx.x >> 5) : blockIdx.x, step = WARP ? gridDim.x * kRows : gridDim.x;
  grid_dependency_wait();
  float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[k][i] = 1.f;
      dw[k][i] = db[k][i] = 0.f;
    }
    if (g.w && c < g.D) unpack(load_group<W, VEC>(static_cast<const W*>(g.w) + c), w[k]);
  }
  const float inv = 1.f / (float)g.D;
  RowOf<T, VEC, K> next;
  if (first < g.rows) load_row(g, first, t, n, next);
  int turn = 0;
  for (int row = first; row < g.rows; row += step, turn ^= 1) {
    const RowOf<T, VEC, K> now = next;
    if (row < g.rows - step) load_row(g, row + step, t, n, next);
    float s1 = 0.f, s2 = 0.f, x[K][VEC], e[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((k * n + t) * VEC < g.D) add_group(now.h[k], now.dy[k], w[k], now.mean, now.rstd, x[k], e[k], s1, s2, dw[k], db[k]);
    if (!g.dx) continue;
    const float2 q = row_sum<WARP>(s1, s2, red, turn);
    const float c1 = q.x * inv * now.rstd, c2 = q.y * inv * now.rstd;
    T* dx = static_cast<T*>(g.dx) + (size_t)row * g.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c < g.D) store_group(dx + c, dx_group(x[k], e[k], g.dh ? &now.dh[k] : nullptr, now.rstd, c1, c2));
    }
  }
  if (!g.partial) return;
  float* to = g.partial + (size_t)blockIdx.x * 2 * g.D;
  if constexpr (WARP) {   // the warps' sums, in their order
    __shared__ float all[2][kRows][kWarpRow];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (k * 32 + t) * VEC + i;
        all[0][warp][c] = dw[k][i];
        all[1][warp][c] = db[k][i];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * g.D; i += 32 * kRows) {
      const int b = i >= g.D, c = i - b * g.D;
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < kRows; ++q) s += all[b][q][c];
      to[i] = s;
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c >= g.D) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        to[c + i] = dw[k][i];
        to[g.D + c + i] = db[k][i];
      }
    }
  }
}

// The same for rows of whole 16-byte groups that a CTA shares: the rows to come are on their way into `slots` places of shared memory.
struct Ring {
  int slots, row;    // places; bytes of a row
};
__device__ __forceinline__ void bulk_load(void* to, const void* from, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(to)), "l"(from), "r"(bytes),
               "r"(tc::smem_u32(bar))
               : "memory");
}
constexpr int kMostSlots = 8;
template <typename T, typename W, int VEC, int K>
__global__ void __launch_bounds__(kGradThreads, 1) norm_grads_ring_kernel(const __grid_constant__ Backward g, const __grid_constant__ Ring ring) {
  extern __shared__ __align__(16) uint8_t places[];   // [slot][h, dy, dh][row]
  __shared__ float red[kRed];
  __shared__ uint64_t full[kMostSlots];
  __shared__ volatile int given_up[2];   // used in turn, so that all threads see the same after a barrier
  const int t = threadIdx.x, n = blockDim.x, step = gridDim.x;
  const bool added = g.dh && g.dx;
  const int arrays = added ? 3 : 2;
  if (t == 0) {
    for (int i = 0; i < ring.slots; ++i) tc::mbar_init(&full[i], 1);
    given_up[0] = given_up[1] = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  const auto fetch = [&](int row, int slot) {
    uint8_t* to = places + (size_t)slot * arrays * ring.row;
    tc::mbar_expect_tx(&full[slot], arrays * ring.row);
    bulk_load(to, static_cast<const T*>(g.h) + (size_t)row * g.D, ring.row, &full[slot]);
    bulk_load(to + ring.row, static_cast<const T*>(g.dy) + (size_t)row * g.D, ring.row, &full[slot]);
    if (added) bulk_load(to + 2 * ring.row, static_cast<const T*>(g.dh) + (size_t)row * g.D, ring.row, &full[slot]);
  };
  if (t == 0)
    for (int i = 0; i < ring.slots && (long long)blockIdx.x + (long long)i * step < g.rows; ++i) fetch(blockIdx.x + i * step, i);
  float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[k][i] = 1.f;
      dw[k][i] = db[k][i] = 0.f;
    }
    if (g.w && c < g.D) unpack(load_group<W, VEC>(static_cast<const W*>(g.w) + c), w[k]);
  }
  const float inv = 1.f / (float)g.D;
  float mean = g.mean[blockIdx.x], rstd = g.rstd[blockIdx.x];
  int turn = 0, slot = 0, phase = 0;
  for (int row = blockIdx.x; row < g.rows; row += step, turn ^= 1) {
    const float mu = mean, rs = rstd;
    const bool more = row < g.rows - step;
    if (more) {
      mean = g.mean[row + step];
      rstd = g.rstd[row + step];
    }
    if (!tc::mbar_wait(&full[slot], phase)) given_up[turn] = 1;
    const T* place = reinterpret_cast<const T*>(places + (size_t)slot * arrays * ring.row);
    Group<T, VEC> dh[K];
    float s1 = 0.f, s2 = 0.f, x[K][VEC], e[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c >= g.D) continue;
      if (added) dh[k] = load_group<T, VEC>(place + 2 * g.D + c);
      add_group(load_group<T, VEC>(place + c), load_group<T, VEC>(place + g.D + c), w[k], mu, rs, x[k], e[k], s1, s2, dw[k], db[k]);
    }
    float2 q = make_float2(0.f, 0.f);
    if (g.dx) q = block_sum(s1, s2, red, turn);
    else __syncthreads();
    if (given_up[turn]) break;
    // (all threads have taken what they need of the place)
    if (t == 0 && (long long)row + (long long)ring.slots * step < g.rows) fetch(row + ring.slots * step, slot);
    if (++slot == ring.slots) {
      slot = 0;
      phase ^= 1;
    }
    if (!g.dx) continue;
    const float c1 = q.x * inv * rs, c2 = q.y * inv * rs;
    T* dx = static_cast<T*>(g.dx) + (size_t)row * g.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * n + t) * VEC;
      if (c < g.D) store_group(dx + c, dx_group(x[k], e[k], added ? &dh[k] : nullptr, rs, c1, c2));
    }
  }
  if (given_up[0] | given_up[1]) {   // copies in flight land before the shared memory is given back
    if (t == 0) atomicCAS(&g_layer_norm_status, 0, (1 << 16) | (blockIdx.x & 0xffff));
    const long long t0 = clock64();
    while (clock64() - t0 < 40000000ll) {
    }
    return;
  }
  if (!g.partial) return;
  float* to = g.partial + (size_t)blockIdx.x * 2 * g.D;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * n + t) * VEC;
    if (c >= g.D) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      to[c + i] = dw[k][i];
      to[g.D + c + i] = db[k][i];
    }
  }
}

// Long rows: dh, a CTA per row.
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(1024) norm_wide_dx_kernel(const __grid_constant__ Backward g) {
  __shared__ float red[kRed];
  grid_dependency_wait();
  const size_t at = (size_t)blockIdx.x * g.D;
  const T *h = static_cast<const T*>(g.h) + at, *dy = static_cast<const T*>(g.dy) + at, *dh = g.dh ? static_cast<const T*>(g.dh) + at : nullptr;
  const W* w = static_cast<const W*>(g.w);
  const float mean = g.mean[blockIdx.x], rstd = g.rstd[blockIdx.x], inv = 1.f / (float)g.D;
  float s1 = 0.f, s2 = 0.f, c1 = 0.f, c2 = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (long long c = threadIdx.x * VEC; c < g.D; c += 1024 * VEC) {
      float x[VEC], d[VEC], m[VEC];
      unpack(load_group<T, VEC>(h + c), x);
      unpack(load_group<T, VEC>(dy + c), d);
      if (w) {
        unpack(load_group<W, VEC>(w + c), m);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] *= m[i];
      }
      if (pass == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s1 += d[i];
          s2 = fmaf(d[i], (x[i] - mean) * rstd, s2);
        }
      } else {
        if (dh) unpack(load_group<T, VEC>(dh + c), m);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          d[i] = rstd * (d[i] - c1 - (x[i] - mean) * rstd * c2);
          if (dh) d[i] += m[i];
        }
        store_group(static_cast<T*>(g.dx) + at + c, pack<T>(d));
      }
    }
    if (pass == 0) {
      const float2 q = block_sum(s1, s2, red, 0);
      c1 = q.x * inv;
      c2 = q.y * inv;
    }
  }
}
// Long rows: the sums over rows blockIdx.y, + gridDim.y, ... of a thread's features.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) norm_columns_kernel(const __grid_constant__ Backward g) {
  grid_dependency_wait();
  const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= g.D) return;
  float dw[VEC] = {}, db[VEC] = {};
#pragma unroll 4
  for (int row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const size_t at = (size_t)row * g.D + c;
    float x[VEC], d[VEC];
    unpack(load_group<T, VEC>(static_cast<const T*>(g.h) + at), x);
    unpack(load_group<T, VEC>(static_cast<const T*>(g.dy) + at), d);
    const float mean = g.mean[row], rstd = g.rstd[row];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      dw[i] = fmaf(d[i], (x[i] - mean) * rstd, dw[i]);
      db[i] += d[i];
    }
  }
  float* to = g.partial + (size_t)blockIdx.y * 2 * g.D + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    to[i] = dw[i];
    to[g.D + i] = db[i];
  }
}

// dw and db from the CTAs' sums: 32 columns of one of them per CTA, a warp for every 32nd part.
template <typename W>
__global__ void __launch_bounds__(1024) norm_join_kernel(int parts, int D, const float* partial, W* dw, W* db) {
  __shared__ float all[32][33];
  const int x = threadIdx.x & 31, q = threadIdx.x >> 5, groups = (D + 31) / 32, second = (int)blockIdx.x >= groups;
  const int c = ((int)blockIdx.x - second * groups) * 32 + x;
  grid_dependency_wait();
  const float* from = partial + (size_t)second * D + c;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int b = q; b < parts; b += 32) s += from[(size_t)b * 2 * D];
  }
  all[q][x] = s;
  __syncthreads();
  s = warp_sum(all[x][q]);   // column q
  const int column = c - x + q;
  W* to = second ? db : dw;
  if (x == 0 && column < D && to) to[column] = from_float<W>(s);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int threads_of(int D, int per) { return std::min(1024, (ceil_div(D, per) + 31) / 32 * 32); }

template <typename T, typename W, int VEC, int K>
int forward_of(const Forward& g, cudaStream_t st) {
  if (g.D <= kWarpRow && VEC * K == 8)
    B200CP_CUDA_OK(launch_kernel(norm_kernel<T, W, VEC, K, true>, dim3(ceil_div(g.rows, kRows)), dim3(32 * kRows), 0, st, true, g));
  else
    B200CP_CUDA_OK(launch_kernel(norm_kernel<T, W, VEC, K, false>, dim3(g.rows), dim3(threads_of(g.D, VEC * K)), 0, st, true, g));
  B200CP_LAUNCH_OK("norm_kernel");
  return B200CP_OK;
}
// Features of a thread.  Few rows (less than four an SM): 8, the shortest way through a row (64 x 4096 2.4 us, with 32 3.0).  Many rows: 32 of 16-bit types, which halves and
// quarters what a row costs beside its values (8192 x 4096 in bfloat16 28.0 us, with 16 34.5, with 8 39.6; with the residual 43.2, 44.2, 47.9; HBM 20.6 and 41.3), 8 in
// rows up to 512 (6.5 us, 7.1).  float32 is bound by HBM sooner: 8 up to 2048, then 32, with the residual 16 (4096: 45.5 of 48.2, 81.9 of 95).
template <typename T, typename W, int VEC>
int forward_by_size(const Forward& g, cudaStream_t st) {
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  const bool half = sizeof(T) == 2;
  int each = g.rows < 4 * di.sm_count || g.D <= (half ? 512 : 2048) ? 8 : half || !g.r ? 32 : 16;
  if (VEC == 1) each = g.D <= 2048 ? 8 : 16;   // (odd rows)
  if (g.D > 1024 * each) each = g.D <= 16384 ? 16 : 32;
  if (each == 8) return forward_of<T, W, VEC, 8 / VEC>(g, st);
  if (each == 16 && g.D <= 16384) return forward_of<T, W, VEC, 16 / VEC>(g, st);
  if constexpr (VEC > 1)
    if (g.D <= 32768) return forward_of<T, W, VEC, 32 / VEC>(g, st);
  B200CP_CUDA_OK(launch_kernel(norm_wide_kernel<T, W, VEC>, dim3(g.rows), dim3(1024), 0, st, true, g));
  B200CP_LAUNCH_OK("norm_wide_kernel");
  return B200CP_OK;
}
template <typename T, typename W>
int forward(const Forward& g, cudaStream_t st) {
  bool vec = true;
  for (const void* p : {g.x, g.r, (const void*)g.y, (const void*)g.h}) vec = vec && rows_of_16<T>(p, g.D);
  for (const void* p : {g.w, g.b}) vec = vec && !(reinterpret_cast<uintptr_t>(p) & (kPerLoad<T> * sizeof(W) - 1));
  return vec ? forward_by_size<T, W, kPerLoad<T>>(g, st) : forward_by_size<T, W, 1>(g, st);
}

// CTAs that share the rows of a gradient: as many as an SM holds, with eight rows each where there are that many (a CTA's sums are 8 bytes a feature, as what
// a row of 16-bit values reads and writes).
int grad_ctas(int rows, int D, int sm_count) {
  const bool warp = D <= kWarpRow;
  const int units = warp ? ceil_div(rows, kRows) : rows;
  const int threads = warp ? 32 * kRows : D > kGradRow ? 256 : threads_of(D, kGradEach);
  const int most = sm_count * std::max(1, kGradThreads / threads);
  return std::max(1, std::min(units, std::max(sm_count, std::min(most, ceil_div(units, 8)))));
}
template <typename T, typename W, int VEC>
int grads(const Backward& g, int ctas, cudaStream_t st) {
  if (g.D <= kWarpRow) {
    B200CP_CUDA_OK(launch_kernel(norm_grads_kernel<T, W, VEC, 8 / VEC, true>, dim3(ctas), dim3(32 * kRows), 0, st, true, g));
    B200CP_LAUNCH_OK("norm_grads_kernel");
    return B200CP_OK;
  }
  if constexpr (VEC > 1) {
    if (g.D <= kGradRow) {
      // (what an SM has of shared memory is shared by as many CTAs as its threads make; two places for rows of 8192 floats are 192 KB)
      const int threads = threads_of(g.D, kGradEach), row = g.D * (int)sizeof(T), slot = (g.dh && g.dx ? 3 : 2) * row,
                room = 216 * 1024 / std::max(1, kGradThreads / threads) - 2048;
      const Ring ring{std::max(2, std::min(kMostSlots, room / slot)), row};
      const auto kern = norm_grads_ring_kernel<T, W, VEC, kGradEach / VEC>;
      static std::atomic<int> set[64];
      B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), set, ring.slots * slot));
      B200CP_CUDA_OK(launch_kernel(kern, dim3(ctas), dim3(threads), (size_t)ring.slots * slot, st, true, g, ring));
      B200CP_LAUNCH_OK("norm_grads_ring_kernel");
      return B200CP_OK;
    }
  } else if (g.D <= kGradThreads * 8) {
    B200CP_CUDA_OK(launch_kernel(norm_grads_kernel<T, W, 1, 8, false>, dim3(ctas), dim3(threads_of(g.D, 8)), 0, st, true, g));
    B200CP_LAUNCH_OK("norm_grads_kernel");
    return B200CP_OK;
  }
  if (g.dx) {
    B200CP_CUDA_OK(launch_kernel(norm_wide_dx_kernel<T, W, VEC>, dim3(g.rows), dim3(1024), 0, st, true, g));
    B200CP_LAUNCH_OK("norm_wide_dx_kernel");
  }
  if (g.partial) {
    const unsigned x = (unsigned)((g.D + 256LL * VEC - 1) / (256LL * VEC));
    B200CP_CUDA_OK(launch_kernel(norm_columns_kernel<T, VEC>, dim3(x, (unsigned)ctas), dim3(256), 0, st, true, g));
    B200CP_LAUNCH_OK("norm_columns_kernel");
  }
  return B200CP_OK;
}
template <typename T, typename W>
int backward(Backward g, int ctas, void* dw, void* db, cudaStream_t st) {
  bool vec = true;
  for (const void* p : {g.dy, g.dh, g.h, (const void*)g.dx}) vec = vec && rows_of_16<T>(p, g.D);
  vec = vec && !(reinterpret_cast<uintptr_t>(g.w) & (kPerLoad<T> * sizeof(W) - 1));
  if (int rc = vec ? grads<T, W, kPerLoad<T>>(g, ctas, st) : grads<T, W, 1>(g, ctas, st)) return rc;
  if (!g.partial) return B200CP_OK;
  B200CP_CUDA_OK(launch_kernel(norm_join_kernel<W>, dim3(2 * ceil_div(g.D, 32)), dim3(1024), 0, st, true, ctas, g.D, g.partial, static_cast<W*>(dw),
                               static_cast<W*>(db)));
  B200CP_LAUNCH_OK("norm_join_kernel");
  return B200CP_OK;
}
int check_norm(const char* who, int rows, int D, int type, int weight_type) {
  if (rows < 0 || D < 1) return fail(B200CP_ERR_INVALID_ARG, "%s: %d rows of %d features", who, rows, D);
  if (type < B200CP_FLOAT32 || type > B200CP_FLOAT16) return fail(B200CP_ERR_INVALID_ARG, "%s: type %d", who, type);
  if (weight_type != type && weight_type != B200CP_FLOAT32)
    return fail(B200CP_ERR_UNSUPPORTED, "%s: weights of type %d for rows of type %d (that type, or float)", who, weight_type, type);
  if (D > (1 << 30) || rows > (1 << 30)) return fail(B200CP_ERR_UNSUPPORTED, "%s: %d rows of %d features (at most 2^30 of both)", who, rows, D);
  return B200CP_OK;
}
template <typename F>
int by_types(int type, int weight_type, F f) {
  const bool full = weight_type == B200CP_FLOAT32;
  if (type == B200CP_FLOAT32) return f((float*)nullptr, (float*)nullptr);
  if (type == B200CP_BFLOAT16) return full ? f((__nv_bfloat16*)nullptr, (float*)nullptr) : f((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr);
  return full ? f((__half*)nullptr, (float*)nullptr) : f((__half*)nullptr, (__half*)nullptr);
}

}  // namespace

int layer_norm_device_status(int* out) {
  int v = 0, zero = 0;
  B200CP_CUDA_OK(cudaMemcpyFromSymbol(&v, g_layer_norm_status, sizeof(int)));
  if (v) B200CP_CUDA_OK(cudaMemcpyToSymbol(g_layer_norm_status, &zero, sizeof(int)));
  *out = v;
  return B200CP_OK;
}

}  // namespace b200cp

using namespace b200cp;

extern "C" {

int b200cp_layer_norm(int rows, int D, int type, int weight_type, const void* X, const void* R, const void* w, const void* b, float eps, void* Y,
                      void* H, float* mean, float* rstd, void* stream) {
  const char* who = "b200cp_layer_norm";
  if (int rc = check_norm(who, rows, D, type, weight_type)) return rc;
  if (!(eps >= 0.f)) return fail(B200CP_ERR_INVALID_ARG, "%s: eps %g", who, (double)eps);
  if (rows == 0) return B200CP_OK;
  if (!X || !Y || !R != !H || !mean != !rstd) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  const Forward g{rows, D, eps, X, R, w, b, Y, H, mean, rstd};
  return by_types(type, weight_type, [&](auto* t, auto* v) {
    return forward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(v)>>(g, static_cast<cudaStream_t>(stream));
  });
}

size_t b200cp_layer_norm_bwd_workspace_bytes(int rows, int D) {
  if (rows < 1 || D < 1) return 0;
  DeviceInfo di;
  if (device_info(&di)) return 0;
  return (size_t)grad_ctas(rows, D, di.sm_count) * 2 * (size_t)D * sizeof(float);
}

int b200cp_layer_norm_bwd(int rows, int D, int type, int weight_type, const void* dY, const void* dH, const void* H, const void* w,
                          const float* mean, const float* rstd, void* dX, void* dw, void* db, void* workspace, size_t workspace_bytes,
                          void* stream) {
  const char* who = "b200cp_layer_norm_bwd";
  if (int rc = check_norm(who, rows, D, type, weight_type)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t wbytes = (size_t)D * (weight_type == B200CP_FLOAT32 ? 4 : 2);
  if (rows == 0) {
    for (void* p : {dw, db})
      if (p) B200CP_CUDA_OK(cudaMemsetAsync(p, 0, wbytes, st));
    return B200CP_OK;
  }
  if (!dX && !dw && !db) return B200CP_OK;
  if (!dY || !H || !mean || !rstd) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  const int ctas = grad_ctas(rows, D, di.sm_count);
  const bool sums = dw || db;
  const size_t need = sums ? (size_t)ctas * 2 * (size_t)D * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, %zu given", who, need, workspace_bytes);
  const Backward g{rows, D, dY, dH, H, w, mean, rstd, dX, sums ? static_cast<float*>(workspace) : nullptr};
  return by_types(type, weight_type, [&](auto* t, auto* v) {
    return backward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(v)>>(g, ctas, dw, db, st);
  });
}

}  // extern "C"
