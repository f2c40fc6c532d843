// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
//   m <- b1 m + (1 - b1) g      v <- b2 v + (1 - b2) g^2      p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// A tensor is cut into pieces of kPiece values, a CTA takes one piece of one tensor; the table of tensors is a kernel parameter (so that a
// captured launch carries it, and nothing is copied), and a CTA finds its tensor by bisection over the pieces' sums.
//
// Moments in 8 bits: blocks of 256 values, which are those of a warp, with the largest magnitude s of each.  |m| = s (c / 127)^2 and
// v = s (c / 254)^4: the codes' steps are relative ones over most of the range, v reaches down to 2.4e-10 s and m to 6e-5 s, which is its
// square root and four times more.  So where a value's v is rounded to nothing, its m has been; a v above zero has a code of one at least all
// the same, and no m is ever divided by eps alone.  A value that is not finite keeps a code of its own (-128; 255) and reads as NaN, so it costs
// the other 255 nothing.  The parameter is updated with the moments before they are rounded.  All arithmetic is fp32, the roundings of the
// moments those of separate products and sums; to fewer bits are rounded the codes (half a step: 0.8 % of the largest values) and a 16-bit
// parameter, whose fp32 copy (master) is what is updated where there is one.
//
// Bound by HBM: 28 bytes a value (p, m, v read and written, g read), 16.06 with 8-bit moments.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace b200cp {
namespace {

constexpr int kThreads = 256, kPiece = 2048, kBlock = 256;   // a warp has 256 values: two groups of four per lane
// Tensors of a launch: tables of 3.5, 9 and 31 KB (32 764 bytes are the most).  A table's bytes are written for each launch: calls of 20, 40, 84 and
// 128 tensors take 8.7, 11.1, 18.3 and 24.0 us, and with the largest table alone 12.4, 15.5, 21.4 and 27.8 (one after another, 4096 values each).
constexpr int kFew = 48, kSome = 128, kMany = 448;

struct Entry {
  void* p;
  const void* g;
  void *m, *v;
  float *ms, *vs, *w;
  long long n;
};
struct Rates {
  float b1, b2, c1, c2;        // c = 1 - b
  float decay, eps;            // lr wd
  float step, root;            // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  const long long* t;          // on the device: step and root are formed by the kernel
  const float* lr;
  double lr_, wd, b1_, b2_;    // then from these
};
template <int CAP>
struct Table {
  Rates r;
  int count;
  int first[CAP + 1];          // pieces before each tensor
  Entry e[CAP];
};

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};
// (`vec`: all four of every thread are inside and on a boundary of four)
template <typename T>
__device__ __forceinline__ void load4(const T* p, long long i, long long n, bool vec, float (&x)[4]) {
  if (vec) {
    const Four<T> q = *reinterpret_cast<const Four<T>*>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)q.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k < n ? (float)p[i + k] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long long i, long long n, bool vec, const float (&x)[4]) {
  if (vec) {
    Four<T> q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = (T)x[k];
    *reinterpret_cast<Four<T>*>(p + i) = q;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = (T)x[k];
  }
}
template <typename T>
__device__ __forceinline__ bool aligned4(const T* p) { return !(reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)); }

// Within 2^-22 of the root and of the quotient: enough for a step, and for a code that is not next to a border.
__device__ __forceinline__ float fast_sqrt(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_sqrt_ftz(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_inverse(float x) {   // (of normal numbers)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Codes to numbers and back by the integer bits of a float around 2^23 and 1.5 2^23 (nearest, ties to even): the conversion instructions share the pipe
// of the roots, sixteen lanes a cycle, and were half of its work.
constexpr float kWhole = 12582912.f;
__device__ __forceinline__ float code_at(uint32_t four, int k, float zero) { return __uint_as_float(__byte_perm(four, 0x4b000000u, 0x7440 + k)) - zero; }
__device__ __forceinline__ void codes_of_m(uint32_t four, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = code_at(four ^ 0x80808080u, k, 8388608.f + 128.f);
}
__device__ __forceinline__ void codes_of_v(uint32_t four, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = code_at(four, k, 8388608.f);
}
__device__ __forceinline__ uint32_t to_codes(const float (&x)[4]) {   // of whole numbers with kWhole added
  const auto bits = [](float c) { return __float_as_uint(c); };
  return __byte_perm(__byte_perm(bits(x[0]), bits(x[1]), 0x0040), __byte_perm(bits(x[2]), bits(x[3]), 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, long long i, long long n, bool vec) {
  if (vec) return *reinterpret_cast<const uint32_t*>(p + i);
  uint32_t c = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) c |= (uint32_t)p[i + k] << (8 * k);
  return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, long long i, long long n, bool vec, uint32_t c) {
  if (vec) {
    *reinterpret_cast<uint32_t*>(p + i) = c;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) p[i + k] = (uint8_t)(c >> (8 * k));
}
// Whether one of four bytes is zero (of the codes xor that of NaN): a value in none but a broken state.
__device__ __forceinline__ bool has_zero(uint32_t x) { return ((x - 0x01010101u) & ~x & 0x80808080u) != 0; }
__device__ __forceinline__ void values_of_m(uint32_t four, float s, float (&x)[4]) {
  codes_of_m(four, x);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float q = x[k] * (1.f / 127);
    x[k] = q * fabsf(q) * s;
  }
  if (has_zero(four ^ 0x80808080u)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if ((four >> (8 * k) & 255) == 128) x[k] = __int_as_float(0x7fffffff);
  }
}
__device__ __forceinline__ void values_of_v(uint32_t four, float s, float (&x)[4]) {
  codes_of_v(four, x);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float q = x[k] * (1.f / 254), r = q * q;
    x[k] = r * r * s;
  }
  if (has_zero(~four)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if ((four >> (8 * k) & 255) == 255) x[k] = __int_as_float(0x7fffffff);
  }
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// The code is that of 127 sqrt(|x| / s) with every operation rounded to nearest: found by the fast operations, and again by the exact
// ones where one of a thread's eight ends within 2e-4 of a border (the two are within 1.1e-4 of a step of one another).  Exact codes do not
// depend on how an operation is approximated: two implementations that round alike hold the same state.
__device__ __noinline__ float exact_m(float x, float s) {
  if (!(fabsf(x) < __int_as_float(0x7f800000))) return -128.f;
  return s > 0.f ? copysignf(rintf(127.f * sqrtf(__fdiv_rn(fabsf(x), s))), x) : 0.f;
}
__device__ __noinline__ float exact_v(float x, float s) {
  if (!(x < __int_as_float(0x7f800000))) return 255.f;
  return x > 0.f && s > 0.f ? fmaxf(rintf(254.f * sqrtf(sqrtf(__fdiv_rn(x, s)))), 1.f) : 0.f;
}
__device__ __forceinline__ void codes_from(const float (&m)[4], const float (&v)[4], float sm, float sv, float im, float iv, uint32_t& cm, uint32_t& cv) {
  float a[4], b[4], off = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float t = copysignf(127.f * fast_sqrt_ftz(fabsf(m[k]) * im), m[k]), u = 254.f * fast_sqrt_ftz(fast_sqrt_ftz(v[k] * iv));
    a[k] = t + kWhole;
    b[k] = u + kWhole;
    off = max_nan(max_nan(off, fabsf(t - (a[k] - kWhole))), fabsf(u - (b[k] - kWhole)));
    b[k] = fmaxf(b[k], v[k] > 0.f ? kWhole + 1.f : kWhole);
  }
  if (!(off <= 0.4998f) || im == 0.f || iv == 0.f) {   // (what is not finite ends here too)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] = exact_m(m[k], sm) + kWhole;
      b[k] = exact_v(v[k], sv) + kWhole;
    }
  }
  cm = to_codes(a);
  cv = to_codes(b);
}
__device__ __forceinline__ float finite_magnitude(float x) { return fabsf(x) < __int_as_float(0x7f800000) ? fabsf(x) : 0.f; }
__device__ __forceinline__ float warp_max(float x) {   // of magnitudes
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x)));
}
// 1 / s, or 0 where s or that is no normal number (then every code of the block is found by the exact operations)
__device__ __forceinline__ float inverse_of(float s) { return s > 1e-37f && s < 1e37f ? 1.f / s : 0.f; }

// A warp's 256 values of a tensor, from `base` on.  WHOLE: all are there and every array is on a boundary of four (without a check per access, which were a
// tenth of the instructions of 8-bit moments).
template <typename P, typename G, bool SMALL, bool WHOLE>
__device__ __forceinline__ void update(const Entry& e, const Rates& r, float step, float root, float decay, long long base) {
  const int lane = threadIdx.x & 31;
  const long long n = e.n, block = base / kBlock;
  P* p = static_cast<P*>(e.p);
  const G* g = static_cast<const G*>(e.g);
  float* w = e.w;
  float x[2][4], d[2][4], m[2][4], v[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long i = base + j * 128 + lane * 4;
    if (w) load4(w, i, n, WHOLE, x[j]); else load4(p, i, n, WHOLE, x[j]);
    load4(g, i, n, WHOLE, d[j]);
  }
  if constexpr (SMALL) {
    const uint8_t *cm = static_cast<const uint8_t*>(e.m), *cv = static_cast<const uint8_t*>(e.v);
    const float ms = e.ms[block], vs = e.vs[block];
    uint32_t pm[2], pv[2];   // (all loads before the first code is looked at)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long i = base + j * 128 + lane * 4;
      pm[j] = load_codes(cm, i, n, WHOLE);
      pv[j] = load_codes(cv, i, n, WHOLE);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      values_of_m(pm[j], ms, m[j]);
      values_of_v(pv[j], vs, v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long i = base + j * 128 + lane * 4;
      load4(static_cast<const float*>(e.m), i, n, WHOLE, m[j]);
      load4(static_cast<const float*>(e.v), i, n, WHOLE, v[j]);
    }
  }
  float mm = 0.f, mv = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[j][k] = fmaf(r.c1, d[j][k], __fmul_rn(r.b1, m[j][k]));
      v[j][k] = fmaf(r.c2, __fmul_rn(d[j][k], d[j][k]), __fmul_rn(r.b2, v[j][k]));
      if (SMALL) {   // (values past the end are zero, and a NaN is never the larger: neither changes a maximum)
        mm = fmaxf(mm, fabsf(m[j][k]));
        mv = fmaxf(mv, v[j][k]);
      }
    }
  if (r.eps >= 1e-12f) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[j][k] = fmaf(-step, m[j][k] * fast_inverse(fmaf(fast_sqrt_ftz(v[j][k]), root, r.eps)), fmaf(-decay, x[j][k], x[j][k]));
  } else {   // the square root of a subnormal v counts beside such an eps, and their sum may be subnormal itself
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[j][k] = fmaf(-step, __fdiv_rn(m[j][k], fmaf(fast_sqrt(v[j][k]), root, r.eps)), fmaf(-decay, x[j][k], x[j][k]));
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long i = base + j * 128 + lane * 4;
    if (w) store4(w, i, n, WHOLE, x[j]);
    store4(p, i, n, WHOLE, x[j]);
  }
  if constexpr (SMALL) {
    uint8_t *cm = static_cast<uint8_t*>(e.m), *cv = static_cast<uint8_t*>(e.v);
    mm = warp_max(mm);
    mv = warp_max(mv);
    if (fmaxf(mm, mv) > 3.4028235e38f) {   // an infinity: the largest of the finite ones
      mm = mv = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mm = fmaxf(mm, finite_magnitude(m[j][k]));
          mv = fmaxf(mv, finite_magnitude(v[j][k]));
        }
      mm = warp_max(mm);
      mv = warp_max(mv);
    }
    const float im = inverse_of(mm), iv = inverse_of(mv);
    if (lane == 0) {
      e.ms[block] = mm;
      e.vs[block] = mv;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long i = base + j * 128 + lane * 4;
      uint32_t p4, q4;
      codes_from(m[j], v[j], mm, mv, im, iv, p4, q4);
      store_codes(cm, i, n, WHOLE, p4);
      store_codes(cv, i, n, WHOLE, q4);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long i = base + j * 128 + lane * 4;
      store4(static_cast<float*>(e.m), i, n, WHOLE, m[j]);
      store4(static_cast<float*>(e.v), i, n, WHOLE, v[j]);
    }
  }
}

// (CTAs of an SM, 59 M values with 8-bit moments: 188 us with four, 172 with five, 165 with six; 42 M in bfloat16 with copies 169, 169, 171.)
template <typename P, typename G, bool SMALL, int CAP>
__global__ void __launch_bounds__(kThreads, SMALL ? 6 : 5) adamw_kernel(const __grid_constant__ Table<CAP> t) {
  int a = 0, b = t.count;   // the tensor whose pieces hold this CTA's
  while (b - a > 1) {
    const int c = (a + b) / 2;
    if (t.first[c] <= (int)blockIdx.x) a = c; else b = c;
  }
  const Entry& e = t.e[a];
  const long long base = (long long)((int)blockIdx.x - t.first[a]) * kPiece + (threadIdx.x >> 5) * kBlock;
  float step = t.r.step, root = t.r.root, decay = t.r.decay;
  if (t.r.t || t.r.lr) {
    __shared__ float rates[3];
    if (threadIdx.x == 0) {
      const double lr = t.r.lr ? (double)*t.r.lr : t.r.lr_;
      double s = t.r.step, q = t.r.root;   // (of lr = 1, where lr is on the device)
      if (t.r.t) {
        const double at = (double)*t.r.t;
        s = 1.0 / (1.0 - pow(t.r.b1_, at));
        q = 1.0 / sqrt(1.0 - pow(t.r.b2_, at));
      }
      rates[0] = (float)(lr * s);
      rates[1] = (float)q;
      rates[2] = (float)(lr * t.r.wd);
    }
    __syncthreads();
    step = rates[0];
    root = rates[1];
    decay = rates[2];
  }
  if (base >= e.n) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(e.p) % (4 * sizeof(P)) | reinterpret_cast<uintptr_t>(e.g) % (4 * sizeof(G)) |
                       reinterpret_cast<uintptr_t>(e.w) % 16 | (reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v)) % (SMALL ? 4 : 16);
  if (base + kBlock <= e.n && at == 0)
    update<P, G, SMALL, true>(e, t.r, step, root, decay, base);
  else
    update<P, G, SMALL, false>(e, t.r, step, root, decay, base);
}

// Four groups of four values per thread, so that enough bytes are in flight (with one group 111 us of 58.7 M values).
constexpr int kMomentGroups = 4;
template <typename T>
__global__ void __launch_bounds__(kThreads) moments_kernel(long long n, const uint8_t* cm, const uint8_t* cv, const float* ms, const float* vs,
                                                           T* m, T* v) {
  const long long i0 = (long long)blockIdx.x * (kThreads * 4 * kMomentGroups) + threadIdx.x * 4;
  const bool whole = i0 + (kMomentGroups - 1) * (kThreads * 4) + 4 <= n, a = whole && aligned4(cm), b = whole && aligned4(cv), c = whole && aligned4(m),
             d = whole && aligned4(v);
  uint32_t p[kMomentGroups], q[kMomentGroups];
  float s[kMomentGroups], r[kMomentGroups];
#pragma unroll
  for (int j = 0; j < kMomentGroups; ++j) {
    const long long i = i0 + j * (kThreads * 4);
    if (i >= n) break;
    p[j] = load_codes(cm, i, n, a);
    q[j] = load_codes(cv, i, n, b);
    s[j] = ms[i / kBlock];
    r[j] = vs[i / kBlock];
  }
#pragma unroll
  for (int j = 0; j < kMomentGroups; ++j) {
    const long long i = i0 + j * (kThreads * 4);
    if (i >= n) break;
    float x[4], y[4];
    values_of_m(p[j], s[j], x);
    values_of_v(q[j], r[j], y);
    store4(m, i, n, c, x);
    store4(v, i, n, d, y);
  }
}

template <typename P, typename G, bool SMALL, int CAP>
int launch_some(const b200cp_adamw_tensor* ts, int count, const Rates& r, cudaStream_t st) {
  Table<CAP> t;
  t.r = r;
  int at = 0;
  while (at < count) {   // tables of up to CAP tensors and 2^30 pieces
    long long pieces = 0;
    t.count = 0;
    for (; at < count && t.count < CAP; ++at) {
      const b200cp_adamw_tensor& s = ts[at];
      if (s.n == 0) continue;
      const long long mine = (long long)((s.n + kPiece - 1) / kPiece);
      if (pieces + mine > 0x3fffffff) {
        if (t.count == 0) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_adamw_step: a tensor of %llu values", s.n);
        break;
      }
      t.first[t.count] = (int)pieces;
      t.e[t.count++] = Entry{s.param, s.grad, s.exp_avg, s.exp_avg_sq, s.scale_avg, s.scale_sq, s.master, (long long)s.n};
      pieces += mine;
    }
    if (t.count == 0) break;
    t.first[t.count] = (int)pieces;
    adamw_kernel<P, G, SMALL, CAP><<<(unsigned)pieces, kThreads, 0, st>>>(t);
    B200CP_LAUNCH_OK("adamw_kernel");
  }
  return B200CP_OK;
}
template <typename P, typename G, bool SMALL>
int launch_all(const b200cp_adamw_tensor* ts, int count, const Rates& r, cudaStream_t st) {
  if (count <= kFew) return launch_some<P, G, SMALL, kFew>(ts, count, r, st);
  return count <= kSome ? launch_some<P, G, SMALL, kSome>(ts, count, r, st) : launch_some<P, G, SMALL, kMany>(ts, count, r, st);
}
template <typename P, typename G>
int launch_bits(const b200cp_adamw_tensor* ts, int count, int bits, const Rates& r, cudaStream_t st) {
  return bits == 8 ? launch_all<P, G, true>(ts, count, r, st) : launch_all<P, G, false>(ts, count, r, st);
}

}  // namespace
}  // namespace b200cp

using namespace b200cp;

extern "C" {

int b200cp_adamw_step(const b200cp_adamw_tensor* tensors, int count, int param_type, int grad_type, int moment_bits,
                      const b200cp_adamw* h, void* stream) {
  if (count < 0 || (count && !tensors) || !h) return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: null argument or negative count");
  if (moment_bits != 8 && moment_bits != 32) return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: moments of %d bits", moment_bits);
  if (!(h->beta1 >= 0 && h->beta1 < 1 && h->beta2 >= 0 && h->beta2 < 1 && h->eps >= 0))
    return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: betas %g, %g or eps %g out of range", h->beta1, h->beta2, h->eps);
  if (!h->device_step && h->step < 1) return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: step %lld (they count from one)", h->step);
  for (int i = 0; i < count; ++i) {
    const b200cp_adamw_tensor& s = tensors[i];
    if (s.n && (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq || (moment_bits == 8 && (!s.scale_avg || !s.scale_sq))))
      return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: null pointer in tensor %d", i);
    if (s.n && s.master && param_type == B200CP_FLOAT32)
      return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_step: a float32 parameter has no float32 copy (tensor %d)", i);
  }
  Rates r{};
  r.b1 = (float)h->beta1; r.b2 = (float)h->beta2; r.c1 = (float)(1 - h->beta1); r.c2 = (float)(1 - h->beta2);
  r.eps = (float)h->eps;
  r.decay = (float)(h->lr * h->weight_decay);
  r.t = h->device_step; r.lr = h->device_lr;
  r.lr_ = h->lr; r.wd = h->weight_decay; r.b1_ = h->beta1; r.b2_ = h->beta2;
  if (!h->device_step) {
    r.step = (float)((h->device_lr ? 1.0 : h->lr) / (1 - std::pow(h->beta1, (double)h->step)));
    r.root = (float)(1 / std::sqrt(1 - std::pow(h->beta2, (double)h->step)));
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define TYPES(P, G) return launch_bits<P, G>(tensors, count, moment_bits, r, st)
  if (param_type == B200CP_FLOAT32 && grad_type == B200CP_FLOAT32) TYPES(float, float);
  if (param_type == B200CP_BFLOAT16 && grad_type == B200CP_BFLOAT16) TYPES(__nv_bfloat16, __nv_bfloat16);
  if (param_type == B200CP_FLOAT16 && grad_type == B200CP_FLOAT16) TYPES(__half, __half);
  if (param_type == B200CP_BFLOAT16 && grad_type == B200CP_FLOAT32) TYPES(__nv_bfloat16, float);
  if (param_type == B200CP_FLOAT16 && grad_type == B200CP_FLOAT32) TYPES(__half, float);
#undef TYPES
  return fail(B200CP_ERR_UNSUPPORTED, "b200cp_adamw_step: parameters of type %d with gradients of type %d", param_type, grad_type);
}

int b200cp_adamw_moments(unsigned long long n, const void* exp_avg, const void* exp_avg_sq, const float* scale_avg, const float* scale_sq,
                         int out_type, void* m, void* v, void* stream) {
  if (n == 0) return B200CP_OK;
  if (!exp_avg || !exp_avg_sq || !scale_avg || !scale_sq || !m || !v)
    return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_moments: null pointer");
  constexpr unsigned long long per = 4 * kThreads * kMomentGroups;
  const unsigned long long ctas = (n + per - 1) / per;
  if (ctas > 0x7fffffffull) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_adamw_moments: %llu values", n);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto* out_m, auto* out_v) {
    moments_kernel<<<(unsigned)ctas, kThreads, 0, st>>>((long long)n, static_cast<const uint8_t*>(exp_avg), static_cast<const uint8_t*>(exp_avg_sq),
                                                        scale_avg, scale_sq, out_m, out_v);
    B200CP_LAUNCH_OK("moments_kernel");
    return (int)B200CP_OK;
  };
  switch (out_type) {
    case B200CP_FLOAT32: return go(static_cast<float*>(m), static_cast<float*>(v));
    case B200CP_BFLOAT16: return go(static_cast<__nv_bfloat16*>(m), static_cast<__nv_bfloat16*>(v));
    case B200CP_FLOAT16: return go(static_cast<__half*>(m), static_cast<__half*>(v));
  }
  return fail(B200CP_ERR_INVALID_ARG, "b200cp_adamw_moments: type %d", out_type);
}

}  // extern "C"
