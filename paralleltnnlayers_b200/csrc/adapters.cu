// Low-rank adapters of many requests beside a shared projection, forward and gradients.
//
//   V[s] = c[a] X[s] A[a],  out[s] = Y[s] + V[s] B[a]            a: the adapter of row s
//   W[s] = c[a] dY[s] B[a]^T,  dX[s] = W[s] A[a]^T,  dA[a] = sum_s X[s]^T W[s],  dB[a] = sum_s V[s]^T dY[s]
//
// Forward and dX are one kernel (the second with the factors transposed): a tile of 16 or 64 rows of one adapter, whose sum over the features runs
// over the CTAs of a cluster and is joined through their shared memory, so that X is read once, V stays on the chip between the two
// products and a few rows still fill the machine.  What bounds it is HBM: X and Y in, out once; the products take 2 R (I + O) operations a row, on
// mma.sync for 16-bit types (R columns are too few to feed anything wider) and FFMA for fp32, whose sums are then those of fp32.
// (Of what was tried to bring rows in sooner, prefetches of their parts into L2 cost 10 % more and copies of whole parts (cp.async.bulk, a thread per row)
// 40 %: such a request takes an SM some 30 cycles, and there are thousands.)
// Rows of a tile are gathered by the plan's order, so requests may lie anywhere in the batch; a row's result depends on its own row and
// adapter only, and values that are not finite stay with theirs.  As operands of the second
// product V and W are two parts of the 16-bit type (rounded once, out of a token and an adapter would be as far off as by its own rounding, and at a
// small rank up to twice that); they are rounded once where they are kept for dA and dB.
//
// dA and dB are one kernel over the rows in the plan's order, cut into ranges of equal length: a CTA has 128 features of a range and adds
// row after row in registers until the adapter changes.  Adapters inside a range are written at once, those that reach into another range as
// partial sums that a second launch joins in order: no atomics, the same bits each time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "cluster_util.cuh"
#include "common.cuh"

namespace b200cp {

__device__ int g_adapters_status = 0;   // 1: a plan of other rows or another number of adapters

namespace {

constexpr int kThreads = 256, kWarps = 8, kMostRank = 128, kMostAdapters = 16384;
static_assert(B200CP_ADAPTERS_WITHOUT_PLAN <= kThreads, "a thread has a row");

// ---- plan -------------------------------------------------------------------------------------------------------------------
// ints: [0] tiles, [1] rows with an adapter, [2] rows, [3] count | start[count + 2] | tile_adapter[tiles] | tile_first[tiles] | order[rows].
// Rows without an adapter are those of "adapter" count, behind the others.  Where the arrays lie depends on rows and count: a kernel that is
// handed the plan of others leaves it alone, records that and returns (plans of neighbouring counts often have the same size).
struct Plan {
  int tm, tiles, likely;   // rows of a tile; the most tiles there can be; as many as adapters whose last tile is half full give
  size_t start, adapter, first, order, ints;
};
Plan plan_of(int rows, int count) {
  Plan p;
  const int groups = std::min(rows, count);
  // Tiles of 64 rows read an adapter once per 64 rows, tiles of 16 waste less of themselves on adapters of a few rows.
  p.tm = groups > 0 && rows / groups >= 48 ? 64 : 16;
  p.tiles = rows / p.tm + std::min(rows, count + 1);
  p.likely = rows / p.tm + (std::min(rows, count + 1) + 1) / 2;
  p.start = 4;
  p.adapter = p.start + count + 2;
  p.first = p.adapter + p.tiles;
  p.order = p.first + p.tiles;
  p.ints = align_up(p.order + rows, 4);
  return p;
}

// exclusive sums of the values of all 1024 threads; `total` gets the sum of all
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int before = warp ? warp_sums[warp - 1] : 0;
  *total = warp_sums[31];
  __syncthreads();
  return before + x - v;
}

// A stable counting sort by one CTA: the first `sorters` warps count the rows of a range each, every (adapter, warp) gets its place, and the warps put
// their rows there in order.  shared: counts[(count + 1) * sorters] | tiles before each adapter [count + 2]
__global__ void __launch_bounds__(1024) plan_kernel(int rows, int count, int tm, int sorters, const int* adapters, int* plan, size_t at_adapter,
                                                    size_t at_first, size_t at_order) {
  extern __shared__ int counts[];
  __shared__ int warp_sums[32];
  grid_launch_dependents();   // the kernel that reads the plan takes its place on the other SMs, and waits for this one there
  const int keys = count + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* tiles_before = counts + keys * sorters;
  for (int i = tid; i < keys * sorters; i += 1024) counts[i] = 0;
  __syncthreads();
  const int per = ((rows + sorters - 1) / sorters + 31) / 32 * 32, r0 = min(rows, warp * per), r1 = min(rows, r0 + per);
  const auto key_of = [&](int r) {
    const int a = adapters[r];
    return a >= 0 && a < count ? a : count;
  };
  constexpr int Q = 8;   // turns of a warp whose loads are in flight together (of a range of one such load they are kept for the second pass)
  int key[Q];
  if (warp < sorters)
    for (int b = r0; b < r1; b += 32 * Q) {
#pragma unroll
      for (int q = 0; q < Q; ++q) key[q] = b + q * 32 + lane < r1 ? key_of(b + q * 32 + lane) : -1;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (b + q * 32 >= r1) break;
        const unsigned same = __match_any_sync(0xffffffffu, key[q]);
        if (key[q] >= 0 && (same & ((1u << lane) - 1)) == 0) counts[key[q] * sorters + warp] += __popc(same);
        __syncwarp();
      }
    }
  __syncthreads();
  {   // places: sums over (adapter, warp)
    const int n = keys * sorters, each = (n + 1023) / 1024, b = min(n, tid * each), e = min(n, b + each);
    int sum = 0, total;
    for (int i = b; i < e; ++i) sum += counts[i];
    int at = block_scan(sum, warp_sums, &total);
    for (int i = b; i < e; ++i) {
      const int c = counts[i];
      counts[i] = at;
      at += c;
    }
  }
  __syncthreads();
  int* start = plan + 4;
  int tiles;
  {
    const int each = (keys + 1023) / 1024, b = min(keys, tid * each), e = min(keys, b + each);
    int sum = 0;
    const auto rows_of = [&](int k) { return (k + 1 < keys ? counts[(k + 1) * sorters] : rows) - counts[k * sorters]; };
    for (int k = b; k < e; ++k) sum += (rows_of(k) + tm - 1) / tm;
    int at = block_scan(sum, warp_sums, &tiles);
    for (int k = b; k < e; ++k) {
      tiles_before[k] = at;
      at += (rows_of(k) + tm - 1) / tm;
      start[k] = counts[k * sorters];
    }
  }
  if (tid == 0) {
    start[keys] = rows;
    plan[0] = tiles;
    plan[1] = counts[count * sorters];
    plan[2] = rows;
    plan[3] = count;
  }
  __syncthreads();
  for (int t = tid; t < tiles; t += 1024) {
    int a = 0, b = keys;   // the last adapter with no more than t tiles before it (the ones after it with as many have none)
    while (b - a > 1) {
      const int c = (a + b) / 2;
      if (tiles_before[c] <= t) a = c; else b = c;
    }
    plan[at_adapter + t] = a;
    plan[at_first + t] = counts[a * sorters] + (t - tiles_before[a]) * tm;
  }
  __syncthreads();
  if (warp < sorters)
    for (int b = r0; b < r1; b += 32 * Q) {
      if (r1 - r0 > 32 * Q) {
#pragma unroll
        for (int q = 0; q < Q; ++q) key[q] = b + q * 32 + lane < r1 ? key_of(b + q * 32 + lane) : -1;
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (b + q * 32 >= r1) break;
        const unsigned same = __match_any_sync(0xffffffffu, key[q]), before = same & ((1u << lane) - 1);
        const bool in = key[q] >= 0;
        const int at = in ? counts[key[q] * sorters + warp] + __popc(before) : 0;
        __syncwarp();
        if (in) {
          plan[at_order + at] = b + q * 32 + lane;
          if (before == 0) counts[key[q] * sorters + warp] += __popc(same);
        }
        __syncwarp();
      }
    }
}

// Whether a plan is one of these rows and adapters: the same answer for all threads of a launch, which reads nothing else of a plan that is not.
__device__ __forceinline__ bool plan_is_of(const int4& head, int rows, int count) {
  if (head.z == rows && head.w == count) return true;
  if (threadIdx.x == 0) atomicCAS(&g_adapters_status, 0, 1);
  return false;
}

// ---- loads ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src, int bytes) {   // the rest of the 16 is zero
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(shared_at(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ROWS rows of PIECES x 16 bytes into shared memory, a thread the same place of every row that it has: row r from row(r) (null: zeros), from column c0
// on, zero past `cols`.  `vec`: the rows start on 16-byte boundaries (then the copies are asynchronous).  Else fp32 comes in asynchronous
// words, and 16-bit values in words that a shift puts in place (a word that reaches past the row's ends is not read).
template <typename T, int ROWS, int PIECES, typename Row>
__device__ __forceinline__ void load_rows(char* dst, int stride, Row row, int c0, int cols, bool vec, const void* any) {
  constexpr int E = 16 / sizeof(T), STEP = kThreads / PIECES, N = (ROWS + STEP - 1) / STEP;
  const int q = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES, c = c0 + q * E, left = min(E, max(0, cols - c));
  dst += r0 * stride + q * 16;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = r0 + i * STEP;
    if (ROWS % STEP != 0 && r >= ROWS) break;
    const T* src = row(r);
    char* to = dst + i * STEP * stride;
    if (vec) {
      copy16(to, src && left ? (const void*)(src + c) : any, src ? left * (int)sizeof(T) : 0);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const bool in = src && k < left;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_at(to + 4 * k)), "l"(in ? (const void*)(src + c + k) : any), "r"(in ? 4 : 0)
                     : "memory");
      }
    } else if (src && c > 0 && c + E < cols) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src + c);
      const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
      uint32_t x[E / 2 + 1];
#pragma unroll
      for (int k = 0; k < E / 2; ++k) x[k] = w[k];
      if (at & 2) {
        x[E / 2] = w[E / 2];
#pragma unroll
        for (int k = 0; k < E / 2; ++k) x[k] = __funnelshift_r(x[k], x[k + 1], 16);
      }
      *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
      alignas(16) T v[E];
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = src && k < left ? src[c + k] : (T)0.f;
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
    }
  }
}

// The same for rows that start on 16-byte boundaries, chunk after chunk: where a thread's pieces come from is worked out once, so that a chunk takes a few
// instructions of it (worked out anew for each chunk: 4096 rows 36 us, and 32).
template <typename T, int ROWS, int PIECES>
struct Rows {
  static constexpr int E = 16 / sizeof(T), EACH = kThreads / PIECES, N = (ROWS + EACH - 1) / EACH;
  const char* from[N];
  bool in[N];
  template <typename Row>
  __device__ __forceinline__ void set(Row row, const void* any) {
    const int q = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r0 + i * EACH;
      const T* p = ROWS % EACH == 0 || r < ROWS ? row(r) : nullptr;
      in[i] = p != nullptr;
      from[i] = p ? reinterpret_cast<const char*>(p + q * E) : static_cast<const char*>(any);
    }
  }
  // `at` bytes on from the first chunk; bytes: of this thread's piece of a row that are inside (16, or less in the last chunk)
  __device__ __forceinline__ void load(char* dst, int stride, size_t at, int bytes) const {
    dst += threadIdx.x / PIECES * stride + threadIdx.x % PIECES * 16;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ROWS % EACH == 0 || threadIdx.x / PIECES + i * EACH < ROWS)
        copy16(dst + i * EACH * stride, bytes > 0 ? from[i] + at : from[i], in[i] ? bytes : 0);
  }
};
// of a thread's piece of a chunk from column c0 on
template <typename T, int PIECES>
__device__ __forceinline__ int piece_bytes(int c0, int cols) {
  constexpr int E = 16 / sizeof(T);
  return c0 + PIECES * E <= cols ? 16 : min(16, max(0, (cols - c0 - (int)(threadIdx.x % PIECES) * E) * (int)sizeof(T)));
}

// ---- products ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(shared_at(p))
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(shared_at(p))
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 16 x 16 block at p of rows `stride` bytes apart, as mma's A (16 rows of 16 k), and as its B for two groups of eight columns (r[0], r[1] and r[2],
// r[3]): `kmajor` where a row holds the k of one column, else a row holds the columns of one k.  For A with a row per k: a_of_k.
__device__ __forceinline__ void a_block(uint32_t (&r)[4], const char* p, int stride) {
  const int l = threadIdx.x & 31;
  ldsm4(r, p + (l & 15) * stride + (l >> 4) * 16);
}
__device__ __forceinline__ void a_of_k(uint32_t (&r)[4], const char* p, int stride) {
  const int l = threadIdx.x & 31;
  ldsm4t(r, p + ((l & 7) + (l >> 4) * 8) * stride + ((l >> 3) & 1) * 16);
}
template <bool KMAJOR>
__device__ __forceinline__ void b_block(uint32_t (&r)[4], const char* p, int stride) {
  const int l = threadIdx.x & 31;
  if (KMAJOR)
    ldsm4(r, p + ((l & 7) + (l >> 4) * 8) * stride + ((l >> 3) & 1) * 16);
  else
    ldsm4t(r, p + ((l & 7) + ((l >> 3) & 1) * 8) * stride + (l >> 4) * 16);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// ---- forward and dX ---------------------------------------------------------------------------------------------------------
struct Args {
  int rows, K, N, R, count;   // the first product sums over K, the second gives N columns
  const void *X, *Y;          // [rows][K]; [rows][N], or null: nothing is added
  const void *F1, *F2;        // forward: A [K][R], B [R][N] of an adapter; BACK: B [R][K], A [N][R]
  const float* scale;
  const int *start, *tile_adapter, *tile_first, *order, *head;   // of the plan; or
  const int* adapters;        // of each row, at most kThreads of them: every CTA finds its tile itself
  void *out, *V;              // [rows][N]; [rows][R] or null
  int vx, vy, v1, v2;         // rows of X, of Y and out, of the factors start on 16-byte boundaries
};

template <typename T, int TM, int RP>
struct Shape {
  // Bytes of a row in a chunk.  Of 64 rows 128, so that two to four CTAs share an SM (at rank 64 43 us with 128, 51 with 256), in fp32 at rank 16, where a
  // chunk's sums take long, 256 (67 us, and 89 with 128); of 16 rows 512 (64 requests 10.5 us with 256, 9.5 with 512).
  static constexpr int CB = TM == 16 ? (RP <= 32 ? 512 : 256) : RP == 16 && sizeof(T) == 4 ? 256 : 128;
  static constexpr int E = 16 / sizeof(T), KC = CB / sizeof(T), pieces = CB / 16;   // values of 16 bytes, values and pieces of a chunk
  static constexpr int xs = CB + 16;                                    // bytes from row to row: ldmatrix and 16-byte reads without conflicts
  static constexpr int ls = RP * (int)sizeof(T) + 16;                   // of a factor with the rank innermost
  static constexpr int factor = KC * ls > RP * xs ? KC * ls : RP * xs;
  static constexpr int stage = TM * xs + factor;
  static constexpr int stages = 3;
  static constexpr int CG = sizeof(T) == 4 && RP > 32 ? RP / 32 : 1;    // fp32: groups of 32 ranks over warps
  static constexpr int MG = sizeof(T) == 4 ? 1 : TM / 16;               // 16-bit: groups of 16 rows over warps
  static constexpr int KG = kWarps / (MG * CG);                         // parts of a chunk's sum over warps
  static constexpr int red = KG * TM * RP * 4;
  static constexpr int ring = stages * stage > red ? stages * stage : red;
  static constexpr int part = TM * RP * 4, vs = TM * ls * (sizeof(T) == 2 ? 2 : 1);   // (V as two parts of a 16-bit type)
  static constexpr int smem = ring + part + vs + TM * 4;
  static constexpr int fit = 227 * 1024 / (smem + 1024), ctas = fit > 4 ? 4 : fit < 1 ? 1 : fit;   // of an SM, which the registers have to allow too
  static_assert(smem <= 227 * 1024, "");
};

template <typename T, int TM, int RP, bool BACK>
__global__ void __launch_bounds__(kThreads, (Shape<T, TM, RP>::ctas)) adapters_kernel(const __grid_constant__ Args g) {
  using S = Shape<T, TM, RP>;
  constexpr int KC = S::KC, E = S::E;
  extern __shared__ __align__(16) char sm[];
  float* part = reinterpret_cast<float*>(sm + S::ring);
  char* vs = sm + S::ring + S::part;
  int* rowat = reinterpret_cast<int*>(vs + S::vs);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t crank, csize;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
  grid_dependency_wait();   // the plan
  const int tile = (int)(blockIdx.x / csize);
  int a, len;
  if (g.adapters) {
    // A row whose rank among its adapter's rows is a multiple of TM leads a tile; the tiles are in the order of their leaders.
    int *keys = reinterpret_cast<int*>(sm), *tiles = keys + kThreads, *mine = tiles + kWarps;   // (where the ring will be)
    int key = -1;
    if (tid < g.rows) {
      key = g.adapters[tid];
      if (key < 0 || key > g.count) key = g.count;
    }
    keys[tid] = key;
    __syncthreads();
    int rank = 0;
    for (int j = 0; j < g.rows; j += 4) {
      const int4 k = *reinterpret_cast<const int4*>(keys + j);
      rank += (k.x == key && j < tid) + (k.y == key && j + 1 < tid) + (k.z == key && j + 2 < tid) + (k.w == key && j + 3 < tid);
    }
    const bool leads = tid < g.rows && rank % TM == 0;
    const unsigned leaders = __ballot_sync(0xffffffffu, leads);
    if (lane == 0) tiles[warp] = __popc(leaders);
    __syncthreads();
    int before = __popc(leaders & ((1u << lane) - 1)), total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before += w < warp ? tiles[w] : 0;
      total += tiles[w];
    }
    if (tile >= total) return;   // (all CTAs of the cluster)
    if (leads && before == tile) {
      mine[0] = key;
      mine[1] = rank;
    }
    __syncthreads();
    a = mine[0];
    const int place = rank - mine[1];
    const bool in = key == a && place >= 0 && place < TM;
    if (in) rowat[place] = tid;
    len = __syncthreads_count(in);
  } else {
    const int4 head = *reinterpret_cast<const int4*>(g.head);
    if (!plan_is_of(head, g.rows, g.count) || tile >= head.x) return;   // (all CTAs of the cluster)
    a = g.tile_adapter[tile];
    const int first = g.tile_first[tile];
    len = min(TM, g.start[a + 1] - first);
    if (tid < len) rowat[tid] = g.order[first + tid];
    __syncthreads();
  }
  const T *X = static_cast<const T*>(g.X), *Y = static_cast<const T*>(g.Y);
  T* out = static_cast<T*>(g.out);
  const int K = g.K, N = g.N, R = g.R;
  const int nn = (N + KC - 1) / KC, nper = (nn + (int)csize - 1) / (int)csize, n0 = min(nn, (int)crank * nper), n1 = min(nn, n0 + nper);
  const auto store_values = [&](const char* src, int c0) {   // [len][KC] in shared memory -> out, value by value
    const int q = tid % KC, c = c0 + q;
    if (c >= N) return;
#pragma unroll 4
    for (int r = tid / KC; r < len; r += kThreads / KC) out[(size_t)rowat[r] * N + c] = reinterpret_cast<const T*>(src + r * S::xs)[q];
  };
  if (a == g.count) {   // rows without an adapter
    if (out == Y) return;
    for (int n = n0; n < n1; ++n) {
      const auto row = [&](int r) { return Y && r < len ? Y + (size_t)rowat[r] * N : nullptr; };
      load_rows<T, TM, S::pieces>(sm, S::xs, row, n * KC, N, g.vy, g.out);
      copies_end_group();
      copies_wait<0>();
      __syncthreads();
      store_values(sm, n * KC);
      __syncthreads();
    }
    return;
  }
  const T *F1 = static_cast<const T*>(g.F1) + (size_t)a * R * K, *F2 = static_cast<const T*>(g.F2) + (size_t)a * R * N;
  // a factor's chunk: KC features by the ranks, as it lies in memory
  const auto load_factor = [&](char* dst, const T* F, int n, bool long_rows, int c0) {
    if (long_rows)
      load_rows<T, RP, S::pieces>(dst, S::xs, [&](int r) { return r < R ? F + (size_t)r * n : nullptr; }, c0, n, false, F);
    else
      load_rows<T, KC, RP / E>(dst, S::ls, [&](int r) { return c0 + r < n ? F + (size_t)(c0 + r) * R : nullptr; }, 0, R, false, F);
  };
  Rows<T, BACK ? RP : KC, BACK ? S::pieces : RP / E> f1;
  const int rank_bytes = min(16, max(0, (R - (int)(tid % (RP / E)) * E) * (int)sizeof(T)));
  f1.set([&](int r) { return BACK ? (r < R ? F1 + (size_t)r * K : nullptr) : F1 + (size_t)r * R; }, F1);
  // a chunk of a factor whose rows are features: KC rows of R ranks, in the last chunk fewer
  const auto load_ranks = [&](const auto& f, char* dst, int c0, int n) {
    constexpr int EACH = kThreads / (RP / E);
    dst += tid / (RP / E) * S::ls + tid % (RP / E) * 16;
#pragma unroll
    for (int i = 0; i < (KC + EACH - 1) / EACH; ++i) {
      const int r = tid / (RP / E) + i * EACH;
      if (KC % EACH != 0 && r >= KC) break;
      const int bytes = c0 + r < n ? rank_bytes : 0;
      copy16(dst + i * EACH * S::ls, bytes ? f.from[i] + (size_t)c0 * R * sizeof(T) : f.from[0], bytes);
    }
  };
  Rows<T, TM, S::pieces> xr;
  xr.set([&](int r) { return r < len ? X + (size_t)rowat[r] * K : nullptr; }, X);

  // ---- V: this CTA's part of the sum over K ----
  const int nk = (K + KC - 1) / KC, kper = (nk + (int)csize - 1) / (int)csize, k0 = min(nk, (int)crank * kper), k1 = min(nk, k0 + kper);
  const auto load_k = [&](int k) {
    if (k < k1) {
      char* st = sm + (k - k0) % S::stages * S::stage;
      const int c0 = k * KC, bytes = piece_bytes<T, S::pieces>(c0, K);
      if (g.vx)
        xr.load(st, S::xs, (size_t)c0 * sizeof(T), bytes);
      else
        load_rows<T, TM, S::pieces>(st, S::xs, [&](int r) { return r < len ? X + (size_t)rowat[r] * K : nullptr; }, c0, K, false, X);
      st += TM * S::xs;
      if (!g.v1) {
        load_factor(st, F1, K, BACK, c0);
      } else if constexpr (BACK) {
        f1.load(st, S::xs, (size_t)c0 * sizeof(T), bytes);
      } else {
        load_ranks(f1, st, c0, K);
      }
    }
    copies_end_group();
  };
  // fp32: a lane has rows lr + 8 i, and ranks lc + 4 j (BACK) or 8 lc + j of its warp's group
  constexpr int RC = RP < 32 ? RP : 32, LC = RC / 4, LR = TM / 8;
  constexpr bool F32 = sizeof(T) == 4;
  float acc[F32 ? LR : RP / 8][F32 ? LC : 4] = {};
  const int mg = warp % S::MG, kg = F32 ? warp / S::CG : warp / S::MG, cg = F32 ? warp % S::CG : 0, lr = lane >> 2, lc = lane & 3;
#pragma unroll
  for (int s = 0; s < S::stages - 1; ++s) load_k(k0 + s);
  for (int k = k0; k < k1; ++k) {
    copies_wait<S::stages - 2>();
    __syncthreads();
    load_k(k + S::stages - 1);
    const char *xt = sm + (k - k0) % S::stages * S::stage, *ft = xt + TM * S::xs;
    if constexpr (F32) {
      constexpr int KW = KC / S::KG;   // 4 or 8, with groups of ranks more
#pragma unroll 2
      for (int q = kg * KW; q < (kg + 1) * KW; q += 4) {
        float x[LR][4];
#pragma unroll
        for (int i = 0; i < LR; ++i) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(xt + (lr + 8 * i) * S::xs + q * 4);
        if (BACK) {
#pragma unroll
          for (int j = 0; j < LC; ++j) {
            const float4 f = *reinterpret_cast<const float4*>(ft + (cg * 32 + lc + 4 * j) * S::xs + q * 4);
#pragma unroll
            for (int i = 0; i < LR; ++i) acc[i][j] = fmaf(x[i][0], f.x, fmaf(x[i][1], f.y, fmaf(x[i][2], f.z, fmaf(x[i][3], f.w, acc[i][j]))));
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < LC; j += 4) {
              const float4 f = *reinterpret_cast<const float4*>(ft + (q + u) * S::ls + (cg * 32 + lc * LC + j) * 4);
#pragma unroll
              for (int i = 0; i < LR; ++i) {
                acc[i][j] = fmaf(x[i][u], f.x, acc[i][j]);
                acc[i][j + 1] = fmaf(x[i][u], f.y, acc[i][j + 1]);
                acc[i][j + 2] = fmaf(x[i][u], f.z, acc[i][j + 2]);
                acc[i][j + 3] = fmaf(x[i][u], f.w, acc[i][j + 3]);
              }
            }
        }
      }
    } else {
      constexpr int KW = KC / S::KG;   // 32 or 16
#pragma unroll
      for (int q = kg * KW; q < (kg + 1) * KW; q += 16) {
        uint32_t x[4];
        a_block(x, xt + mg * 16 * S::xs + q * 2, S::xs);
#pragma unroll
        for (int j = 0; j < RP; j += 16) {
          uint32_t f[4];
          if (BACK)
            b_block<true>(f, ft + j * S::xs + q * 2, S::xs);
          else
            b_block<false>(f, ft + q * S::ls + j * 2, S::ls);
          mma16<T>(acc[j / 8], x, f[0], f[1]);
          mma16<T>(acc[j / 8 + 1], x, f[2], f[3]);
        }
      }
    }
  }
  copies_wait<0>();
  __syncthreads();
  // the warps' parts, then the cluster's
  float* red = reinterpret_cast<float*>(sm) + kg * TM * RP;
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < LR; ++i)
#pragma unroll
      for (int j = 0; j < LC; ++j) red[(lr + 8 * i) * RP + cg * 32 + (BACK ? lc + 4 * j : lc * LC + j)] = acc[i][j];
  } else {
#pragma unroll
    for (int j = 0; j < RP / 8; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(&red[(mg * 16 + lr + 8 * h) * RP + j * 8 + lc * 2]) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
  }
  __syncthreads();
  for (int i = tid; i < TM * RP; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < S::KG; ++q) v += reinterpret_cast<const float*>(sm)[q * TM * RP + i];
    part[i] = v;
  }
  __syncthreads();
  // (set here, and not before: what the second product needs takes no registers of the first)
  Rows<T, BACK ? KC : RP, BACK ? RP / E : S::pieces> f2;
  f2.set([&](int r) { return BACK ? F2 + (size_t)r * R : (r < R ? F2 + (size_t)r * N : nullptr); }, F2);
  Rows<T, TM, S::pieces> yr;
  if (Y) yr.set([&](int r) { return r < len ? Y + (size_t)rowat[r] * N : nullptr; }, Y);
  constexpr int STORES = TM * S::pieces / kThreads;
  T* outat[STORES];   // where a thread's pieces of a chunk go, in the first one
#pragma unroll
  for (int i = 0; i < STORES; ++i) {
    const int r = tid / S::pieces + i * (kThreads / S::pieces);
    outat[i] = out + (size_t)(r < len ? rowat[r] : 0) * N + tid % S::pieces * E;
  }
  const auto store_chunk = [&](const char* src, int c0) {
    if (!g.vy) return store_values(src, c0);
    const int q = tid % S::pieces;
    if (c0 + q * E >= N) return;   // (rows of whole pieces)
#pragma unroll
    for (int i = 0; i < STORES; ++i)
      if (tid / S::pieces + i * (kThreads / S::pieces) < len)
        *reinterpret_cast<uint4*>(outat[i] + c0) = *reinterpret_cast<const uint4*>(src + (tid / S::pieces + i * (kThreads / S::pieces)) * S::xs + q * 16);
  };
  const auto load_n = [&](int n) {
    if (n < n1) {
      char* st = sm + (n - n0) % S::stages * S::stage;
      const int c0 = n * KC, bytes = piece_bytes<T, S::pieces>(c0, N);
      if (Y && g.vy)
        yr.load(st, S::xs, (size_t)c0 * sizeof(T), bytes);
      else if (Y)
        load_rows<T, TM, S::pieces>(st, S::xs, [&](int r) { return r < len ? Y + (size_t)rowat[r] * N : nullptr; }, c0, N, false, Y);
      st += TM * S::xs;
      if (!g.v2) {
        load_factor(st, F2, N, !BACK, c0);
      } else if constexpr (BACK) {
        load_ranks(f2, st, c0, N);
      } else {
        f2.load(st, S::xs, (size_t)c0 * sizeof(T), bytes);
      }
    }
    copies_end_group();
  };
#pragma unroll
  for (int s = 0; s < S::stages - 1; ++s) load_n(n0 + s);   // while the cluster's parts are joined
  const float c = g.scale ? g.scale[a] : 1.f;
  if (csize > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = tid * 2; i < TM * RP; i += kThreads * 2) {
    float2 v = make_float2(0.f, 0.f);
    if (csize == 1) {
      v = *reinterpret_cast<const float2*>(part + i);
    } else {
      float2 from[8];
#pragma unroll
      for (uint32_t p = 0; p < 8; ++p) {
        from[p] = make_float2(0.f, 0.f);
        if (p < csize) {
          uint32_t at;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_at(part + i)), "r"(p));
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(from[p].x), "=f"(from[p].y) : "r"(at) : "memory");
        }
      }
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        v.x += from[p].x;
        v.y += from[p].y;
      }
    }
    const int r = i / RP, j = i - r * RP;
    // (Ranks that are not there are zero whatever the row holds: an infinity times their zeros would be NaN, and so would the whole row of out.)
    v.x = j < R ? v.x * c : 0.f;
    v.y = j + 1 < R ? v.y * c : 0.f;
    T* to = reinterpret_cast<T*>(vs + r * S::ls) + j;
    to[0] = (T)v.x;
    to[1] = (T)v.y;
    if constexpr (sizeof(T) == 2) {   // what the rounding left (of an infinity nothing)
      T* rest = reinterpret_cast<T*>(vs + (TM + r) * S::ls) + j;
      const float a0 = (float)to[0], a1 = (float)to[1];
      rest[0] = fabsf(a0) < __int_as_float(0x7f800000) ? (T)(v.x - a0) : (T)0.f;
      rest[1] = fabsf(a1) < __int_as_float(0x7f800000) ? (T)(v.y - a1) : (T)0.f;
    }
    if (g.V && crank == 0 && r < len) {
      T* w = static_cast<T*>(g.V) + (size_t)rowat[r] * R + j;
      if (j < R) w[0] = to[0];
      if (j + 1 < R) w[1] = to[1];
    }
  }
  __syncthreads();
  if (csize > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this CTA reads no other's part any more

  // ---- out = Y + V F2 ----
  constexpr int NG = kWarps / (TM / 16);
  uint32_t va[F32 ? 1 : RP / 16][4], vr[F32 ? 1 : RP / 16][4];
  if constexpr (!F32) {
#pragma unroll
    for (int j = 0; j < RP / 16; ++j) {
      a_block(va[j], vs + mg * 16 * S::ls + j * 32, S::ls);
      a_block(vr[j], vs + (TM + mg * 16) * S::ls + j * 32, S::ls);
    }
  }
  for (int n = n0; n < n1; ++n) {
    copies_wait<S::stages - 2>();
    __syncthreads();
    load_n(n + S::stages - 1);
    char* yt = sm + (n - n0) % S::stages * S::stage;
    const char* ft = yt + TM * S::xs;
    if constexpr (F32) {
      // a warp has 16 columns of some rows, a lane four of them (BACK: every fourth, whose ranks lie on other banks) and every eighth row
      constexpr int WC = KC / 16, RW = TM / (kWarps / WC), OR = RW / 8;
      const int wr = warp / WC * RW + lr, wc = warp % WC * 16 + (BACK ? lc : lc * 4);
      float o[OR][4];
#pragma unroll
      for (int i = 0; i < OR; ++i)
        *reinterpret_cast<float4*>(o[i]) = !BACK && Y ? *reinterpret_cast<const float4*>(yt + (wr + 8 * i) * S::xs + wc * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
      for (int j = 0; j < RP; j += 4) {
        float v[OR][4], f[4][4];   // f: [rank][column], BACK: [column][rank]
#pragma unroll
        for (int i = 0; i < OR; ++i) *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(vs + (wr + 8 * i) * S::ls + j * 4);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *reinterpret_cast<float4*>(f[u]) = BACK ? *reinterpret_cast<const float4*>(ft + (wc + 4 * u) * S::ls + j * 4)
                                                  : *reinterpret_cast<const float4*>(ft + (j + u) * S::xs + wc * 4);
#pragma unroll
        for (int i = 0; i < OR; ++i)
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[i][h] = fmaf(v[i][u], BACK ? f[h][u] : f[u][h], o[i][h]);
      }
#pragma unroll
      for (int i = 0; i < OR; ++i) {
        float* to = reinterpret_cast<float*>(yt + (wr + 8 * i) * S::xs) + wc;
        if (BACK) {
#pragma unroll
          for (int h = 0; h < 4; ++h) to[4 * h] = o[i][h];
        } else {
          *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(o[i]);
        }
      }
    } else {
      constexpr int NW = KC / NG;   // columns of a warp: 32 or 16
      const int nc = (warp / S::MG) * NW;
#pragma unroll
      for (int q = 0; q < NW; q += 16) {
        uint32_t* at = reinterpret_cast<uint32_t*>(yt + (mg * 16 + lr) * S::xs + (nc + q + lc * 2) * 2);   // two columns; of the other half 4 words on, of eight rows more
        float o[2][4] = {};
        if (Y) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 y = unpack2<T>(at[h * 4 + e * 8 * (S::xs / 4)]);
              o[h][2 * e] = y.x;
              o[h][2 * e + 1] = y.y;
            }
        }
#pragma unroll
        for (int j = 0; j < RP; j += 16) {
          uint32_t f[4];
          if (BACK)
            b_block<true>(f, ft + (nc + q) * S::ls + j * 2, S::ls);
          else
            b_block<false>(f, ft + j * S::xs + (nc + q) * 2, S::xs);
          mma16<T>(o[0], va[j / 16], f[0], f[1]);
          mma16<T>(o[1], va[j / 16], f[2], f[3]);
          mma16<T>(o[0], vr[j / 16], f[0], f[1]);
          mma16<T>(o[1], vr[j / 16], f[2], f[3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) at[h * 4 + e * 8 * (S::xs / 4)] = pack2<T>(o[h][2 * e], o[h][2 * e + 1]);
      }
    }
    __syncthreads();
    store_chunk(yt, n * KC);
  }
  copies_wait<0>();
  if (csize > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- dA and dB --------------------------------------------------------------------------------------------------------------
struct GradArgs {
  int rows, I, O, R, count, tiles_i, ranges;
  const void *X, *W, *V, *dY;   // [rows][I], [rows][R], [rows][R], [rows][O]
  const int *start, *order, *head;
  void *dA, *dB;
  float* partial;               // [range][2][I + O][RP]
  int vx, vy, vr;
};
constexpr int kFeatures = 128;   // of a CTA of the gradients
template <typename T, int RP>
struct GradShape {
  static constexpr int E = 16 / sizeof(T), LT = kFeatures, KT = sizeof(T) == 4 ? 32 : 64;   // features and rows of a step
  static constexpr int pieces = LT / E, zs = LT * (int)sizeof(T) + 16, ws = RP * (int)sizeof(T) + 16;
  static constexpr int stage = KT * (zs + ws), stages = 3;
  static constexpr int index = 2 * KT * 4, table = 1024;   // rows of two steps; adapters whose starts fit beside them
  static constexpr int smem = stages * stage + index + table * 4;
  static constexpr int ctas() { return 227 * 1024 / (smem + 1024); }   // of an SM
};
__device__ __forceinline__ int range_rows(const GradArgs& g) {   // of a range: a multiple of 16
  const int each = (g.head[1] + g.ranges - 1) / g.ranges;
  return max(16, (each + 15) / 16 * 16);
}
__device__ __forceinline__ int adapter_at(const int* start, int count, int pos) {   // the adapter that has row `pos` of the order
  int a = 0, b = count + 1;
  while (b - a > 1) {
    const int c = (a + b) / 2;
    if (start[c] <= pos) a = c; else b = c;
  }
  return a;
}
// The steps of a range: up to KT rows of one adapter each.
struct Steps {
  const int* start;
  int count, end, pos, a, stop;   // stop: where the adapter's rows (of the range) end
  __device__ Steps(const int* start_, int count_, int b, int e) : start(start_), count(count_), end(e), pos(b), a(0), stop(b) { find(); }
  __device__ void find() {
    if (pos >= end) return;
    a = adapter_at(start, count, pos);
    stop = min(end, start[a + 1]);
  }
  __device__ bool done() const { return pos >= end; }
  __device__ void next(int kt) {
    pos = min(pos + kt, stop);
    if (pos == stop) find();
  }
};

template <typename T, int RP>
__global__ void __launch_bounds__(kThreads) adapter_grads_kernel(const __grid_constant__ GradArgs g) {
  using S = GradShape<T, RP>;
  constexpr int KT = S::KT, LT = S::LT, E = S::E;
  constexpr bool F32 = sizeof(T) == 4;
  extern __shared__ __align__(16) char sm[];
  grid_dependency_wait();
  if (!plan_is_of(*reinterpret_cast<const int4*>(g.head), g.rows, g.count)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool second = (int)blockIdx.x >= g.tiles_i;   // dB
  const int L = second ? g.O : g.I, l0 = ((int)blockIdx.x - (second ? g.tiles_i : 0)) * LT, R = g.R;
  const T *Z = static_cast<const T*>(second ? g.dY : g.X), *W = static_cast<const T*>(second ? g.V : g.W);
  T* out = static_cast<T*>(second ? g.dB : g.dA);
  const bool vz = second ? g.vy : g.vx;
  const int per = range_rows(g), b = min(g.head[1], (int)blockIdx.y * per), e = min(g.head[1], b + per);
  // Where the adapters' rows start, beside the ring where they fit: a step that begins an adapter searches them.
  int *index = reinterpret_cast<int*>(sm + S::stages * S::stage), *table = index + 2 * KT;
  const bool fits = g.count + 2 <= S::table;
  if (fits)
    for (int i = tid; i < g.count + 2; i += kThreads) table[i] = g.start[i];
  __syncthreads();
  const int* start = fits ? table : g.start;
  Steps load(start, g.count, b, e), at = load;
  int loaded = 0;
  // The rows of a step come from the order: read one step ahead into a register, and into shared memory before the barrier that the copies wait for.
  int ahead = tid < KT && load.pos + tid < e ? g.order[load.pos + tid] : 0;
  const auto next_rows = [&] {
    if (tid < KT) index[loaded % 2 * KT + tid] = ahead;
    if (load.done()) return;
    Steps then = load;
    then.next(KT);
    ahead = tid < KT && then.pos + tid < e ? g.order[then.pos + tid] : 0;
  };
  const auto load_step = [&] {
    if (!load.done()) {
      char* st = sm + loaded % S::stages * S::stage;
      const int n = min(KT, load.stop - load.pos);
      const int* rows = index + loaded % 2 * KT;
      load_rows<T, KT, S::pieces>(st, S::zs, [&](int r) { return r < n ? Z + (size_t)rows[r] * L : nullptr; }, l0, L, vz, Z);
      load_rows<T, KT, RP / E>(st + KT * S::zs, S::ws, [&](int r) { return r < n ? W + (size_t)rows[r] * R : nullptr; }, 0, R, g.vr, W);
      load.next(KT);
      ++loaded;
    }
    copies_end_group();
  };
  next_rows();
#pragma unroll
  for (int s = 0; s < S::stages - 1; ++s) {
    __syncthreads();
    load_step();
    next_rows();
  }
  // A warp has sixteen features and all ranks; fp32: a lane LR of them and LC ranks
  constexpr int LC = RP == 16 ? 2 : 4, CGN = RP / LC, LR = CGN / 2;   // 16 / (32 / CGN)
  float acc[F32 ? LR : RP / 8][F32 ? LC : 4] = {};
  const int lr = F32 ? lane / CGN : lane >> 2, lc = F32 ? lane % CGN : lane & 3;
  for (int k = 0; !at.done(); ++k) {
    copies_wait<S::stages - 2>();
    __syncthreads();
    load_step();
    next_rows();
    const char *zt = sm + k % S::stages * S::stage, *wt = zt + KT * S::zs;
    if constexpr (F32) {
#pragma unroll 4
      for (int t = 0; t < KT; ++t) {
        const float *z = reinterpret_cast<const float*>(zt + t * S::zs) + warp * 16 + lr * LR, *w = reinterpret_cast<const float*>(wt + t * S::ws) + lc * LC;
        float x[LR], y[LC];
#pragma unroll
        for (int i = 0; i < LR; i += 4) *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(z + i);
        if constexpr (LC == 2) *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(w);
        else *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(w);
#pragma unroll
        for (int i = 0; i < LR; ++i)
#pragma unroll
          for (int j = 0; j < LC; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < KT; t += 16) {
        uint32_t z[4];
        a_of_k(z, zt + t * S::zs + warp * 32, S::zs);
#pragma unroll
        for (int j = 0; j < RP; j += 16) {
          uint32_t w[4];
          b_block<false>(w, wt + t * S::ws + j * 2, S::ws);
          mma16<T>(acc[j / 8], z, w[0], w[1]);
          mma16<T>(acc[j / 8 + 1], z, w[2], w[3]);
        }
      }
    }
    const int a = at.a;
    const bool last = at.pos + KT >= at.stop;
    at.next(KT);
    if (!last) continue;
    // the adapter's rows of this range end here
    const int ab = start[a], ae = start[a + 1];
    const bool whole = ab >= b && ae <= e;
    float* p = g.partial + ((size_t)(blockIdx.y * 2 + (ab >= b ? 1 : 0)) * (g.I + g.O) + (second ? g.I : 0)) * RP;
    const auto put = [&](int l, int r, float v) {
      l += l0;
      if (l >= L) return;
      if (!whole)
        p[(size_t)l * RP + r] = v;
      else if (r < R)
        out[second ? ((size_t)a * R + r) * L + l : ((size_t)a * L + l) * R + r] = (T)v;
    };
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < LR; ++i)
#pragma unroll
        for (int j = 0; j < LC; ++j) {
          put(warp * 16 + lr * LR + i, lc * LC + j, acc[i][j]);
          acc[i][j] = 0.f;
        }
    } else {
#pragma unroll
      for (int j = 0; j < RP / 8; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          put(warp * 16 + lr + (v >> 1) * 8, j * 8 + lc * 2 + (v & 1), acc[j][v]);
          acc[j][v] = 0.f;
        }
    }
  }
  copies_wait<0>();
}

// Adapters that lie in several ranges: the sum of their parts in the order of the ranges.  Adapters without rows: zero.
template <typename T, int RP>
__global__ void __launch_bounds__(kThreads) join_grads_kernel(const __grid_constant__ GradArgs g) {
  grid_dependency_wait();
  if (!plan_is_of(*reinterpret_cast<const int4*>(g.head), g.rows, g.count)) return;
  const int a = blockIdx.x, ab = g.start[a], ae = g.start[a + 1], per = range_rows(g);
  const int r0 = ab / per, r1 = ae > ab ? (ae - 1) / per : r0;
  if (ae > ab && r0 == r1) return;
  // A thread has a feature and four ranks: neighbours have neighbouring ranks of dA, and neighbouring features of dB, as they lie there.
  constexpr int Q = RP / 4;
  const int quads = (g.R + 3) / 4, na = g.dA ? g.I * quads : 0, n = na + (g.dB ? g.O * quads : 0);
  const size_t step = (size_t)(g.I + g.O) * Q;
  const bool vec = g.R % 4 == 0 && reinterpret_cast<uintptr_t>(g.dA) % (4 * sizeof(T)) == 0;
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < n; i += gridDim.y * kThreads) {
    const bool second = i >= na;
    const int x = second ? i - na : i, q = second ? x / g.O : x % quads, l = second ? x - q * g.O : x / quads;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ae > ab) {
      const float4* p = reinterpret_cast<const float4*>(g.partial) + ((size_t)(second ? g.I : 0) + l) * Q + q;
      v = p[(size_t)(2 * r0 + 1) * step];
#pragma unroll 4
      for (int k = r0 + 1; k <= r1; ++k) {
        const float4 w = p[(size_t)(2 * k) * step];
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
    if (!second) {
      T* out = static_cast<T*>(g.dA) + ((size_t)a * g.I + l) * g.R + q * 4;
      if (vec) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = v;
        else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (q * 4 + j < g.R) out[j] = (T)e[j];
      }
    } else {
      T* out = static_cast<T*>(g.dB) + ((size_t)a * g.R + q * 4) * g.O + l;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (q * 4 + j < g.R) out[(size_t)j * g.O] = (T)e[j];
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
bool rows16(const void* p, size_t row_bytes) { return !(reinterpret_cast<uintptr_t>(p) & 15) && row_bytes % 16 == 0; }

template <typename T, int TM, int RP, bool BACK>
int launch_tiles(const Args& g, const Plan& p, cudaStream_t st) {
  using S = Shape<T, TM, RP>;
  const auto kern = adapters_kernel<T, TM, RP, BACK>;
  static std::atomic<int> set[64];
  B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), set, S::smem));
  // CTAs of a tile: as many as the machine is likely to hold at once, with a chunk of the longer product for each
  static ClusterCounts counts;
  int c = 1, dev = 0;
  B200CP_CUDA_OK(cudaGetDevice(&dev));
  const int chunks = std::max(ceil_div(g.K, S::KC), ceil_div(g.N, S::KC));
  for (int q = 2; q <= 8 && q <= chunks; q *= 2) {
    int n = 0;
    B200CP_CUDA_OK(resident_clusters(kern, kThreads, S::smem, dev, q, counts, &n));
    if (p.likely <= n) c = q;
  }
  B200CP_CUDA_OK(launch_clusters(kern, p.tiles, c, kThreads, S::smem, st, g));
  B200CP_LAUNCH_OK("adapters_kernel");
  return B200CP_OK;
}
template <typename T, bool BACK>
int launch_rank(const Args& g, const Plan& p, cudaStream_t st) {
#define RANK(RP) return p.tm == 64 ? launch_tiles<T, 64, RP, BACK>(g, p, st) : launch_tiles<T, 16, RP, BACK>(g, p, st)
  if (g.R <= 16) RANK(16);
  if (g.R <= 32) RANK(32);
  if (g.R <= 64) RANK(64);
  RANK(128);
#undef RANK
}
int padded(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }
template <typename T, int RP>
int ranges_for(int rows, int I, int O) {   // as many as the machine holds at once with all tiles of features
  using S = GradShape<T, RP>;
  const int tiles = ceil_div(I, S::LT) + ceil_div(O, S::LT);
  return std::max(1, std::min({148 * S::ctas() / tiles, ceil_div(rows, 16), 65535}));
}
int ranges_of(int rows, int I, int O, int R, int type) {
  const bool f32 = type == B200CP_FLOAT32;
  switch (padded(R)) {
    case 16: return f32 ? ranges_for<float, 16>(rows, I, O) : ranges_for<__half, 16>(rows, I, O);
    case 32: return f32 ? ranges_for<float, 32>(rows, I, O) : ranges_for<__half, 32>(rows, I, O);
    case 64: return f32 ? ranges_for<float, 64>(rows, I, O) : ranges_for<__half, 64>(rows, I, O);
    default: return f32 ? ranges_for<float, 128>(rows, I, O) : ranges_for<__half, 128>(rows, I, O);
  }
}
template <typename T, int RP>
int launch_grads(const GradArgs& g, cudaStream_t st) {
  using S = GradShape<T, RP>;
  static std::atomic<int> set[64];
  const int tiles = g.tiles_i + (g.dB ? ceil_div(g.O, S::LT) : 0);
  if (g.rows) {
    const auto kern = adapter_grads_kernel<T, RP>;
    B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), set, S::smem));
    B200CP_CUDA_OK(launch_kernel(kern, dim3(tiles, g.ranges), dim3(kThreads), S::smem, st, true, g));
    B200CP_LAUNCH_OK("adapter_grads_kernel");
  }
  const long n = (long)ceil_div(g.R, 4) * ((g.dA ? g.I : 0) + (g.dB ? g.O : 0));
  const int per = (int)std::min<long>((n + kThreads - 1) / kThreads, std::max(1, 16 * 148 / g.count));
  B200CP_CUDA_OK(launch_kernel(join_grads_kernel<T, RP>, dim3(g.count, per), dim3(kThreads), 0, st, true, g));
  B200CP_LAUNCH_OK("join_grads_kernel");
  return B200CP_OK;
}
template <typename T>
int launch_grads_rank(const GradArgs& g, cudaStream_t st) {
  switch (padded(g.R)) {
    case 16: return launch_grads<T, 16>(g, st);
    case 32: return launch_grads<T, 32>(g, st);
    case 64: return launch_grads<T, 64>(g, st);
    default: return launch_grads<T, 128>(g, st);
  }
}
int check_sizes(const char* who, int rows, int I, int O, int R, int count, int type) {
  if (rows < 0 || I < 1 || O < 1 || R < 1 || count < 1)
    return fail(B200CP_ERR_INVALID_ARG, "%s: rows=%d I=%d O=%d R=%d count=%d", who, rows, I, O, R, count);
  if (type != B200CP_FLOAT32 && type != B200CP_BFLOAT16 && type != B200CP_FLOAT16)
    return fail(B200CP_ERR_INVALID_ARG, "%s: type %d", who, type);
  if (R > kMostRank || count > kMostAdapters || rows > (1 << 28) || I > (1 << 24) || O > (1 << 24))
    return fail(B200CP_ERR_UNSUPPORTED, "%s: rank %d (at most %d), %d adapters (at most %d), %d rows (2^28), %d and %d features (2^24)", who, R,
                kMostRank, count, kMostAdapters, rows, I, O);
  return B200CP_OK;
}
void plan_into(const int* plan, const Plan& p, const int** head, const int** start, const int** order) {
  *head = plan;
  *start = plan + p.start;
  *order = plan + p.order;
}
template <bool BACK>
int run_tiles(int type, Args& g, const Plan& p, const int* plan, cudaStream_t st) {
  const size_t size = type == B200CP_FLOAT32 ? 4 : 2;
  if (plan) {
    plan_into(plan, p, &g.head, &g.start, &g.order);
    g.tile_adapter = plan + p.adapter;
    g.tile_first = plan + p.first;
  }
  g.vx = rows16(g.X, g.K * size);
  g.vy = rows16(g.out, g.N * size) && (!g.Y || rows16(g.Y, g.N * size));
  g.v1 = rows16(g.F1, (BACK ? g.K : g.R) * size) && (size_t)g.K * g.R * size % 16 == 0;
  g.v2 = rows16(g.F2, (BACK ? g.R : g.N) * size) && (size_t)g.N * g.R * size % 16 == 0;
  if (type == B200CP_FLOAT32) return launch_rank<float, BACK>(g, p, st);
  if (type == B200CP_BFLOAT16) return launch_rank<__nv_bfloat16, BACK>(g, p, st);
  return launch_rank<__half, BACK>(g, p, st);
}
size_t w_bytes(int rows, int R, int type) { return align_up((size_t)rows * R * (type == B200CP_FLOAT32 ? 4 : 2), 256); }

}  // namespace

int adapters_device_status(int* out) {
  int v = 0, zero = 0;
  B200CP_CUDA_OK(cudaMemcpyFromSymbol(&v, g_adapters_status, sizeof(int)));
  if (v) B200CP_CUDA_OK(cudaMemcpyToSymbol(g_adapters_status, &zero, sizeof(int)));
  *out = v;
  return B200CP_OK;
}

}  // namespace b200cp

using namespace b200cp;

extern "C" {

size_t b200cp_adapter_plan_bytes(int rows, int count) {
  if (rows < 0 || count < 1 || count > kMostAdapters || rows > (1 << 28)) return 0;
  return plan_of(rows, count).ints * sizeof(int);
}

int b200cp_adapter_plan(int rows, int count, const int* adapters, void* plan, size_t plan_bytes, void* stream) {
  const size_t need = b200cp_adapter_plan_bytes(rows, count);
  if (!need) return fail(B200CP_ERR_INVALID_ARG, "b200cp_adapter_plan: %d rows, %d adapters (1 to %d)", rows, count, kMostAdapters);
  if ((rows && !adapters) || !plan) return fail(B200CP_ERR_INVALID_ARG, "b200cp_adapter_plan: null pointer");
  if (plan_bytes < need || (reinterpret_cast<uintptr_t>(plan) & 15))
    return fail(B200CP_ERR_WORKSPACE, "b200cp_adapter_plan: a 16-byte aligned plan of %zu bytes is needed, %zu given", need, plan_bytes);
  const Plan p = plan_of(rows, count);
  const int keys = count + 1;
  const int sorters = std::max(1, std::min({32, ceil_div(std::max(rows, 1), 32), 40000 / keys - 1}));   // counts: at most 156 KB
  const size_t smem = ((size_t)keys * sorters + keys + 1) * sizeof(int);
  static std::atomic<int> set[64];
  B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(plan_kernel), set, (int)smem));
  plan_kernel<<<1, 1024, smem, static_cast<cudaStream_t>(stream)>>>(rows, count, p.tm, sorters, adapters, static_cast<int*>(plan), p.adapter, p.first,
                                                                    p.order);
  B200CP_LAUNCH_OK("plan_kernel");
  return B200CP_OK;
}

int b200cp_dense_adapters(int rows, int I, int O, int R, int count, int type, const void* Y, const void* X, const void* A, const void* B,
                          const float* scale, const int* adapters, const void* plan, void* out, void* V, void* stream) {
  if (int rc = check_sizes("b200cp_dense_adapters", rows, I, O, R, count, type)) return rc;
  if (rows == 0) return B200CP_OK;
  if (!Y || !X || !A || !B || (!plan && !adapters) || !out) return fail(B200CP_ERR_INVALID_ARG, "b200cp_dense_adapters: null pointer");
  if (reinterpret_cast<uintptr_t>(plan) & 15) return fail(B200CP_ERR_INVALID_ARG, "b200cp_dense_adapters: the plan is not on a 16-byte boundary");
  if (!plan && rows > B200CP_ADAPTERS_WITHOUT_PLAN)
    return fail(B200CP_ERR_UNSUPPORTED, "b200cp_dense_adapters: %d rows without a plan (at most %d)", rows, B200CP_ADAPTERS_WITHOUT_PLAN);
  Args g{};
  g.rows = rows; g.K = I; g.N = O; g.R = R; g.count = count;
  g.X = X; g.Y = Y; g.F1 = A; g.F2 = B; g.scale = scale; g.out = out; g.V = V;
  g.adapters = plan ? nullptr : adapters;
  return run_tiles<false>(type, g, plan_of(rows, count), static_cast<const int*>(plan), static_cast<cudaStream_t>(stream));
}

size_t b200cp_dense_adapters_bwd_workspace_bytes(int rows, int I, int O, int R, int count, int type) {
  if (check_sizes("b200cp_dense_adapters_bwd_workspace_bytes", rows, I, O, R, count, type)) return 0;
  return w_bytes(rows, R, type) + (size_t)ranges_of(rows, I, O, R, type) * 2 * ((size_t)I + O) * padded(R) * sizeof(float);
}

int b200cp_dense_adapters_bwd(int rows, int I, int O, int R, int count, int type, const void* dY, const void* X, const void* V,
                              const void* A, const void* B, const float* scale, const void* plan, void* dX, void* dA, void* dB,
                              void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "b200cp_dense_adapters_bwd";
  if (int rc = check_sizes(who, rows, I, O, R, count, type)) return rc;
  if (!plan || (rows && (!dY || ((dX || dA) && (!A || !B)) || (dA && !X) || (dB && !V)))) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  if (reinterpret_cast<uintptr_t>(plan) & 15) return fail(B200CP_ERR_INVALID_ARG, "%s: the plan is not on a 16-byte boundary", who);
  const size_t need = b200cp_dense_adapters_bwd_workspace_bytes(rows, I, O, R, count, type);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, %zu given", who, need, workspace_bytes);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Plan p = plan_of(rows, count);
  const size_t size = type == B200CP_FLOAT32 ? 4 : 2;
  void* W = workspace;
  if (rows && (dX || dA)) {
    Args g{};
    g.rows = rows; g.K = O; g.N = dX ? I : 0; g.R = R; g.count = count;
    g.X = dY; g.F1 = B; g.F2 = A; g.scale = scale; g.out = dX; g.V = W;
    if (int rc = run_tiles<true>(type, g, p, static_cast<const int*>(plan), st)) return rc;
  }
  if (!dA && !dB) return B200CP_OK;
  GradArgs g{};
  g.rows = rows; g.I = I; g.O = O; g.R = R; g.count = count; g.ranges = ranges_of(rows, I, O, R, type);
  g.tiles_i = dA ? ceil_div(I, kFeatures) : 0;
  g.X = X; g.W = W; g.V = V; g.dY = dY; g.dA = dA; g.dB = dB;
  plan_into(static_cast<const int*>(plan), p, &g.head, &g.start, &g.order);
  g.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + w_bytes(rows, R, type));
  g.vx = rows16(X, I * size);
  g.vy = rows16(dY, O * size);
  g.vr = rows16(V, R * size) && R * size % 16 == 0;
  if (type == B200CP_FLOAT32) return launch_grads_rank<float>(g, st);
  if (type == B200CP_BFLOAT16) return launch_grads_rank<__nv_bfloat16>(g, st);
  return launch_grads_rank<__half>(g, st);
}

}  // extern "C"
