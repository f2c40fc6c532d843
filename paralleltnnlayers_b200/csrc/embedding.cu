// Embedding of tokens and its gradient.
//
//   out[s] = c W[t_s] (zeros where t_s is outside 0 .. V-1),  dW[v] = c sum over s with t_s = v of dY[s]
//
// The forward is a copy of rows, bound by HBM.  The gradient writes all of dW and reads dY once.  Rows of dY are added in the order in which their tokens
// lie in the batch, by sorting the tokens' places first, so that a result has the same bits each time (atomic sums would not):
//   1. one cluster of eight CTAs sorts the places by token (stable, digits of up to ten bits) while all other CTAs fill dW with zeros, which takes
//      longer where the table is large;
//   2. the sorted places are cut into chunks of equal length, whatever tokens they belong to: a thread adds its columns of a chunk's rows
//      in fp32 and stores a token's sum when the next one begins.  A token whose places reach over the end of a chunk leaves parts;
//   3. which are joined in their order, up to 64 by a CTA, and the sums of 64 by another launch: a token that makes up the whole batch has as many CTAs for its parts
//      as there are groups of 64 of them.
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"
#include "vec_io.cuh"

namespace b200cp {
namespace {

namespace cg = cooperative_groups;

enum { kInt32 = 0, kInt64 = 1 };

// A token as a key of 32 bits; V: none.
__device__ __forceinline__ uint32_t key_of(const void* tokens, int wide, size_t i, uint32_t V) {
  const long long t = wide ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
  return t >= 0 && t < (long long)V ? (uint32_t)t : V;
}

// ---- forward ------------------------------------------------------------------------------------------------------------------
struct Lookup {
  int rows, D, wide;
  uint32_t V;
  float scale;
  const void *tokens, *W;
  void* out;
};
constexpr int kEach = 4;   // groups of a thread, in flight together
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_kernel(const __grid_constant__ Lookup g) {
  grid_dependency_wait();
  const unsigned per = (unsigned)(g.D / VEC);   // groups of a row
  const size_t total = (size_t)g.rows * per, first = (size_t)blockIdx.x * (256 * kEach) + threadIdx.x;
  const T* W = static_cast<const T*>(g.W);
  Group<T, VEC> v[kEach];
  uint32_t key[kEach];
  unsigned col[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const size_t i = first + j * 256;
    key[j] = g.V;
    col[j] = 0;
    if (i < total) {
      const size_t row = total <= 0xffffffffu ? (size_t)((unsigned)i / per) : i / per;
      key[j] = key_of(g.tokens, g.wide, row, g.V);
      col[j] = (unsigned)(i - row * per) * VEC;
    }
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (key[j] < g.V) v[j] = load_group<T, VEC>(W + (size_t)key[j] * g.D + col[j]);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const size_t i = first + j * 256;
    if (i >= total) break;
    float x[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = key[j] < g.V ? to_float(v[j].v[k]) * g.scale : 0.f;
    store_group(static_cast<T*>(g.out) + i * VEC, pack<T>(x));
  }
}

// ---- gradient, 1: places by token, and zeros ------------------------------------------------------------------------------------
constexpr int kSorters = 8, kSortThreads = 1024, kFill = 4, kBins = 1024, kWarps = kSortThreads / 32;
struct Sort {
  int rows, wide, passes, bits;   // bits of a digit
  uint32_t V;
  const void* tokens;
  uint32_t *key[2], *place[2];
  int cap;                        // entries of a CTA
  uint4* zeros;                   // to be filled, from a 16-byte boundary on; `before` and `after` bytes beside
  size_t groups;
  unsigned char *head, *tail;
  int before, after;
};
__global__ void __cluster_dims__(kSorters, 1, 1) __launch_bounds__(kSortThreads) embedding_sort_kernel(const __grid_constant__ Sort g) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dependency_wait();
  if (blockIdx.x >= kSorters) {   // zeros
    // (a CTA has 64 KB and leaves: a table of 410 MB in 58 us, where CTAs that stay take 66)
    const size_t first = (size_t)(blockIdx.x - kSorters) * (kSortThreads * kFill) + tid;
#pragma unroll
    for (int i = 0; i < kFill; ++i)
      if (first + i * kSortThreads < g.groups) g.zeros[first + i * kSortThreads] = make_uint4(0, 0, 0, 0);
    if (blockIdx.x == kSorters) {
      if (tid < g.before) g.head[tid] = 0;
      if (tid < g.after) g.tail[tid] = 0;
    }
    return;
  }
  __shared__ uint32_t counts[kBins], start[kBins], next[kBins], sums[32];   // (counts are read by the other CTAs)
  __shared__ uint8_t mine[kWarps][kBins];   // of a warp's 32 entries
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), e0 = min((long long)g.rows, (long long)rank * g.cap), e1 = min((long long)g.rows, (long long)e0 + g.cap);
  const uint32_t bins = 1u << g.bits, mask = bins - 1;
  for (int pass = 0; pass < g.passes; ++pass) {
    const int shift = pass * g.bits;
    const uint32_t *key = g.key[(pass + 1) & 1], *place = g.place[(pass + 1) & 1];
    uint32_t *to_key = g.key[pass & 1], *to_place = g.place[pass & 1];
    const auto at = [&](int i) { return pass == 0 ? key_of(g.tokens, g.wide, i, g.V) : __ldcg(key + i); };
    counts[tid] = 0;
    __syncthreads();
    for (int i = e0 + tid; i < e1; i += kSortThreads) atomicAdd(&counts[(at(i) >> shift) & mask], 1u);
    cl.sync();
    // where the digit's entries of this CTA begin: behind those of all smaller digits, and of this one in the CTAs before
    uint32_t all = 0, before = 0;
#pragma unroll
    for (int q = 0; q < kSorters; ++q) {
      const uint32_t c = cl.map_shared_rank(counts, q)[tid];
      all += c;
      if (q < rank) before += c;
    }
    uint32_t run = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += v;
    }
    if (lane == 31) sums[warp] = run;
    __syncthreads();
    uint32_t base = lane < warp ? sums[lane] : 0;
    base = __reduce_add_sync(0xffffffffu, base);
    next[tid] = base + run - all + before;
    for (int i0 = e0; i0 < e1; i0 += kSortThreads) {
      const int i = i0 + tid;
      const bool in = i < e1;
      const uint32_t k = in ? at(i) : 0, p = in ? (pass == 0 ? (uint32_t)i : __ldcg(place + i)) : 0, d = (k >> shift) & mask;
      for (uint32_t b = lane; b < bins; b += 32) mine[warp][b] = 0;
      __syncwarp();
      const unsigned same = __match_any_sync(0xffffffffu, in ? d : 0xffffffffu), below = same & ((1u << lane) - 1);
      if (in && !below) mine[warp][d] = (uint8_t)__popc(same);
      __syncthreads();
      if (tid < (int)bins) {   // where the digit's entries of these 1024 begin, and the next ones'
        uint32_t s = next[tid];
        start[tid] = s;
#pragma unroll 8
        for (int w = 0; w < kWarps; ++w) s += mine[w][tid];
        next[tid] = s;
      }
      __syncthreads();
      if (in) {
        uint32_t to = start[d] + __popc(below);
        for (int w = 0; w < warp; ++w) to += mine[w][d];
        __stcg(to_key + to, k);
        __stcg(to_place + to, p);
      }
      __syncthreads();
    }
    cl.sync();   // all entries are in place, and nobody reads this CTA's counts any more
  }
}

// ---- gradient, 2: sums of chunks --------------------------------------------------------------------------------------------------
struct Sums {
  int rows, D, chunk, chunks;
  int lanes;                      // threads of a row's part: a power of two, at most 256
  uint32_t V;
  float scale;
  const uint32_t *key, *place;
  const void* dy;
  void* dW;
  float* parts;                   // [chunk][the token that began before, the one that goes on][D]
};
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 4) embedding_sums_kernel(const __grid_constant__ Sums g) {
  grid_dependency_wait();
  const int per = 256 / g.lanes, c = blockIdx.x * per + (int)threadIdx.x / g.lanes;
  const int col = ((int)blockIdx.y * g.lanes + ((int)threadIdx.x & (g.lanes - 1))) * VEC;
  if (c >= g.chunks || col >= g.D) return;
  const int e0 = c * g.chunk, e1 = (int)min((long long)g.rows, (long long)e0 + g.chunk);
  const T* dy = static_cast<const T*>(g.dy) + col;
  T* dW = static_cast<T*>(g.dW) + col;
  float* part = g.parts + (size_t)c * 2 * g.D + col;
  uint32_t now = g.key[e0];
  bool head = e0 > 0 && now < g.V && g.key[e0 - 1] == now;
  float acc[VEC] = {};
  const auto to_part = [&](float* to) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) to[i] = acc[i];
  };
  const auto to_row = [&] {
    float x[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = acc[i] * g.scale;
    store_group(dW + (size_t)now * g.D, pack<T>(x));
  };
  constexpr int U = 4;   // rows on their way together (64 registers: four CTAs an SM)
  for (int e = e0; e < e1 && now < g.V; e += U) {
    uint32_t key[U];
    Group<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) key[u] = e + u < e1 ? g.key[e + u] : g.V;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (key[u] < g.V) v[u] = load_group<T, VEC>(dy + (size_t)g.place[e + u] * g.D);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e + u >= e1 || now >= g.V) break;
      if (key[u] != now) {
        if (head) to_part(part);
        else to_row();
        head = false;
        now = key[u];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
        if (now >= g.V) break;
      }
      float x[VEC];
      unpack(v[u], x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += x[i];
    }
  }
  if (now >= g.V) return;
  if (head) to_part(part);
  else if (e1 < g.rows && g.key[e1] == now) to_part(part + g.D);
  else to_row();
}

// ---- gradient, 3: tokens of several chunks --------------------------------------------------------------------------------------------
// A token that goes on behind its first chunk has parts: that chunk's second one, and the first ones of the chunks that begin with it.  Chunks are taken in groups of 64.
//   grid (chunks, columns / 4096): what a token has within a group is added up by the CTA of its first chunk there, and kept in that chunk's place; or written, if that is all.
//   grid (groups, columns / 4096), where there are several: what a token has in the group where it begins and in those behind it.
// A thread has four columns.  (One CTA for all of a token's parts: 65536 times one token, rows of 64: 1140 us, so 68; of different tokens 74.)
constexpr int kJoinCols = 4096, kGroup = 64;
// The places from `first` on, `step` apart and before `end`, at which chunks begin with the token: they are the first ones.  All lanes have the answer.
__device__ __forceinline__ int begin_with(const Sums& g, uint32_t token, long long first, int step, long long end) {
  for (int n = 0;; n += 32) {
    const long long c = first + (long long)(n + (int)(threadIdx.x & 31)) * step;
    const unsigned not_it = ~__ballot_sync(0xffffffffu, c < end && g.key[c * g.chunk] == token);
    if (not_it) return n + __ffs(not_it) - 1;
  }
}
// s += a part's four columns, as many as there are.
__device__ __forceinline__ void add_part(const Sums& g, const float* from, int left, float (&s)[4]) {
  float v[4] = {};
  if ((g.D & 3) == 0) {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] = from[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] += v[i];
}
template <typename T>
__device__ __forceinline__ void store_row(const Sums& g, uint32_t token, int col, int left, const float (&s)[4]) {
  T* to = static_cast<T*>(g.dW) + (size_t)token * g.D + col;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) to[i] = from_float<T>(s[i] * g.scale);
}
template <typename T>
__global__ void __launch_bounds__(1024) embedding_join_kernel(const __grid_constant__ Sums g) {
  grid_dependency_wait();
  const int c = blockIdx.x;
  const long long e0 = (long long)c * g.chunk, e1 = e0 + g.chunk;
  if (e1 >= g.rows) return;
  const uint32_t now = g.key[e1];
  if (now >= g.V || g.key[e1 - 1] != now) return;
  const bool begun = e0 > 0 && g.key[e0 - 1] == now;   // in an earlier chunk
  if (begun && c % kGroup) return;
  const long long next = ((long long)c / kGroup + 1) * kGroup;   // group
  const int more = begin_with(g, now, c + 1, 1, min(next, (long long)g.chunks));
  const bool all = !begun && !(next < g.chunks && g.key[next * g.chunk] == now);
  const int col = blockIdx.y * kJoinCols + threadIdx.x * 4, left = g.D - col;
  if (left <= 0) return;
  float s[4] = {};
  float* place = g.parts + ((size_t)c * 2 + !begun) * g.D + col;
  add_part(g, place, left, s);
#pragma unroll 8
  for (int p = 1; p <= more; ++p) add_part(g, g.parts + (size_t)(c + p) * 2 * g.D + col, left, s);
  if (all) {
    store_row<T>(g, now, col, left, s);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) place[i] = s[i];
}
template <typename T>
__global__ void __launch_bounds__(1024) embedding_join_groups_kernel(const __grid_constant__ Sums g) {
  grid_dependency_wait();
  const long long first = (long long)blockIdx.x * kGroup, next = first + kGroup;
  if (next >= g.chunks) return;
  const uint32_t now = g.key[next * g.chunk];
  if (now >= g.V || g.key[next * g.chunk - 1] != now || (first > 0 && g.key[first * g.chunk - 1] == now)) return;   // (does not reach over the end, or began before)
  int before = 0;   // chunks of the group that end with other tokens
#pragma unroll
  for (int n = 0; n < kGroup; n += 32) before += __popc(__ballot_sync(0xffffffffu, g.key[(first + n + (threadIdx.x & 31) + 1) * g.chunk - 1] != now));
  const int more = begin_with(g, now, next, kGroup, g.chunks);
  const int col = blockIdx.y * kJoinCols + threadIdx.x * 4, left = g.D - col;
  if (left <= 0) return;
  float s[4] = {};
  add_part(g, g.parts + ((size_t)(first + before) * 2 + 1) * g.D + col, left, s);
#pragma unroll 8
  for (int p = 0; p < more; ++p) add_part(g, g.parts + (size_t)(next + (long long)p * kGroup) * 2 * g.D + col, left, s);
  store_row<T>(g, now, col, left, s);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int check_embedding(const char* who, int rows, int V, int D, int type, int number_type) {
  if (rows < 0 || V < 1 || D < 1) return fail(B200CP_ERR_INVALID_ARG, "%s: %d tokens of %d, rows of %d", who, rows, V, D);
  if (type < B200CP_FLOAT32 || type > B200CP_FLOAT16) return fail(B200CP_ERR_INVALID_ARG, "%s: type %d", who, type);
  if (number_type != kInt32 && number_type != kInt64) return fail(B200CP_ERR_INVALID_ARG, "%s: tokens of type %d", who, number_type);
  if (D > (1 << 30) || rows > (1 << 30)) return fail(B200CP_ERR_UNSUPPORTED, "%s: %d rows of %d values (at most 2^30 of both)", who, rows, D);
  return B200CP_OK;
}
template <typename F>
int by_type(int type, F f) {
  if (type == B200CP_FLOAT32) return f((float*)nullptr);
  if (type == B200CP_BFLOAT16) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}
template <typename T, int VEC>
int lookup(const Lookup& g, cudaStream_t st) {
  const size_t groups = (size_t)g.rows * (g.D / VEC), ctas = (groups + 256 * kEach - 1) / (256 * kEach);
  if (ctas > 0x7fffffffull) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_embedding: %d rows of %d values", g.rows, g.D);
  B200CP_CUDA_OK(launch_kernel(embedding_kernel<T, VEC>, dim3((unsigned)ctas), dim3(256), 0, st, true, g));
  B200CP_LAUNCH_OK("embedding_kernel");
  return B200CP_OK;
}
// Where the parts of a row's columns, a chunk's length and its parts are
struct Cut {
  int lanes, slabs, chunk, chunks;
};
// Chunks are as long as 64 where that leaves four CTAs for each SM, and eight at least: their parts are 8 / chunk of dY's size.  Their length goes by the loads that
// the type and the rows' length allow (each), so that sums have one order wherever the arrays lie; vec: the values of a load that their addresses allow too.
Cut cut_of(int rows, int D, int each, int vec, int sm_count) {
  const auto lanes = [&](int n) {
    int l = 1;
    while (l < 256 && l * n < D) l *= 2;
    return l;
  };
  const auto slabs = [&](int n) { return (int)((D + (long long)lanes(n) * n - 1) / ((long long)lanes(n) * n)); };
  Cut c{lanes(vec), slabs(vec), 64, 1};
  while (c.chunk > 8 && (long long)ceil_div(rows, c.chunk) * slabs(each) * lanes(each) < 4LL * 256 * sm_count) c.chunk /= 2;
  c.chunks = ceil_div(rows, c.chunk);
  return c;
}
size_t keys_bytes(int rows) { return align_up((size_t)rows * 4, 256); }
template <typename T, int VEC>
int sums(Sums g, const Cut& c, cudaStream_t st) {
  const int per = 256 / c.lanes;
  if (c.slabs > 65535 || (g.D + kJoinCols - 1) / kJoinCols > 65535) return fail(B200CP_ERR_UNSUPPORTED, "b200cp_embedding_bwd: rows of %d values", g.D);
  B200CP_CUDA_OK(launch_kernel(embedding_sums_kernel<T, VEC>, dim3((unsigned)ceil_div(c.chunks, per), (unsigned)c.slabs), dim3(256), 0, st, true, g));
  B200CP_LAUNCH_OK("embedding_sums_kernel");
  if (c.chunks < 2) return B200CP_OK;
  const unsigned slabs = (unsigned)ceil_div(g.D, kJoinCols);
  const dim3 threads(std::min(1024, (ceil_div(g.D, 4) + 31) / 32 * 32));
  B200CP_CUDA_OK(launch_kernel(embedding_join_kernel<T>, dim3((unsigned)c.chunks, slabs), threads, 0, st, true, g));
  B200CP_LAUNCH_OK("embedding_join_kernel");
  if (c.chunks <= kGroup) return B200CP_OK;
  B200CP_CUDA_OK(launch_kernel(embedding_join_groups_kernel<T>, dim3((unsigned)ceil_div(c.chunks, kGroup), slabs), threads, 0, st, true, g));
  B200CP_LAUNCH_OK("embedding_join_groups_kernel");
  return B200CP_OK;
}

}  // namespace
}  // namespace b200cp

using namespace b200cp;

extern "C" {

int b200cp_embedding(int rows, int V, int D, int type, int number_type, const void* tokens, const void* W, float scale, void* out, void* stream) {
  const char* who = "b200cp_embedding";
  if (int rc = check_embedding(who, rows, V, D, type, number_type)) return rc;
  if (rows == 0) return B200CP_OK;
  if (!tokens || !W || !out) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  const Lookup g{rows, D, number_type == kInt64, (uint32_t)V, scale, tokens, W, out};
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return rows_of_16<T>(W, D) && rows_of_16<T>(out, D) ? lookup<T, kPerLoad<T>>(g, st) : lookup<T, 1>(g, st);
  });
}

size_t b200cp_embedding_bwd_workspace_bytes(int rows, int D) {
  if (rows < 1 || D < 1) return 0;
  DeviceInfo di;
  if (device_info(&di)) return 0;
  int chunks = 0;   // (those of the shortest chunk that any type gives)
  for (int each : {1, 4, 8}) chunks = std::max(chunks, cut_of(rows, D, each, 1, di.sm_count).chunks);
  return 4 * keys_bytes(rows) + (size_t)chunks * 2 * (size_t)D * sizeof(float);
}

int b200cp_embedding_bwd(int rows, int V, int D, int type, int number_type, const void* tokens, const void* dY, float scale, void* dW, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* who = "b200cp_embedding_bwd";
  if (int rc = check_embedding(who, rows, V, D, type, number_type)) return rc;
  if (!dW) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t bytes = (size_t)V * D * (type == B200CP_FLOAT32 ? 4 : 2);
  if (rows == 0) {
    B200CP_CUDA_OK(cudaMemsetAsync(dW, 0, bytes, st));
    return B200CP_OK;
  }
  if (!tokens || !dY) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  const size_t need = b200cp_embedding_bwd_workspace_bytes(rows, D);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, %zu given", who, need, workspace_bytes);
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  char* ws = static_cast<char*>(workspace);
  const size_t kb = keys_bytes(rows);
  Sort s{};
  s.rows = rows;
  s.wide = number_type == kInt64;
  s.V = (uint32_t)V;
  s.tokens = tokens;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<uint32_t*>(ws + i * kb);
    s.place[i] = reinterpret_cast<uint32_t*>(ws + (2 + i) * kb);
  }
  int bits = 1;   // of the keys 0 .. V
  while ((s.V >> bits) != 0) ++bits;
  s.passes = ceil_div(bits, 10);
  s.bits = ceil_div(bits, s.passes);
  s.cap = ceil_div(rows, kSorters);
  const uintptr_t begin = reinterpret_cast<uintptr_t>(dW), end = begin + bytes, from = std::min(end, (begin + 15) & ~uintptr_t(15)),
                  to = std::max(from, end & ~uintptr_t(15));
  s.zeros = reinterpret_cast<uint4*>(from);
  s.groups = (to - from) / 16;
  s.head = static_cast<unsigned char*>(dW);
  s.before = (int)(from - begin);
  s.tail = reinterpret_cast<unsigned char*>(to);
  s.after = (int)(end - to);
  const size_t fillers = std::max<size_t>(1, (s.groups + kSortThreads * kFill - 1) / (kSortThreads * kFill));
  const size_t ctas = kSorters * (1 + (fillers + kSorters - 1) / kSorters);
  if (ctas > 0x7fffffffull) return fail(B200CP_ERR_UNSUPPORTED, "%s: a table of %zu bytes", who, bytes);
  B200CP_CUDA_OK(launch_kernel(embedding_sort_kernel, dim3((unsigned)ctas), dim3(kSortThreads), 0, st, true, s));
  B200CP_LAUNCH_OK("embedding_sort_kernel");
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool vec = rows_of_16<T>(dY, D) && rows_of_16<T>(dW, D);
    const Cut c = cut_of(rows, D, D % kPerLoad<T> ? 1 : kPerLoad<T>, vec ? kPerLoad<T> : 1, di.sm_count);
    const int last = (s.passes - 1) & 1;
    Sums g{rows, D, c.chunk, c.chunks, c.lanes, (uint32_t)V, scale, s.key[last], s.place[last], dY, dW, reinterpret_cast<float*>(ws + 4 * kb)};
    return vec ? sums<T, kPerLoad<T>>(g, c, st) : sums<T, 1>(g, c, st);
  });
}

}  // extern "C"
