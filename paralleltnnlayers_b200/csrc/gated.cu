// Gated feed-forward block: H = act(X Wg) * (X Wu) and its gradients, 16-bit operands, fp32 sums, on the tcgen05 tensor cores.
//
//   G = X Wg, U = X Wu, H = act(G) U;  dG = dH U act'(G), dU = dH act(G);  dX = dG Wg^T + dU Wu^T;  dWg = X^T dG, dWu = X^T dU
//
// One kernel in three forms.  A pair of CTAs (cta_group::2) forms 256 x 256 sums, 128 rows in each CTA's tensor memory, from a ring of 64-deep
// steps that TMA fills; one thread issues the products, the other warps move finished sums out while the next tile's products run.
//   forward   128 columns of G and the same 128 of U are one tile: the first CTA loads the columns of Wg, the second those of Wu, and both
//             halves of a sum lie side by side in tensor memory, so that act(G) U is formed there and neither G nor U need leave the chip.
//   data      dG Wg^T and dU Wu^T are one sum, twice as long.
//   weights   X^T dG and X^T dU are two results of one launch.
// Weights lie as [inputs][outputs] and activations as [rows][features]; tcgen05 takes either order of either operand, so nothing is transposed.
// For the backward the forward keeps G and U in fp32 (8 bytes a value, where the 16-bit tensors that autograd would keep take 6): with 16-bit
// copies dG and dU would carry two roundings more.  They are rounded once, as operands.
// Rows of odd length are copied to rows of a multiple of eight values first (TMA's strides are multiples of 16 bytes).
// Every wait is bounded: one that runs out sets a status word and the CTA leaves through its normal exit.
#include <algorithm>
#include <type_traits>

#include "cluster_util.cuh"
#include "common.cuh"
#include "tc_common.cuh"
#include "tc_pair.cuh"

namespace b200cp {

__device__ int g_gated_status = 0;   // 0 ok; otherwise (code << 16) | (linear block index & 0xffff)

namespace {

using namespace tc;

enum Form { kForward, kData, kWeights };
constexpr int kTile = 256, kStep = 64, kHalf = 128 * kStep * 2, kStage = 2 * kHalf;   // bytes: of an operand's half, of a step
constexpr int kBox = 64 * kStep * 2;              // a box of 64 columns by 64 k
constexpr int kReaders = 8, kThreads = 64 + 32 * kReaders;
constexpr int kPitch = 80, kPatch = 32 * kPitch;   // bytes of a row and of a warp's 32 x 32 block on its way out
constexpr int kKept = 32 * 32 * 4;                 // bytes of a warp's 32 x 32 block of G or U
constexpr int kStages = 6;                         // 192 KB in flight
template <bool KEEP>
struct Ring {
  static constexpr int out = KEEP ? kKept : kPatch;   // a read-out warp's block
  static constexpr size_t smem = (size_t)kStages * kStage + kReaders * out + 1024 + 256;
  static_assert(smem <= 227 * 1024 && out >= kPatch && kPatch % 16 == 0 && (kStages * kStage) % 1024 == 0 && kKept % 1024 == 0, "");
};

struct Gemm {
  int M, N;                      // of a result
  int tiles_m, tiles_n, units;   // units: tiles of all results
  int steps, first;              // of a sum; steps of its first product
  int act;
  void* out[2];
  int vec;                       // values that a store takes: 8, 2 or 1, by how the rows of out are aligned
  float *G, *U;                  // forward: where the sums are kept, or null
  int ldg;                       // of their rows, a multiple of eight
};

__device__ __forceinline__ void tma_load_pair_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
template <typename T>
__host__ __device__ constexpr uint32_t instruction(uint32_t m, uint32_t n, uint32_t a_mn, uint32_t b_mn) {
  constexpr uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (bf << 7) | (bf << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// ---- the activation -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }   // (exp(-x) = inf: 0)
constexpr float kRootHalf = 0.70710678118654752f, kRootPi = 0.79788456080286536f;   // sqrt(1/2), sqrt(2/pi)
// act(g) = g * share; *slope = act'(g)
template <bool SLOPE>
__device__ __forceinline__ float gate_share(int act, float g, float* slope) {
  if (act == B200CP_SILU) {
    const float s = sigmoid(g);
    if (SLOPE) *slope = s * fmaf(g, 1.f - s, 1.f);
    return s;
  }
  if (act == B200CP_GELU) {
    const float s = 0.5f * erfcf(-kRootHalf * g);   // (1 + erf would lose the left tail)
    if (SLOPE) *slope = fmaf(g * (0.5f * kRootPi), __expf(-0.5f * g * g), s);
    return s;
  }
  const float q = kRootPi * fmaf(0.044715f * g, g * g, g), s = sigmoid(2.f * q);   // (1 + tanh q) / 2
  // (s (1 - s) first: it is zero from some |g| on, where the other factors' product would be infinite)
  if (SLOPE) *slope = fmaf(g * (2.f * s * (1.f - s)), fminf(kRootPi * fmaf(3.f * 0.044715f * g, g, 1.f), 3.4028235e38f), s);
  return s;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// A warp's 32 rows of 32 values (a lane has a row) go through shared memory, so that neighbouring lanes store neighbouring columns: stores of a row
// per lane write 32 sectors each, which in rows of odd length (one value per store) took ten times as long as the products.
template <typename T>
__device__ __forceinline__ void put_block(uint8_t* patch, T* out, int vec, int m0, int M, int n, int N, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  // (rows on 16-byte boundaries straight from the registers: 64 bytes of each, 3 % of a large product less)
  uint4* mine = vec == 8 ? reinterpret_cast<uint4*>(out + (size_t)(m0 + lane) * N + n) : reinterpret_cast<uint4*>(patch + lane * kPitch);
  const int pieces = vec == 8 ? (m0 + lane < M ? min(4, (N - n) / 8) : 0) : 4;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < pieces) mine[j] = make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]), pack2<T>(v[8 * j + 4], v[8 * j + 5]),
                         pack2<T>(v[8 * j + 6], v[8 * j + 7]));
  if (vec == 8) return;
  __syncwarp();
  const int rows = min(32, M - m0), cols = min(32, N - n);
  if (vec == 2) {
    const int q = lane & 15;
    if (q * 2 < cols)
#pragma unroll 4
      for (int r = lane >> 4; r < rows; r += 2)
        *reinterpret_cast<uint32_t*>(out + (size_t)(m0 + r) * N + n + q * 2) = *reinterpret_cast<const uint32_t*>(patch + r * kPitch + q * 4);
  } else {
    if (lane < cols)
#pragma unroll 4
      for (int r = 0; r < rows; ++r) out[(size_t)(m0 + r) * N + n + lane] = reinterpret_cast<const T*>(patch + r * kPitch)[lane];
  }
  __syncwarp();
}
// The warp's 32 kept rows of 32 floats as the box of a tensor store (128-byte rows, swizzled: neighbouring lanes on other banks).  G and U are 8
// of the 10 bytes that a value of the forward writes, and what a tile of few inputs waits for.  4096 x 4096 -> 10240, 8192 x 1024 -> 2816 and 2048 x
// 2048 -> 5120, cold and alone: 449, 102 and 78 us; 440, 131 and 84 where the lanes store them, 64 bytes of a row at a time through the patch; 412,
// 92 and 70 where nothing is kept.  One block for both, not two, which leave room for five steps of the ring: 460, 100 and 80 us.
__device__ __forceinline__ void keep_block(uint8_t* block, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) *reinterpret_cast<float4*>(block + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
// A box from shared memory; what lies outside the tensor is not written.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void stores_end_group() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stores_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// 32 columns of the warp's lane quarter
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------------
struct UnitAt {
  int m0, n0, result;
};
// Groups of kGroup tiles along M share the columns: their rows of A stay in L2 while the columns of B pass by once.
constexpr int kGroup = 16;
template <Form FORM>
__device__ __forceinline__ UnitAt unit_at(const Gemm& g, int unit) {
  const int per = g.tiles_m * g.tiles_n, r = unit / per, t = unit - r * per, band = t / (kGroup * g.tiles_n);
  const int m1 = band * kGroup, height = min(kGroup, g.tiles_m - m1), q = t - m1 * g.tiles_n;
  return UnitAt{(m1 + q % height) * kTile, (q / height) * (FORM == kForward ? kTile / 2 : kTile), r};
}

// KEEP (forward): G and U are kept, through mapA1 and mapK.
template <Form FORM, bool KEEP, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gated_kernel(const __grid_constant__ Gemm g, const __grid_constant__ CUtensorMap mapA0, const __grid_constant__ CUtensorMap mapA1,
             const __grid_constant__ CUtensorMap mapB0, const __grid_constant__ CUtensorMap mapB1, const __grid_constant__ CUtensorMap mapK) {
  constexpr int kOut = Ring<KEEP>::out;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = sm + kStages * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(patches + kReaders * kOut);
  uint64_t* full = bars;                 // [kStages] the leader's: the step of both CTAs has landed  (tx bytes)
  uint64_t* empty = full + kStages;      // [kStages] the products that read the step are done         (commit, both CTAs)
  uint64_t* accfull = empty + kStages;   // [2] the sums of a tile are complete                        (commit, both CTAs)
  uint64_t* accfree = accfull + 2;       // [2] the leader's: read out by the warps of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accfree + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accfull[i], 1);
      mbar_init(&accfree[i], 2 * kReaders);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mapA0);
    tma_prefetch_desc(&mapB0);
    if (FORM != kWeights) tma_prefetch_desc(FORM == kData ? &mapA1 : &mapB1);
    if (KEEP) {
      tma_prefetch_desc(&mapA1);
      tma_prefetch_desc(&mapK);
    }
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot, ring = smem_u32(sm);
  const uint32_t fullb = smem_u32(full), emptyb = smem_u32(empty), accfullb = smem_u32(accfull), accfreeb = smem_u32(accfree),
                 abortb = smem_u32(const_cast<int*>(abort_flag));
  grid_dependency_wait();

  if (warp == 0) {
    // ================= TMA: this CTA's rows of A and its half of the columns of B ===========================================
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int unit = pair; unit < g.units && ok; unit += npairs) {
        const UnitAt t = unit_at<FORM>(g, unit);
        for (int k = 0; k < g.steps; ++k, ++it) {
          const int slot = it % kStages;
          if (it >= kStages && !(ok = wait_or_abort(emptyb + slot * 8, ((it / kStages) - 1) & 1, abortb))) break;
          if (rank == 0) mbar_expect_tx(&full[slot], 2 * kStage);
          const uint32_t bar = leader_addr(fullb + slot * 8), a = ring + slot * kStage, b = a + kHalf;
          if (FORM == kForward) {
            const CUtensorMap* w = rank == 0 ? &mapB0 : &mapB1;
            tma_load_pair_2d(a, &mapA0, bar, k * kStep, t.m0 + rank * 128);
            tma_load_pair_2d(b, w, bar, t.n0, k * kStep);
            tma_load_pair_2d(b + kBox, w, bar, t.n0 + 64, k * kStep);
          } else if (FORM == kData) {
            const bool second = k >= g.first;
            const int x = (k - (second ? g.first : 0)) * kStep;
            tma_load_pair_2d(a, second ? &mapA1 : &mapA0, bar, x, t.m0 + rank * 128);
            tma_load_pair_2d(b, second ? &mapB1 : &mapB0, bar, x, t.n0 + rank * 128);
          } else {
            const CUtensorMap* w = t.result ? &mapB1 : &mapB0;
            tma_load_pair_2d(a, &mapA0, bar, t.m0 + rank * 128, k * kStep);
            tma_load_pair_2d(a + kBox, &mapA0, bar, t.m0 + rank * 128 + 64, k * kStep);
            tma_load_pair_2d(b, w, bar, t.n0 + rank * 128, k * kStep);
            tma_load_pair_2d(b + kBox, w, bar, t.n0 + rank * 128 + 64, k * kStep);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ================= products: one thread of the pair ======================================================================
    if (rank == 0 && elect_one()) {
      constexpr bool a_mn = FORM == kWeights, b_mn = FORM != kData;
      constexpr uint32_t idesc = instruction<T>(256, 256, a_mn, b_mn);
      // K-major: rows of 128 bytes, eight rows per swizzle atom (1024 bytes); 16 k = 32 bytes on.
      // MN-major: 64 columns (128 bytes) per k, eight k per atom, the next 64 columns a box on; 16 k = 2048 bytes on.
      const uint64_t da = make_smem_desc(0, a_mn ? kBox : 16, 1024, kSwizzle128B), db = make_smem_desc(0, b_mn ? kBox : 16, 1024, kSwizzle128B);
      constexpr uint64_t sa = (a_mn ? 2048 : 32) >> 4, sb = (b_mn ? 2048 : 32) >> 4;
      int it = 0, done = 0;
      bool ok = true;
      for (int unit = pair; unit < g.units && ok; unit += npairs, ++done) {
        const int buf = done & 1;
        if (done >= 2 && !(ok = wait_or_abort(accfreeb + buf * 8, (done / 2 - 1) & 1, abortb))) break;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + buf * 256;
        for (int k = 0; k < g.steps; ++k, ++it) {
          const int slot = it % kStages;
          if (!(ok = wait_or_abort(fullb + slot * 8, (it / kStages) & 1, abortb))) break;
          tc_fence_after_sync();
          const uint32_t a = ring + slot * kStage;
          const uint64_t ad = da + (a >> 4), bd = db + ((a + kHalf) >> 4);
#pragma unroll
          for (int i = 0; i < kStep / 16; ++i) mma_f16_pair(d, ad + i * sa, bd + i * sb, idesc, k > 0 || i > 0);
          commit_pair(emptyb + slot * 8);
        }
        if (ok) commit_pair(accfullb + buf * 8);
      }
    }
  } else {
    // ================= read-out ===============================================================================================
    const int qd = warp & 3, half = (warp - 2) >> 2;   // the lane quarter that this warp may read, and its half of the columns
    int done = 0;
    for (int unit = pair; unit < g.units; unit += npairs, ++done) {
      const UnitAt t = unit_at<FORM>(g, unit);
      const int buf = done & 1;
      if (!__all_sync(0xffffffffu, wait_or_abort(accfullb + buf * 8, (done / 2) & 1, abortb))) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + ((uint32_t)(qd * 32) << 16) + buf * 256;
      const int m0 = t.m0 + rank * 128 + qd * 32;
      uint8_t* patch = patches + (warp - 2) * kOut;
      T* out = static_cast<T*>(g.out[FORM == kWeights ? t.result : 0]);
      constexpr int cols = FORM == kForward ? 64 : 128;
      if (m0 < g.M)
#pragma unroll 1
        for (int j = half * cols; j < half * cols + cols && t.n0 + j < g.N; j += 32) {
          float a[32];
          tmem_ld32(taddr + j, a);
          if constexpr (FORM == kForward) {
            float u[32];
            tmem_ld32(taddr + 128 + j, u);
            if constexpr (KEEP) {
              // (nobody reads the blocks any more, nor is the patch in them in use)
              if (lane == 0) stores_wait_read();
              __syncwarp();
              keep_block(patch, a);
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&mapA1, patch, t.n0 + j, m0);
                stores_end_group();
                stores_wait_read();
              }
              __syncwarp();
              keep_block(patch, u);
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&mapK, patch, t.n0 + j, m0);
                stores_end_group();
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) a[i] = a[i] * gate_share<false>(g.act, a[i], nullptr) * u[i];
          }
          if (KEEP && g.vec != 8) {   // the patch lies in a block that is on its way out
            if (lane == 0) stores_wait_read();
            __syncwarp();
          }
          put_block(patch, out, g.vec, m0, g.M, t.n0 + j, g.N, a);
        }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_cluster(leader_addr(accfreeb + buf * 8));
    }
    if (KEEP && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // (written, not only read)
  }
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    atomicCAS(&g_gated_status, 0, (1 << 16) | (blockIdx.x & 0xffff));
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

// ---- few rows -------------------------------------------------------------------------------------------------------------------
// G^T = Wg^T X^T and U^T: the weights are the 128 rows of the products and X's rows their NT columns, so that nothing of a product is wasted on rows that
// are not there, and every weight is read once.  Bound by HBM (the weights).  An SM holds one CTA that uses tensor memory and reads some
// 54 bytes per nanosecond, so what counts is how many SMs have one: a CTA has W x 128 columns, a cluster of up to eight shares the sum over
// the inputs (each adds the parts of its share of the columns, in their order), and W and the cluster are those that give the most CTAs
// (48 rows 4096 -> 10240: 80 CTAs of 128 columns 39 us, 40 clusters of three with 256 columns 34; 64 rows 8192 -> 8192 47, 5.7 TB/s).
template <int NT, int W>
struct Few {
  static constexpr int weights = 128 * kStep * 2, stage = 2 * W * weights + NT * kStep * 2;   // bytes: of a tile of a weight, of a step
  static constexpr int stages = W == 2 ? 3 : NT <= 32 ? 6 : NT == 64 ? 5 : 4;                 // 192 to 216 KB
  static constexpr int tmem = 2 * W * NT < 32 ? 32 : 2 * W * NT, cols = 128 * W;
  static constexpr int parts = 2 * NT * cols * 4;                                             // sums, in place of the ring
  static constexpr size_t smem = (size_t)stages * stage + 1024 + 128;
  static_assert(parts <= stages * stage && smem <= 227 * 1024 && (tmem & (tmem - 1)) == 0, "");
};
struct FewArgs {
  int M, N, steps, act;   // steps: of K, all CTAs of a cluster together
  void* H;
  int vec;                // four columns of H start on 8-byte boundaries
  float *G, *U;
  int ldg;
};
constexpr int kFewThreads = 192;
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
      "r"(x), "r"(y)
      : "memory");
}
template <int NT, int W, typename T>
__global__ void __launch_bounds__(kFewThreads) gated_few_kernel(const __grid_constant__ FewArgs g, const __grid_constant__ CUtensorMap mapX,
                                                                const __grid_constant__ CUtensorMap mapG, const __grid_constant__ CUtensorMap mapU) {
  using F = Few<NT, W>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + F::stages * F::stage);
  uint64_t *empty = full + F::stages, *ready = empty + F::stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t csize;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
  const int rank = (int)cluster_rank(), f0 = (int)(blockIdx.x / csize) * F::cols;
  if (tid == 0) {
    for (int i = 0; i < F::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(ready, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mapX);
    tma_prefetch_desc(&mapG);
    tma_prefetch_desc(&mapU);
  }
  if (warp == 1) tmem_alloc(tmem_slot, F::tmem);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot, ring = smem_u32(sm), abortb = smem_u32(const_cast<int*>(abort_flag));
  grid_dependency_wait();
  // this CTA's steps of K
  const int per = (g.steps + (int)csize - 1) / (int)csize, k0 = min(g.steps, rank * per), n = min(g.steps, k0 + per) - k0;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < n; ++i) {
        const int slot = i % F::stages, k = (k0 + i) * kStep;
        if (i >= F::stages && !wait_or_abort(smem_u32(&empty[slot]), (i / F::stages - 1) & 1, abortb)) break;
        mbar_expect_tx(&full[slot], F::stage);
        const uint32_t bar = smem_u32(&full[slot]), a = ring + slot * F::stage;
#pragma unroll
        for (int w = 0; w < 2 * W; ++w) {
          tma_load_2d(a + w * kBox, &mapG, bar, f0 + w * 64, k);
          tma_load_2d(a + W * F::weights + w * kBox, &mapU, bar, f0 + w * 64, k);
        }
        tma_load_2d(a + 2 * W * F::weights, &mapX, bar, k, 0);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = instruction<T>(128, NT, 1, 0);
      const uint64_t da = make_smem_desc(0, kBox, 1024, kSwizzle128B), db = make_smem_desc(0, 16, 1024, kSwizzle128B);
      bool ok = true;
      for (int i = 0; i < n && ok; ++i) {
        const int slot = i % F::stages;
        if (!(ok = wait_or_abort(smem_u32(&full[slot]), (i / F::stages) & 1, abortb))) break;
        tc_fence_after_sync();
        const uint32_t a = ring + slot * F::stage;
        // (a shared address of a CTA other than the cluster's first has bits above those of the descriptor's field)
        const auto at = [](uint32_t p) { return (uint64_t)((p >> 4) & 0x3fff); };
        const uint64_t b = db + at(a + 2 * W * F::weights);
#pragma unroll
        for (int w = 0; w < 2 * W; ++w) {   // tiles of Wg, then of Wu
          const uint64_t p = da + at(a + w * F::weights);
#pragma unroll
          for (int j = 0; j < kStep / 16; ++j) mma_f16_ss(tmem_base + w * NT, p + j * (2048 >> 4), b + j * (32 >> 4), idesc, i > 0 || j > 0);
        }
        mma_commit(&empty[slot]);
      }
      if (ok) mma_commit(ready);
    }
  } else {
    // sums -> shared memory, [G, U][row of X][column of the weights]: the ring is free once the last product is done
    const bool ok = __all_sync(0xffffffffu, wait_or_abort(smem_u32(ready), 0, abortb));
    tc_fence_after_sync();
    if (ok) {
      const int qd = warp & 3;
      float* part = reinterpret_cast<float*>(sm) + qd * 32 + lane;
      const uint32_t taddr = tmem_base + ((uint32_t)(qd * 32) << 16);
#pragma unroll 1
      for (int j = 0; j < 2 * W * NT; j += 16) {
        const int w = j / NT, m = j % NT;   // the tile, and the row of X
        float* to = part + ((w / W) * NT + m) * F::cols + (w % W) * 128;
        float v[16];
        if (n > 0) tmem_ld16(taddr + j, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i * F::cols] = n > 0 ? v[i] : 0.f;
      }
    }
    tc_fence_before_sync();
  }
  __syncthreads();
  cluster_sync();
  // The cluster's parts of a share of the columns, four at a time (a read of another CTA's memory takes half a microsecond).
  const int quads = (32 * W + (int)csize - 1) / (int)csize, q0 = rank * quads, rows = min(NT, g.M);
#pragma unroll 2
  for (int i = tid; i < quads * rows; i += kFewThreads) {
    const int m = i / quads, q = q0 + (i - m * quads), f = f0 + 4 * q;
    if (q >= 32 * W || f >= g.N) continue;
    float4 v[2][8];
    const uint32_t at = ring + (m * F::cols + 4 * q) * 4;
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
      if (p < csize) {
        uint32_t from;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at), "r"(p));
#pragma unroll
        for (int k = 0; k < 2; ++k)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[k][p].x), "=f"(v[k][p].y), "=f"(v[k][p].z), "=f"(v[k][p].w)
                       : "r"(from + k * NT * F::cols * 4)
                       : "memory");
      }
    float a[4] = {}, u[4] = {};
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
      if (p < csize) {
        a[0] += v[0][p].x; a[1] += v[0][p].y; a[2] += v[0][p].z; a[3] += v[0][p].w;
        u[0] += v[1][p].x; u[1] += v[1][p].y; u[2] += v[1][p].z; u[3] += v[1][p].w;
      }
    if (g.G) {   // (columns past the end are those of the row's padding)
      *reinterpret_cast<float4*>(g.G + (size_t)m * g.ldg + f) = make_float4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<float4*>(g.U + (size_t)m * g.ldg + f) = make_float4(u[0], u[1], u[2], u[3]);
    }
    T* h = static_cast<T*>(g.H) + (size_t)m * g.N + f;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = a[k] * gate_share<false>(g.act, a[k], nullptr) * u[k];
    if (g.vec) {
      *reinterpret_cast<uint2*>(h) = make_uint2(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (f + k < g.N) h[k] = (T)a[k];
    }
  }
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    atomicCAS(&g_gated_status, 0, (2 << 16) | (blockIdx.x & 0xffff));
    const long long t0 = clock64();   // copies in flight land before the shared memory is given back
    while (clock64() - t0 < 40000000ll) {
    }
  }
  cluster_sync();   // nobody reads this CTA's parts any more
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, F::tmem);
  }
}

// ---- elementwise -----------------------------------------------------------------------------------------------------------------
// dG = dH U act'(G), dU = dH act(G): dH has rows of N values, the others of ld, eight per thread (the padding is written, and read by nothing).  Bound by HBM: 14 bytes a value.
template <typename T>
__global__ void __launch_bounds__(256) slopes_kernel(int M, int N, int ld, int act, int vec, const float* G, const float* U, const T* dH, T* dG, T* dU) {
  const int groups = (N + 7) / 8;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)M * groups) return;
  const size_t m = i / groups;
  const int n = (int)(i - m * groups) * 8, left = min(8, N - n);
  const size_t src = m * N + n, dst = m * ld + n;
  float a[8], u[8], d[8];
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    *reinterpret_cast<float4*>(a + j) = *reinterpret_cast<const float4*>(G + dst + j);
    *reinterpret_cast<float4*>(u + j) = *reinterpret_cast<const float4*>(U + dst + j);
  }
  if (vec) {
    alignas(16) T h[8];
    *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(dH + src);
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = (float)h[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = j < left ? (float)dH[src + j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float slope;
    const float share = gate_share<true>(act, a[j], &slope);
    const float up = d[j] * a[j] * share;
    a[j] = d[j] * u[j] * slope;
    u[j] = up;
  }
  *reinterpret_cast<uint4*>(dG + dst) = make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(a[4], a[5]), pack2<T>(a[6], a[7]));
  *reinterpret_cast<uint4*>(dU + dst) = make_uint4(pack2<T>(u[0], u[1]), pack2<T>(u[2], u[3]), pack2<T>(u[4], u[5]), pack2<T>(u[6], u[7]));
}

// Rows of `cols` 16-bit values to rows of ld (a multiple of eight), up to three matrices in one launch.
struct PadJob {
  const uint16_t* src;
  uint16_t* dst;
  int rows, cols, ld;
  unsigned first;   // CTA
};
struct PadJobs {
  PadJob job[3];
  int count;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadJobs p) {
  int k = 0;
  while (k + 1 < p.count && blockIdx.x >= p.job[k + 1].first) ++k;
  const PadJob& q = p.job[k];
  const int groups = q.ld / 8;
  const size_t i = (size_t)(blockIdx.x - q.first) * 256 + threadIdx.x;
  if (i >= (size_t)q.rows * groups) return;
  const size_t r = i / groups;
  const int c = (int)(i - r * groups) * 8;
  const uint16_t* s = q.src + r * q.cols + c;
  alignas(16) uint16_t v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < q.cols ? s[j] : (uint16_t)0;
  *reinterpret_cast<uint4*>(q.dst + r * q.ld + c) = *reinterpret_cast<const uint4*>(v);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int ld8(int n) { return (n + 7) / 8 * 8; }
size_t plane(size_t rows, int cols) { return align_up(rows * ld8(cols) * 2, 256); }
bool odd(int cols) { return cols % 8 != 0; }

struct Matrix {   // as the kernel reads it
  const void* p;
  int rows, cols, ld;
};
template <typename T>
int encode(CUtensorMap* map, const Matrix& m, unsigned box_rows) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B200CP_ERR_NO_DEVICE, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dim[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows}, stride[1] = {(cuuint64_t)m.ld * 2};
  const cuuint32_t box[2] = {64, box_rows}, estr[2] = {1, 1};
  const CUresult cr = enc(map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                          const_cast<void*>(m.p), dim, stride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (cr != CUDA_SUCCESS) return fail(B200CP_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)cr);
  return B200CP_OK;
}
// Copies the matrices whose rows are of odd length to the workspace, which is moved on.
int pad(Matrix** ms, int count, char*& ws, cudaStream_t st) {
  PadJobs jobs{};
  unsigned ctas = 0;
  for (int i = 0; i < count; ++i) {
    Matrix& m = *ms[i];
    m.ld = ld8(m.cols);
    if (!odd(m.cols)) continue;
    const size_t n = ((size_t)m.rows * (m.ld / 8) + 255) / 256;
    jobs.job[jobs.count++] = PadJob{static_cast<const uint16_t*>(m.p), reinterpret_cast<uint16_t*>(ws), m.rows, m.cols, m.ld, ctas};
    ctas += (unsigned)n;
    m.p = ws;
    ws += plane(m.rows, m.cols);
  }
  if (!ctas) return B200CP_OK;
  pad_rows_kernel<<<ctas, 256, 0, st>>>(jobs);
  B200CP_LAUNCH_OK("pad_rows_kernel");
  return B200CP_OK;
}
size_t pad_bytes(int rows, int I, int F) { return (odd(I) ? plane(rows, I) : 0) + (odd(F) ? 2 * plane(I, F) : 0); }
bool rows16(const void* p, size_t row_bytes) { return !(reinterpret_cast<uintptr_t>(p) & 15) && row_bytes % 16 == 0; }

// rows of floats for boxes of 32 x 32
int encode_kept(CUtensorMap* map, const float* p, int rows, int ld) {
  PFN_encodeTiled enc = get_encode_tiled();
  const cuuint64_t dim[2] = {(cuuint64_t)ld, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)ld * 4};
  const cuuint32_t box[2] = {32, 32}, estr[2] = {1, 1};
  const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(p), dim, stride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (cr != CUDA_SUCCESS) return fail(B200CP_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)cr);
  return B200CP_OK;
}
template <Form FORM, bool KEEP, typename T>
int launch(Gemm g, int results, const Matrix& a0, const Matrix& a1, const Matrix& b0, const Matrix& b1, cudaStream_t st) {
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  CUtensorMap ma0, ma1, mb0, mb1, mk;
  constexpr unsigned ra = FORM == kWeights ? kStep : 128, rb = FORM == kData ? 128 : kStep;
  if (int rc = encode<T>(&ma0, a0, ra)) return rc;
  g.ldg = ld8(g.N);
  if constexpr (KEEP) {
    if (int rc = encode_kept(&ma1, g.G, g.M, g.ldg)) return rc;
    if (int rc = encode_kept(&mk, g.U, g.M, g.ldg)) return rc;
  } else {
    if (int rc = encode<T>(&ma1, a1, ra)) return rc;
    mk = ma1;
  }
  if (int rc = encode<T>(&mb0, b0, rb)) return rc;
  if (int rc = encode<T>(&mb1, b1, rb)) return rc;
  g.tiles_m = ceil_div(g.M, kTile);
  g.tiles_n = ceil_div(g.N, FORM == kForward ? kTile / 2 : kTile);
  const long units = (long)g.tiles_m * g.tiles_n * results;
  if (units > 0x3fffffff) return fail(B200CP_ERR_UNSUPPORTED, "gated feed-forward block: %d x %d is too large", g.M, g.N);
  g.units = (int)units;
  const uintptr_t at = reinterpret_cast<uintptr_t>(g.out[0]) | reinterpret_cast<uintptr_t>(g.out[results - 1]) | (uintptr_t)g.N * 2;
  g.vec = at % 16 == 0 ? 8 : at % 4 == 0 ? 2 : 1;
  constexpr size_t kSmem = Ring<KEEP>::smem;
  const auto kern = gated_kernel<FORM, KEEP, T>;
  static std::atomic<int> set[64];
  B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), set, (int)kSmem));
  const int pairs = std::min(g.units, di.sm_count / 2);
  B200CP_CUDA_OK(launch_kernel(kern, dim3(2 * pairs), dim3(kThreads), kSmem, st, true, g, ma0, ma1, mb0, mb1, mk));
  B200CP_LAUNCH_OK("gated_kernel");
  return B200CP_OK;
}

constexpr int kFewRows = 128;   // batches of up to this many rows
// CTAs that a shape of the kernel gives: the largest cluster (and two steps for each of its CTAs) of which the device holds all tiles at once
template <int NT, int W, typename T>
int few_ctas(const FewArgs& g, int* cluster, int* ctas) {
  using F = Few<NT, W>;
  const auto kern = gated_few_kernel<NT, W, T>;
  static std::atomic<int> set[64];
  static ClusterCounts counts;
  int dev = 0;
  B200CP_CUDA_OK(cudaGetDevice(&dev));
  B200CP_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), set, (int)F::smem));
  const int tiles = ceil_div(g.N, F::cols);
  *cluster = 1;
  for (int q = 2; q <= 8 && g.steps >= 2 * q; ++q) {
    int n = 0;
    B200CP_CUDA_OK(resident_clusters(kern, kFewThreads, F::smem, dev, q, counts, &n));
    if (tiles <= n) *cluster = q;
  }
  *ctas = tiles * *cluster;
  return B200CP_OK;
}
template <int NT, int W, typename T>
int launch_few(const FewArgs& g, int cluster, const CUtensorMap& x, const CUtensorMap& wg, const CUtensorMap& wu, cudaStream_t st) {
  using F = Few<NT, W>;
  B200CP_CUDA_OK(launch_clusters(gated_few_kernel<NT, W, T>, ceil_div(g.N, F::cols), cluster, kFewThreads, F::smem, st, g, x, wg, wu));
  B200CP_LAUNCH_OK("gated_few_kernel");
  return B200CP_OK;
}
template <int NT, typename T>
int run_few(const FewArgs& g, const Matrix& x, const Matrix& wg, const Matrix& wu, cudaStream_t st) {
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  CUtensorMap mx, mg, mu;
  if (int rc = encode<T>(&mx, x, NT)) return rc;
  if (int rc = encode<T>(&mg, wg, kStep)) return rc;
  if (int rc = encode<T>(&mu, wu, kStep)) return rc;
  int c1 = 1, n1 = 0;
  if (int rc = few_ctas<NT, 1, T>(g, &c1, &n1)) return rc;
  if constexpr (NT <= 64) {
    int c2 = 1, n2 = 0;
    if (n1 < di.sm_count) {
      if (int rc = few_ctas<NT, 2, T>(g, &c2, &n2)) return rc;
      if (n2 > n1) return launch_few<NT, 2, T>(g, c2, mx, mg, mu, st);
    }
  }
  return launch_few<NT, 1, T>(g, c1, mx, mg, mu, st);
}

template <typename T>
int forward(int rows, int I, int F, int act, const void* X, const void* Wg, const void* Wu, void* H, float* G, float* U, char* ws, cudaStream_t st) {
  Matrix x{X, rows, I, 0}, g{Wg, I, F, 0}, u{Wu, I, F, 0}, *ms[3] = {&x, &g, &u};
  if (int rc = pad(ms, 3, ws, st)) return rc;
  if (rows <= kFewRows) {
    const FewArgs f{rows, F, ceil_div(I, kStep), act, H, F % 4 == 0 && reinterpret_cast<uintptr_t>(H) % 8 == 0, G, U, ld8(F)};
    if (rows <= 16) return run_few<16, T>(f, x, g, u, st);
    if (rows <= 32) return run_few<32, T>(f, x, g, u, st);
    if (rows <= 64) return run_few<64, T>(f, x, g, u, st);
    return run_few<128, T>(f, x, g, u, st);
  }
  Gemm p{};
  p.M = rows; p.N = F; p.steps = p.first = ceil_div(I, kStep); p.act = act;
  p.out[0] = p.out[1] = H; p.G = G; p.U = U;
  return G ? launch<kForward, true, T>(p, 1, x, x, g, u, st) : launch<kForward, false, T>(p, 1, x, x, g, u, st);
}

template <typename T>
int backward(int rows, int I, int F, int act, const void* X, const void* Wg, const void* Wu, const float* G, const float* U, const void* dH, void* dX,
             void* dWg, void* dWu, char* ws, cudaStream_t st) {
  const int ld = ld8(F);
  T *dG = reinterpret_cast<T*>(ws), *dU = reinterpret_cast<T*>(ws + plane(rows, F));
  ws += 2 * plane(rows, F);
  Matrix x{X, rows, I, 0}, g{Wg, I, F, 0}, u{Wu, I, F, 0}, *ms[3];
  int count = 0;
  if (dWg) ms[count++] = &x;
  if (dX) {
    ms[count++] = &g;
    ms[count++] = &u;
  }
  if (int rc = pad(ms, count, ws, st)) return rc;
  const size_t n = ((size_t)rows * (ld / 8) + 255) / 256;
  if (n > 0x7fffffffull) return fail(B200CP_ERR_UNSUPPORTED, "gated feed-forward block: %d x %d is too large", rows, F);
  const int vec = rows16(dH, (size_t)F * 2);
  slopes_kernel<T><<<(unsigned)n, 256, 0, st>>>(rows, F, ld, act, vec, G, U, static_cast<const T*>(dH), dG, dU);
  B200CP_LAUNCH_OK("slopes_kernel");
  const Matrix a{dG, rows, F, ld}, b{dU, rows, F, ld};
  Gemm p{};
  if (dX) {
    p.M = rows; p.N = I; p.first = ceil_div(F, kStep); p.steps = 2 * p.first;
    p.out[0] = p.out[1] = dX;
    if (int rc = launch<kData, false, T>(p, 1, a, b, g, u, st)) return rc;
  }
  if (dWg) {
    p.M = I; p.N = F; p.steps = p.first = ceil_div(rows, kStep);
    p.out[0] = dWg; p.out[1] = dWu;
    if (int rc = launch<kWeights, false, T>(p, 2, x, x, a, b, st)) return rc;
  }
  return B200CP_OK;
}

int check_gated(const char* who, int rows, int I, int F, int type, int act) {
  if (rows < 0 || I < 1 || F < 1 || act < B200CP_SILU || act > B200CP_GELU_TANH)
    return fail(B200CP_ERR_INVALID_ARG, "%s: rows=%d I=%d F=%d activation=%d", who, rows, I, F, act);
  if (type != B200CP_BFLOAT16 && type != B200CP_FLOAT16) return fail(B200CP_ERR_UNSUPPORTED, "%s: type %d (16-bit types only)", who, type);
  if (rows > (1 << 28) || I > (1 << 28) || F > (1 << 28)) return fail(B200CP_ERR_UNSUPPORTED, "%s: sizes above 2^28", who);
  return B200CP_OK;
}

}  // namespace

int gated_device_status(int* out) {
  int v = 0, zero = 0;
  B200CP_CUDA_OK(cudaMemcpyFromSymbol(&v, g_gated_status, sizeof(int)));
  if (v) B200CP_CUDA_OK(cudaMemcpyToSymbol(g_gated_status, &zero, sizeof(int)));
  *out = v;
  return B200CP_OK;
}

}  // namespace b200cp

using namespace b200cp;

extern "C" {

size_t b200cp_dense_gated_workspace_bytes(int rows, int I, int F, int type) {
  if (check_gated("b200cp_dense_gated_workspace_bytes", rows, I, F, type, 0)) return 0;
  return pad_bytes(rows, I, F);
}

int b200cp_dense_gated(int rows, int I, int F, int type, int activation, const void* X, const void* Wg, const void* Wu, void* H, float* G,
                       float* U, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "b200cp_dense_gated";
  if (int rc = check_gated(who, rows, I, F, type, activation)) return rc;
  if (rows == 0) return B200CP_OK;
  if (!X || !Wg || !Wu || !H || !G != !U) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  for (const void* p : {X, Wg, Wu, (const void*)G, (const void*)U})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(B200CP_ERR_INVALID_ARG, "%s: X, Wg, Wu, G and U have to start on 16-byte boundaries", who);
  const size_t need = b200cp_dense_gated_workspace_bytes(rows, I, F, type);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, %zu given", who, need, workspace_bytes);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  return type == B200CP_BFLOAT16 ? forward<__nv_bfloat16>(rows, I, F, activation, X, Wg, Wu, H, G, U, ws, st)
                                 : forward<__half>(rows, I, F, activation, X, Wg, Wu, H, G, U, ws, st);
}

size_t b200cp_dense_gated_bwd_workspace_bytes(int rows, int I, int F, int type) {
  if (check_gated("b200cp_dense_gated_bwd_workspace_bytes", rows, I, F, type, 0)) return 0;
  return 2 * plane(rows, F) + pad_bytes(rows, I, F);
}

int b200cp_dense_gated_bwd(int rows, int I, int F, int type, int activation, const void* X, const void* Wg, const void* Wu, const float* G,
                           const float* U, const void* dH, void* dX, void* dWg, void* dWu, void* workspace, size_t workspace_bytes,
                           void* stream) {
  const char* who = "b200cp_dense_gated_bwd";
  if (int rc = check_gated(who, rows, I, F, type, activation)) return rc;
  if (!dWg != !dWu) return fail(B200CP_ERR_INVALID_ARG, "%s: one of dWg and dWu is null", who);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (void* p : {dWg, dWu})
      if (p) B200CP_CUDA_OK(cudaMemsetAsync(p, 0, (size_t)I * F * 2, st));
    return B200CP_OK;
  }
  if (!G || !U || !dH || (dWg && !X) || (dX && (!Wg || !Wu))) return fail(B200CP_ERR_INVALID_ARG, "%s: null pointer", who);
  for (const void* p : {X, Wg, Wu, (const void*)G, (const void*)U})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(B200CP_ERR_INVALID_ARG, "%s: X, Wg, Wu, G and U have to start on 16-byte boundaries", who);
  const size_t need = b200cp_dense_gated_bwd_workspace_bytes(rows, I, F, type);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(B200CP_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, %zu given", who, need, workspace_bytes);
  char* ws = static_cast<char*>(workspace);
  return type == B200CP_BFLOAT16 ? backward<__nv_bfloat16>(rows, I, F, activation, X, Wg, Wu, G, U, dH, dX, dWg, dWu, ws, st)
                                 : backward<__half>(rows, I, F, activation, X, Wg, Wu, G, U, dH, dX, dWg, dWu, ws, st);
}

}  // extern "C"
