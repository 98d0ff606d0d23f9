// The experts' products on rows sorted by expert, and their gradients, on tcgen05 / TMEM.
//
//   h = x W1[e]^T,   a = silu(h_gate) * h_up  or  gelu(h),   y = a W2[e]^T             (rows of expert e: offsets[e] .. offsets[e+1])
//   da = dy W2[e],   dh = da * (derivative of the activation at h),   dx = dh W1[e]
//   dW2[e] = dy_e^T a_e,   dW1[e] = dh_e^T x_e                                          (sums over the expert's rows)
//
// One kernel template computes all of them on CTA pairs (tcgen05.mma.cta_group::2): the result's features (its contiguous
// dimension) are the M side, 256 of them, 128 in each CTA's TMEM lanes; its rows are the N side, up to 256, in sixteens.
// An expert's rows are split evenly over the fewest tiles, so ragged experts cost what they hold: with rows on the M side
// (128 at a time) 128 experts of 256 rows on average took 1.25 times the instructions, on pairs (256) 1.5 times, and that
// was the bound.  Each CTA loads its 128 features and half of the rows, 32 KB per K step of 64, two thirds of what a CTA on
// its own needs; more would pass what L2 delivers to an SM.
//   rows x features (h, y, da, dx): the rows are K-major as stored; the weights K-major as stored for the forward products
//     and MN-major for the gradients (W is then read along its other dimension, nothing is transposed in memory).  For the
//     gated activation a CTA's features are 64 gate and the 64 up rows that go with them.
//   weight gradients: both operands MN-major, the result's rows on the M side (then a lane holds a row of the result and
//     packs it before it passes through shared memory), K = the expert's rows, of any number.  The last K step takes only as many
//     instructions as it has rows in sixteens; rows behind the expert's last one in it belong to the next expert and are
//     zeroed in shared memory first (in both operands: 0 * inf would not vanish), by a warp that runs ahead of the MMAs.
// Persistent CTAs, one per SM: warp 0 loads (TMA), warp 1 issues the MMAs (the pair's first CTA) and owns TMEM, warp 2 clears
// foreign rows, warps 4..11 are the epilogue (two per quadrant of TMEM lanes, each every other 32 columns); two accumulators
// of 256 columns let it run under the next tile's MMAs.  A lane holds a feature, so results are turned in shared memory
// and leave as contiguous pieces of a row.  Every wait is bounded.
//
// Measured (B200, 32768 rows of 128 experts, H 2048, I 768, SwiGLU): h and a 222 us, y 116, dh 150, dx 200, dW2 128, dW1 229;
// HBM alone, with reads at 6.5 TB/s and writes at about 4.2, would take 204, 102, 138, 171, 124, 228.  With thousands of rows
// per expert: 1.2 to 1.5 PFLOP/s (cuBLAS on one large product: 1.65).
//
// Roundings: products accumulate in fp32; h is kept as it is, in fp32, for the backward pass (in bf16 its rounding made the
// gradients of rows and w1 a quarter less exact, 3.0e-3 of their norm against 2.4e-3; it is twice the bytes, 0.2 GB written
// and read again for 32768 rows of 1536); a and dh are rounded to bf16 because the next product's operands are bf16; y, dx, dW once at the end.
#pragma once
#include "gemm.cuh"
#include "op_common.cuh"

namespace zepp {

enum FfnMode : int {
  FFN_UP_SWIGLU = 0,      // rows [n, H], W1 [G, 2I, H]  -> a [n, I] (+ h [n, 2I])
  FFN_UP_GELU = 1,        // rows [n, H], W1 [G, I, H]   -> a [n, I] (+ h [n, I])
  FFN_DOWN = 2,           // a [n, I], W2 [G, H, I]      -> y [n, H]
  FFN_DACT_SWIGLU = 3,    // dy [n, H], W2 [G, H, I], h  -> dh [n, 2I]
  FFN_DACT_GELU = 4,      // dy [n, H], W2 [G, H, I], h  -> dh [n, I]
  FFN_DROWS = 5,          // dh [n, f1], W1 [G, f1, H]   -> dx [n, H]
  FFN_DWEIGHT = 6         // p [n, M], q [n, N]          -> [G, M, N] = p_e^T q_e
};

constexpr int kFfnMaxGroups = 1024;
constexpr int kFfnThreads = 384;
constexpr int kFfnEpiWarp0 = 4;
constexpr int kFfnEpiWarps = 8;
constexpr int kFfnRows = 256;                           // rows of a tile at most
constexpr int kFfnHalfBytes = 128 * 128;                // 128 rows x 64 bf16, or two blocks of 64 K rows x 64 elements
constexpr int kFfnBlockBytes = 64 * 128;                // an MN-major operand block: 64 K rows x 64 elements
constexpr int kFfnStageBytes = 2 * kFfnHalfBytes;       // this CTA's features, its half of the rows
constexpr int kFfnMaxStages = 6;
constexpr int kFfnStagingBytes = 4096;                  // per epilogue warp: 32 rows x 32 fp32 features
constexpr unsigned long long kFfnDrainNs = 2000000000ull;       // limit of each wait for copies and MMAs after a role gave up

struct FfnArgs {
  const int* offsets;        // [G + 1]
  int G;
  long long n;               // rows of the buffers
  int K;                     // length of the contraction (not used by FFN_DWEIGHT)
  int M;                     // FFN_DWEIGHT: rows of a group's result
  int N;                     // features of the result (FFN_UP_SWIGLU, FFN_DACT_SWIGLU: of each half)
  int feat;                  // features per tile: 128 (FFN_UP_SWIGLU) or 256
  int stages;
  __nv_bfloat16* out;        // a, y, dh, dx or dW
  float* h;                  // FFN_UP_*: written if not null; FFN_DACT_*: read
  unsigned long long* status;
  unsigned long long limit_ns;
};

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* tmap, uint32_t leader_bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Arrival on a barrier of either CTA of the pair, at the scope of both (a CTA-scoped one does not order anything for a thread
// of the other CTA).  Relaxed: what it announces is ordered by a fence of its own before it, TMEM reads by tcgen05.fence,
// cleared rows by the two below.  With release semantics the arrival would also wait for the thread's stores to global
// memory: 3600 cycles for the epilogue of a weight gradient's tile, 3300 for clearing rows.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_addr) : "memory");
}
// The other side, once a bounded wait for this phase has returned: the same phase seen at the pair's scope.
__device__ __forceinline__ void mbar_seen_pair(uint64_t* bar, uint32_t parity) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.relaxed.cluster.shared::cta.b64 p, [%0], %1;\n\t}"
      ::"r"(smem_u32(bar)), "r"(parity)
      : "memory");
}
// Stores to this CTA's shared memory, made before the arrival that follows, for the thread that waits for it in either CTA ...
__device__ __forceinline__ void fence_release_pair_shared() {
  asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
}
// ... and that thread's side of it
__device__ __forceinline__ void fence_acquire_pair_shared() {
  asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
}
// this thread's stores to shared memory before what the copies and MMAs do there
__device__ __forceinline__ void fence_proxy_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ uint32_t ld_shared_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_shared_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
// One lane of a converged warp, always the same.  The copies and MMAs take their operands from uniform registers: issued
// under `lane == 0` they cost 570 cycles per K step on the issuing thread (380 of them without a single MMA), more than
// the 4 MMAs themselves; a branch on elect.sync is known to be taken by one lane, and the operands stay uniform.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// Descriptor of an MN-major bf16 operand: blocks of 64 elements x 64 K rows (128-byte rows, 128-byte swizzle, 8 KB), one
// behind the other along the M / N dimension.  The stride between blocks is the leading offset, between groups of eight K
// rows the stride offset; 16 K rows further is 2048 bytes.
__device__ __forceinline__ uint64_t make_mnmajor_sw128_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(kFfnBlockBytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ float ffn_sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// A warp's 32 features (lanes) x 32 rows (registers) turned in its staging: fp32 [row][feature], the 16-byte units of a row
// XOR-swizzled by the row so that neither side's accesses conflict.
__device__ __forceinline__ void ffn_turn_in(float* stg, const uint32_t (&v)[32], int lane) {
#pragma unroll
  for (int j = 0; j < 32; ++j) stg[j * 32 + (((lane >> 2) ^ (j & 7)) << 2) + (lane & 3)] = __uint_as_float(v[j]);
}
// eight neighbouring features of row j (units 2 * part and 2 * part + 1)
__device__ __forceinline__ void ffn_turn_out(const float* stg, int j, int part, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 w = *reinterpret_cast<const float4*>(stg + j * 32 + (((2 * part + i) ^ (j & 7)) << 2));
    x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
  }
}
__device__ __forceinline__ void ffn_store8(__nv_bfloat16* out, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
    w[e] = *reinterpret_cast<const uint32_t*>(&p);
  }
  *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void ffn_store8(float* out, const float (&x)[8]) {
  reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// A warp's 32 rows (lanes) x 64 features (registers) as bf16 through its staging: 128 bytes a row, its 16-byte units
// XOR-swizzled by the row, then eight lanes write a row's whole line.
__device__ __forceinline__ void ffn_put(uint4* stg, const uint32_t (&v)[32], const uint32_t (&w)[32], void* base, long long ld,
                                        int rows, int bytes, int lane) {
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    uint32_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = (u & 3) * 8 + 2 * e;
      const __nv_bfloat162 b = u < 4 ? __floats2bfloat162_rn(__uint_as_float(v[i]), __uint_as_float(v[i + 1]))
                                     : __floats2bfloat162_rn(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
      p[e] = *reinterpret_cast<const uint32_t*>(&b);
    }
    stg[lane * 8 + (u ^ (lane & 7))] = make_uint4(p[0], p[1], p[2], p[3]);
  }
  __syncwarp();
  const int q = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    const uint4 x = stg[r * 8 + (q ^ (r & 7))];
    if (r < rows && q * 16 < bytes) *reinterpret_cast<uint4*>(static_cast<char*>(base) + r * ld + q * 16) = x;
  }
  __syncwarp();
}

// h of eight features from f of row `row`, for the modes that read it: fetched before the accumulators are waited for
struct FfnH {
  float4 g[2], u[2];
};
template <int MODE>
__device__ __forceinline__ void ffn_load_h(const FfnArgs& a, long long row, int f, FfnH& h) {
  const float4* p = reinterpret_cast<const float4*>(a.h + row * (MODE == FFN_DACT_SWIGLU ? 2 : 1) * a.N + f);
  h.g[0] = __ldg(p);
  h.g[1] = __ldg(p + 1);
  if (MODE == FFN_DACT_SWIGLU) {
    const float4* q = reinterpret_cast<const float4*>(a.h + row * 2 * a.N + a.N + f);
    h.u[0] = __ldg(q);
    h.u[1] = __ldg(q + 1);
  }
}

// Eight features from f of row `row`: what the mode makes of the accumulators x and stores.
template <int MODE>
__device__ __forceinline__ void ffn_finish8(const FfnArgs& a, long long row, int f, float (&x)[8], const FfnH& h) {
  const float* hg = reinterpret_cast<const float*>(h.g);
  if (MODE == FFN_DACT_SWIGLU) {
    const float* hu = reinterpret_cast<const float*>(h.u);
    float g[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = ffn_sigmoid(hg[e]);
      g[e] = x[e] * hu[e] * s * (1.0f + hg[e] * (1.0f - s));
      u[e] = x[e] * hg[e] * s;
    }
    ffn_store8(a.out + row * 2 * a.N + f, g);
    ffn_store8(a.out + row * 2 * a.N + a.N + f, u);
    return;
  }
  if (MODE == FFN_DACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] *= 0.5f * (1.0f + erff(hg[e] * 0.70710678118654752f)) + hg[e] * 0.39894228040143268f * __expf(-0.5f * hg[e] * hg[e]);
  }
  if (MODE == FFN_UP_GELU) {
    if (a.h != nullptr) ffn_store8(a.h + row * a.N + f, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.5f * x[e] * (1.0f + erff(x[e] * 0.70710678118654752f));
  }
  ffn_store8(a.out + row * a.N + f, x);
}

// A tile of the schedule.  rows x features: tiles of a group lie together, its row tiles innermost (they share the
// weights); weight gradients: every group has the same tiles, whether it has rows or not.
struct FfnTile {
  int group;
  int m0;              // first of the 256 on the M side: a feature (FFN_DWEIGHT: a row of the group's result)
  int n0, n;           // the N side: first row of the buffers (FFN_DWEIGHT: first feature) and how many
  int k0, k_rows;      // FFN_DWEIGHT: the group's rows
  int k_steps;
};
// rows of each of a group's tiles but the last, which has the rest
__device__ __forceinline__ int ffn_split(int cnt) {
  const int tiles = (cnt + kFfnRows - 1) / kFfnRows;
  return tiles <= 1 ? kFfnRows : ((cnt + tiles - 1) / tiles + 15) / 16 * 16;
}
template <int MODE>
__device__ __forceinline__ FfnTile ffn_tile(const FfnArgs& a, const int* s_off, const int* s_items, int item) {
  FfnTile t;
  if (MODE == FFN_DWEIGHT) {
    const int nt = (a.N + kFfnRows - 1) / kFfnRows, mt = (a.M + 255) / 256;
    t.group = item / (nt * mt);
    const int r = item - t.group * nt * mt;
    t.n0 = (r / mt) * kFfnRows;
    t.n = min(kFfnRows, a.N - t.n0);
    t.m0 = (r % mt) * 256;
    t.k0 = s_off[t.group];
    t.k_rows = s_off[t.group + 1] - t.k0;
    t.k_steps = (t.k_rows + 63) / 64;
  } else {
    int lo = 0, hi = a.G - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_items[mid] <= item) lo = mid; else hi = mid - 1;
    }
    const int first = s_off[lo], cnt = s_off[lo + 1] - first;
    const int split = ffn_split(cnt);
    const int mt = (cnt + split - 1) / split;
    const int r = item - s_items[lo];
    t.group = lo;
    t.m0 = (r / mt) * a.feat;
    const int skip = (r % mt) * split;
    t.n0 = first + skip;
    t.n = min(split, cnt - skip);
    t.k0 = t.k_rows = 0;
    t.k_steps = (a.K + 63) / 64;
  }
  return t;
}
// The limit of a wait that lasts as long as `steps` steps of sums (0.28 us each with one tile on the machine: 2 s would be 460
// million rows): 2^-20 of what was set more for each.  All other waits are for a step or two.
__device__ __forceinline__ unsigned long long ffn_limit(const FfnArgs& a, unsigned long long steps) {
  return a.limit_ns + (a.limit_ns >> 20) * steps;
}
// rows of the last K step of a weight gradient that an instruction would read but that belong to other experts
__device__ __forceinline__ int ffn_foreign(int rows) { return (16 - (rows & 15)) & 15; }

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFfnThreads, 1)
ffn_kernel(const __grid_constant__ CUtensorMap tm_f, const __grid_constant__ CUtensorMap tm_r32,
           const __grid_constant__ CUtensorMap tm_r128, const FfnArgs a) {
  constexpr bool kWeightsK = MODE == FFN_UP_SWIGLU || MODE == FFN_UP_GELU || MODE == FFN_DOWN;   // features are K-major
  __shared__ __align__(8) uint64_t full_bar[kFfnMaxStages], empty_bar[kFfnMaxStages], tail_bar[kFfnMaxStages];
  __shared__ __align__(8) uint64_t acc_full_bar[kAccStages], acc_empty_bar[kAccStages], drain_bar;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ unsigned long long s_issued;                // this CTA's loads, for a kernel that gave up
  __shared__ uint32_t s_tail[kFfnMaxStages];             // 1 + parity on tail_bar of a load that warp 2 has yet to pass on, else 0
  extern __shared__ __align__(16) uint8_t smem_raw[];
  int* s_off = reinterpret_cast<int*>(smem_raw);         // [G + 1] first row of each group
  int* s_items = s_off + a.G + 1;                        // [G + 1] tiles before it
  uint8_t* smem = (uint8_t*)(((uintptr_t)(s_items + a.G + 1) + 1023) & ~(uintptr_t)1023);
  float* staging = reinterpret_cast<float*>(smem + (size_t)a.stages * kFfnStageBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int stages = a.stages;
  const int cta = (int)cluster_ctarank();                // 0: the pair's CTA that issues the MMAs
  const int pair = (int)blockIdx.x >> 1;
  const int pairs = (int)gridDim.x >> 1;
  const int n_tiles = (a.N + a.feat - 1) / a.feat;

  if (warp == 2) {
    // the offsets, made safe against any contents: not decreasing, within the buffers, the first one 0
    int last = 0, items = 0;
    for (int g0 = 0; g0 <= a.G; g0 += 32) {
      const int g = g0 + lane;
      int v = 0;
      if (g > 0 && g <= a.G) v = (int)min((long long)max(a.offsets[g], 0), a.n);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
      }
      v = max(v, last);
      int before = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0) before = last;
      const int split = ffn_split(v - before);
      int cnt = g > 0 && g <= a.G ? (v - before + split - 1) / split * n_tiles : 0;       // tiles of group g - 1
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, cnt, o);
        if (lane >= o) cnt += u;
      }
      if (g <= a.G) {
        s_off[g] = g == 0 ? 0 : v;
        s_items[g] = items + cnt;
      }
      last = __shfl_sync(0xffffffffu, v, 31);
      items += __shfl_sync(0xffffffffu, cnt, 31);
    }
  }
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < stages; ++s) {
      s_tail[s] = 0;
      mbar_init(&full_bar[s], 2);                        // one arrival (with its byte count) per CTA
      mbar_init(&empty_bar[s], 1);
      mbar_init(&tail_bar[s], 1);
    }
    for (int s = 0; s < kAccStages; ++s) {
      mbar_init(&acc_full_bar[s], 1);
      mbar_init(&acc_empty_bar[s], 2 * kFfnEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_f);
    tma_prefetch_desc(&tm_r32);
    tma_prefetch_desc(&tm_r128);
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_base_smem, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                    // both CTAs' barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_smem;
  volatile int* abortp = &abort_flag;
  const uint32_t peer_abort = map_to_cta(smem_u32(&abort_flag), (uint32_t)cta ^ 1u);
  const uint32_t lead_full = map_to_cta(smem_u32(&full_bar[0]), 0u);            // + 8 * stage
  const uint32_t lead_acc_empty = map_to_cta(smem_u32(&acc_empty_bar[0]), 0u);
  const int total = MODE == FFN_DWEIGHT ? a.G * ((a.N + kFfnRows - 1) / kFfnRows) * ((a.M + 255) / 256) : s_items[a.G];
  auto give_up = [&](int what, int item, int step) {
    record_timeout(a.status, what, item, step);
    abort_flag = 1;
    st_shared_cluster_u32(peer_abort, 1u);
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (one per CTA)
    int stage = 0;
    uint32_t phase = 0, tail_phase = 0;
    unsigned long long issued = 0;
    bool ok = true;
    for (int item = pair; item < total && ok; item += pairs) {
      const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
      const int half = (t.n + 15) / 16 * 8;              // this CTA's share of the N side: a multiple of 8
      const bool whole = MODE == FFN_DWEIGHT || half > 96;
      const int pieces = (half + 31) / 32;               // else: boxes of 32 rows
      const uint32_t tx = kFfnHalfBytes + (whole ? (uint32_t)kFfnHalfBytes : (uint32_t)pieces * 32u * 128u);
      const int row = t.n0 + cta * half;
      for (int kb = 0; kb < t.k_steps; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abortp, a.limit_ns));
        if (!ok) {
          if (lane == 0) give_up(WAIT_MBAR_EMPTY, item, kb);
          break;
        }
        uint8_t* sf = smem + (size_t)stage * kFfnStageBytes;
        uint8_t* sr = sf + kFfnHalfBytes;
        const uint32_t bar = lead_full + 8u * (uint32_t)stage;
        if (elect_one()) {
          if (MODE == FFN_DWEIGHT) {
            const int k = t.k0 + kb * 64, f = t.m0 + cta * 128;
            if (kb == t.k_steps - 1 && ffn_foreign(t.k_rows) != 0) {
              // a step with rows of other experts lands on a barrier of this CTA's own: warp 2 clears them first
              s_tail[stage] = 1u + ((tail_phase >> stage) & 1u);
              mbar_expect_tx(&tail_bar[stage], tx);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d(sf + i * kFfnBlockBytes, &tm_f, &tail_bar[stage], f + 64 * i, k);
                tma_load_2d(sr + i * kFfnBlockBytes, &tm_r128, &tail_bar[stage], row + 64 * i, k);
              }
            } else {
              mbar_arrive_expect_tx_cluster(bar, tx);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d_pair(sf + i * kFfnBlockBytes, &tm_f, bar, f + 64 * i, k);
                tma_load_2d_pair(sr + i * kFfnBlockBytes, &tm_r128, bar, row + 64 * i, k);
              }
            }
          } else {
            mbar_arrive_expect_tx_cluster(bar, tx);
            if (MODE == FFN_UP_SWIGLU) {
              tma_load_3d_pair(sf, &tm_f, bar, kb * 64, t.m0 + cta * 64, t.group);
              tma_load_3d_pair(sf + kFfnBlockBytes, &tm_f, bar, kb * 64, a.N + t.m0 + cta * 64, t.group);
            } else if (kWeightsK) {
              tma_load_3d_pair(sf, &tm_f, bar, kb * 64, t.m0 + cta * 128, t.group);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i)
                tma_load_3d_pair(sf + i * kFfnBlockBytes, &tm_f, bar, t.m0 + cta * 128 + 64 * i, kb * 64, t.group);
            }
            if (whole) {
              tma_load_2d_pair(sr, &tm_r128, bar, kb * 64, row);
            } else {
              for (int i = 0; i < pieces; ++i) tma_load_2d_pair(sr + i * 32 * 128, &tm_r32, bar, kb * 64, row + 32 * i);
            }
          }
        }
        __syncwarp();
        if (MODE == FFN_DWEIGHT && kb == t.k_steps - 1 && ffn_foreign(t.k_rows) != 0) tail_phase ^= 1u << stage;
        ++issued;
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
    }
    if (lane == 0) s_issued = issued;
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (cta == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int item = pair; item < total && ok; item += pairs) {
        const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
        if (t.k_steps == 0) continue;                    // a weight gradient without rows
        uint32_t idesc = make_idesc_bf16(256u, (uint32_t)((t.n + 15) / 16 * 16));
        if (!kWeightsK) idesc |= 1u << 15;               // the features are MN-major
        if (MODE == FFN_DWEIGHT) idesc |= 1u << 16;      // the rows too
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_empty_bar[acc], acc_phase ^ 1, abortp, a.limit_ns));
        if (!ok) {
          if (lane == 0) give_up(WAIT_TMEM_EMPTY, item, acc);
          break;
        }
        mbar_seen_pair(&acc_empty_bar[acc], acc_phase ^ 1);
        tc_fence_after();
        const uint32_t d0 = tmem_base + acc * 256;
        for (int kb = 0; kb < t.k_steps; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full_bar[stage], phase, abortp, a.limit_ns));
          if (!ok) {
            if (lane == 0) give_up(WAIT_MBAR_FULL, item, kb);
            break;
          }
          int steps = 4;
          if (MODE == FFN_DWEIGHT && kb == t.k_steps - 1) {
            steps = (t.k_rows - kb * 64 + 15) / 16;
            if (ffn_foreign(t.k_rows) != 0) {            // both CTAs' cleared rows
              mbar_seen_pair(&full_bar[stage], phase);
              fence_acquire_pair_shared();
            }
          }
          tc_fence_after();
          const uint32_t sf = smem_u32(smem + (size_t)stage * kFfnStageBytes), sr = sf + kFfnHalfBytes;
          const uint64_t fd = kWeightsK ? make_kmajor_sw128_desc(sf) : make_mnmajor_sw128_desc(sf);
          const uint64_t rd = MODE == FFN_DWEIGHT ? make_mnmajor_sw128_desc(sr) : make_kmajor_sw128_desc(sr);
          constexpr uint64_t df = kWeightsK ? 2 : 128, dr = MODE == FFN_DWEIGHT ? 128 : 2;      // 16 K further, 16-byte units
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (MODE != FFN_DWEIGHT || k < steps) umma_bf16_pair(d0, fd + df * k, rd + dr * k, idesc, (kb | k) != 0 ? 1u : 0u);
            umma_commit_pair(&empty_bar[stage]);
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (elect_one()) umma_commit_pair(&acc_full_bar[acc]);
        __syncwarp();
        if (++acc == kAccStages) { acc = 0; acc_phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------------ clears the other experts' rows of last K steps
    if (MODE == FFN_DWEIGHT) {
      int stage = 0;
      uint32_t tail_phase = 0;
      unsigned long long steps = 0;                      // since the last wait
      for (int item = pair; item < total; item += pairs) {
        const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
        const int foreign = ffn_foreign(t.k_rows);
        if (t.k_steps == 0) continue;
        stage = (stage + t.k_steps - 1) % stages;
        steps += t.k_steps;
        if (foreign != 0) {
          const bool ok = mbar_wait_bounded(&tail_bar[stage], (tail_phase >> stage) & 1u, abortp, ffn_limit(a, steps));
          steps = 0;
          if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0) give_up(WAIT_MBAR_FULL, item, -1);
            break;
          }
          tail_phase ^= 1u << stage;
          // lane: one of the 4 blocks x 8 units of 16 bytes that a K row has in a stage; the swizzle stays inside a block's row
          uint8_t* at = smem + (size_t)stage * kFfnStageBytes + (lane >> 3) * kFfnBlockBytes + (lane & 7) * 16;
          const int used = (t.k_rows - 1) % 64 + 1;
          for (int r = used; r < used + foreign; ++r) *reinterpret_cast<uint4*>(at + r * 128) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            s_tail[stage] = 0;
            fence_release_pair_shared();
            mbar_arrive_pair(lead_full + 8u * (uint32_t)stage);
          }
        }
        if (++stage == stages) stage = 0;
      }
    }
  } else if (warp >= kFfnEpiWarp0) {
    // ------------------------------------------------------------------ epilogue (8 warps, this CTA's TMEM)
    const int ew = warp - kFfnEpiWarp0;
    const int quad = ew & 3;                             // the TMEM lanes this warp may read
    const int group = ew >> 2;                           // which of every two chunks of 32 columns
    float* stg = staging + ew * (kFfnStagingBytes / 4);
    const int part = lane & 3, tr = lane >> 2;           // after the turn: eight features, a row of eight
    if (MODE == FFN_DOWN || MODE == FFN_DROWS) {
      // rows behind the last expert's: zero
      for (long long r = s_off[a.G] + (long long)blockIdx.x * kFfnEpiWarps + ew; r < a.n; r += (long long)kFfnEpiWarps * gridDim.x)
        for (int c = lane * 8; c < a.N; c += 256) *reinterpret_cast<uint4*>(a.out + r * a.N + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    // gate features are in quadrants 0 and 1, their up features in 2 and 3: two warps work on the same 32
    const int bar_id = 1 + group * 2 + (quad & 1);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool left = false;
    for (int item = pair; item < total && !left; item += pairs) {
      const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
      const int f = MODE == FFN_UP_SWIGLU ? t.m0 + cta * 64 + (quad & 1) * 32 + part * 8 : t.m0 + cta * 128 + quad * 32 + part * 8;
      // FFN_DWEIGHT: this warp's rows of the result
      const int wr0 = t.m0 + cta * 128 + quad * 32, w_rows = min(32, a.M - wr0);
      __nv_bfloat16* w_out = MODE == FFN_DWEIGHT ? a.out + ((long long)t.group * a.M + wr0) * a.N + t.n0 : nullptr;
      if (MODE == FFN_DWEIGHT && t.k_steps == 0) {
        for (int r = group; r < w_rows; r += 2)
          if (lane * 8 < t.n) *reinterpret_cast<uint4*>(w_out + (long long)r * a.N + lane * 8) = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      int got = 1;
      if (lane == 0) {
        got = mbar_wait_bounded(&acc_full_bar[acc], acc_phase, abortp, ffn_limit(a, t.k_steps)) ? 1 : 0;
        if (!got && !*abortp) give_up(WAIT_TMEM_FULL, item, acc);
      }
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) {
        if (MODE == FFN_UP_SWIGLU) asm volatile("bar.arrive %0, 64;" ::"r"(bar_id) : "memory");      // its partner goes on to leave
        break;
      }
      tc_fence_after();
      const uint32_t t0 = tmem_base + acc * 256 + ((uint32_t)(quad * 32) << 16);
      if (MODE == FFN_DWEIGHT) {
        for (int c = group * 64; c < t.n && w_rows > 0; c += 128) {
          uint32_t v[32], w[32];
          tmem_ld_32x32(t0 + c, v);
          tmem_ld_32x32(t0 + c + 32, w);
          tmem_ld_wait();
          ffn_put(reinterpret_cast<uint4*>(stg), v, w, w_out + c, 2ll * a.N, w_rows, 2 * (t.n - c), lane);
        }
      }
      for (int c = group * 32; MODE != FFN_DWEIGHT && c < t.n; c += 64) {
        uint32_t v[32];
        FfnH h[4];
        if (MODE == FFN_DACT_SWIGLU || MODE == FFN_DACT_GELU) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i * 8 + tr < t.n && f < a.N) ffn_load_h<MODE>(a, t.n0 + c + i * 8 + tr, f, h[i]);
        }
        tmem_ld_32x32(t0 + c, v);
        tmem_ld_wait();
        ffn_turn_in(stg, v, lane);
        if (MODE == FFN_UP_SWIGLU) {
          asm volatile("bar.sync %0, 64;" ::"r"(bar_id) : "memory");
          if (__any_sync(0xffffffffu, *abortp)) {        // the partner may have left: go too, and count for its next round
            asm volatile("bar.arrive %0, 64;" ::"r"(bar_id) : "memory");
            left = true;
            break;
          }
          // the gate's warp takes the first sixteen rows, the up's warp the others
          const float* sg = staging + (ew & ~2) * (kFfnStagingBytes / 4);
          const float* su = staging + (ew | 2) * (kFfnStagingBytes / 4);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int j = (quad >> 1) * 16 + i * 8 + tr;
            if (c + j < t.n && f < a.N) {
              float g[8], u[8];
              ffn_turn_out(sg, j, part, g);
              ffn_turn_out(su, j, part, u);
              const long long row = t.n0 + c + j;
              if (a.h != nullptr) {
                ffn_store8(a.h + row * 2 * a.N + f, g);
                ffn_store8(a.h + row * 2 * a.N + a.N + f, u);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) g[e] = g[e] * ffn_sigmoid(g[e]) * u[e];
              ffn_store8(a.out + row * a.N + f, g);
            }
          }
          asm volatile("bar.sync %0, 64;" ::"r"(bar_id) : "memory");       // both have read: the staging is free
          if (__any_sync(0xffffffffu, *abortp)) {
            asm volatile("bar.arrive %0, 64;" ::"r"(bar_id) : "memory");
            left = true;
            break;
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = i * 8 + tr;
            if (c + j < t.n && f < a.N) {
              float x[8];
              ffn_turn_out(stg, j, part, x);
              ffn_finish8<MODE>(a, t.n0 + c + j, f, x, h[i]);
            }
          }
          __syncwarp();
        }
      }
      if (left) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_pair(lead_acc_empty + 8u * (uint32_t)acc);
      if (++acc == kAccStages) { acc = 0; acc_phase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                  // no MMA reads this CTA's shared memory any more, no arrival is in flight
  // Unless a role gave up, in either CTA (both have the flag then): its partners may have issued loads and MMAs that nobody
  // waited for.  They end before the pair leaves and frees its TMEM.
  if (*abortp) {
    int never = 0;
    if (warp == 1) {
      if (cta == 0 && elect_one()) umma_commit_pair(&drain_bar);
      __syncwarp();
      mbar_wait_bounded(&drain_bar, 0, &never, kFfnDrainNs);
    }
    if (warp == 0 && lane == 0) {
      for (int s = 0; s < stages; ++s)
        if (s_tail[s] != 0) mbar_wait_bounded(&tail_bar[s], s_tail[s] - 1, &never, kFfnDrainNs);
      if (cta == 0) {
        // All others land on this CTA's full barriers: one that lacks an arrival (a load that one CTA did not come to, or
        // cleared rows that were not passed on) is given it, so that its phase ends with the bytes of the other.
        const unsigned long long mine = s_issued, peer = ld_shared_cluster_u64(map_to_cta(smem_u32(&s_issued), 1u));
        const unsigned long long most = mine > peer ? mine : peer;
        for (unsigned long long i = most > (unsigned)stages ? most - stages : 0; i < most; ++i) {
          const int s = (int)(i % stages);
          if (i >= mine || s_tail[s] != 0) mbar_arrive(&full_bar[s]);
          if (i >= peer || ld_shared_cluster_u32(map_to_cta(smem_u32(&s_tail[s]), 1u)) != 0) mbar_arrive(&full_bar[s]);
          mbar_wait_bounded(&full_bar[s], (uint32_t)(i / stages) & 1u, &never, kFfnDrainNs);
        }
      }
    }
    __syncthreads();
    cluster_sync_all();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace zepp
