// The experts' products on rows sorted by expert, and their gradients, on tcgen05 / TMEM.
//
//   h = x W1[e]^T,   a = silu(h_gate) * h_up  or  gelu(h),   y = a W2[e]^T             (rows of expert e: offsets[e] .. offsets[e+1])
//   da = dy W2[e],   dh = da * (derivative of the activation at h),   dx = dh W1[e]
//   dW2[e] = dy_e^T a_e,   dW1[e] = dh_e^T x_e                                          (sums over the expert's rows)
//
// One kernel template computes all of them: a tile is 128 x 256 fp32 accumulators, K steps of 64.
//   rows x features (h, y, da, dx): the rows are the M side, K-major as stored; the weights are the N side, K-major as
//     stored for the forward products and MN-major for the gradients (W is then read along its other dimension, nothing
//     is transposed in memory).  Features 0..255 of a tile are two blocks of 128 weight rows: for the gated
//     activation the gate and the up block of the same features, so that one thread holds both.
//   weight gradients: both operands MN-major, K = the expert's rows, of any number.  The last K step takes only as many
//     instructions as it has rows in sixteens; rows behind the expert's last one in it belong to the next expert and are
//     zeroed in shared memory first (in both operands: 0 * inf would not vanish).
// One persistent CTA per SM: warp 0 loads (TMA), warp 1 issues the MMAs and owns TMEM, warps 2..5 are the epilogue, two
// accumulators of 256 columns let it run under the next tile's MMAs.  Every wait is bounded.
//
// Roundings: products accumulate in fp32; h is kept as it is, in fp32, for the backward pass (in bf16 its rounding made the
// gradients of rows and w1 a quarter less exact, 3.0e-3 of their norm against 2.4e-3, for 2 % of the time of a training
// step); a and dh are rounded to bf16 because the next product's operands are bf16; y, dx, dW once at the end.
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
constexpr int kFfnStages = 4;
constexpr int kFfnABytes = 128 * 128;                   // 128 rows x 64 bf16, or two blocks of 64 rows x 64 columns
constexpr int kFfnBBytes = 256 * 128;
constexpr int kFfnStageBytes = kFfnABytes + kFfnBBytes;  // 48 KB
constexpr int kFfnSmemBytes = kFfnStages * kFfnStageBytes + 1024;
constexpr int kFfnBlockBytes = 64 * 128;                // an MN-major operand block: 64 K rows x 64 elements

struct FfnArgs {
  const int* offsets;        // [G + 1]
  int G;
  long long n;               // rows of the buffers
  int K;                     // length of the contraction (not used by FFN_DWEIGHT)
  int M, N;                  // FFN_DWEIGHT: rows of the result; all: features of the result before the activation's halving
  int up_offset;             // FFN_UP_SWIGLU: weight rows between gate and up (I); else 128
  int feat;                  // features per tile: 128 (FFN_UP_SWIGLU) or 256
  __nv_bfloat16* out;        // a, y, dh, dx or dW
  float* h;                  // FFN_UP_*: written if not null; FFN_DACT_*: read
  int wide;                  // output rows start on 32-byte boundaries
  unsigned long long* status;
  unsigned long long limit_ns;
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* tmap, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
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

// 32 consecutive features of one output row; `left`: features the row still has from here (a multiple of 8)
__device__ __forceinline__ void ffn_store32(__nv_bfloat16* out, int left, bool wide, const float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    w[e] = *reinterpret_cast<const uint32_t*>(&p);
  }
  if (wide && left >= 32) {
    st_global_v8(out, reinterpret_cast<const uint32_t(&)[8]>(w[0]));
    st_global_v8(out + 16, reinterpret_cast<const uint32_t(&)[8]>(w[8]));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (left >= 8 * (q + 1)) *reinterpret_cast<uint4*>(out + 8 * q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
  }
}
// the same of an fp32 row (eight features are 32 bytes, on a boundary of as many)
__device__ __forceinline__ void ffn_store32(float* out, int left, const uint32_t (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (left >= 8 * (q + 1)) {
      const uint32_t w[8] = {v[8 * q], v[8 * q + 1], v[8 * q + 2], v[8 * q + 3], v[8 * q + 4], v[8 * q + 5], v[8 * q + 6], v[8 * q + 7]};
      st_global_v8(out + 8 * q, w);
    }
}
__device__ __forceinline__ void ffn_load32(const float* in, int left, float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    if (left >= 4 * (q + 1)) w = *reinterpret_cast<const float4*>(in + 4 * q);
    v[4 * q] = w.x; v[4 * q + 1] = w.y; v[4 * q + 2] = w.z; v[4 * q + 3] = w.w;
  }
}
__device__ __forceinline__ float ffn_sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// The epilogue of one accumulator quadrant: this thread's row of the tile (TMEM lane), `row` its index in the buffers
// (FFN_DWEIGHT: the row of the result, counted over all groups), f0 the tile's first feature.
template <int MODE>
__device__ __forceinline__ void ffn_epilogue(const FfnArgs& a, uint32_t t0, bool mine, long long row, int f0) {
  const int feats = MODE == FFN_UP_SWIGLU ? a.N / 2 : a.N;
  const int end = min(a.feat, feats - f0);
  for (int c = 0; c < end; c += 32) {
    uint32_t r0[32];
    tmem_ld_32x32(t0 + c, r0);
    const int left = end - c;
    if (MODE == FFN_UP_SWIGLU) {
      uint32_t r1[32];
      tmem_ld_32x32(t0 + 128 + c, r1);
      tmem_ld_wait();
      if (mine) {
        float g[32], u[32], v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          g[e] = __uint_as_float(r0[e]);
          u[e] = __uint_as_float(r1[e]);
          v[e] = g[e] * ffn_sigmoid(g[e]) * u[e];
        }
        ffn_store32(a.out + row * feats + f0 + c, left, a.wide, v);
        if (a.h != nullptr) {
          ffn_store32(a.h + row * a.N + f0 + c, left, r0);
          ffn_store32(a.h + row * a.N + feats + f0 + c, left, r1);
        }
      }
    } else if (MODE == FFN_DACT_SWIGLU) {
      float g[32], u[32];
      if (mine) {
        ffn_load32(a.h + row * 2 * a.N + f0 + c, left, g);
        ffn_load32(a.h + row * 2 * a.N + a.N + f0 + c, left, u);
      }
      tmem_ld_wait();
      if (mine) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float da = __uint_as_float(r0[e]);
          const float s = ffn_sigmoid(g[e]);
          const float dg = da * u[e] * s * (1.0f + g[e] * (1.0f - s));
          u[e] = da * g[e] * s;
          g[e] = dg;
        }
        ffn_store32(a.out + row * 2 * a.N + f0 + c, left, a.wide, g);
        ffn_store32(a.out + row * 2 * a.N + a.N + f0 + c, left, a.wide, u);
      }
    } else if (MODE == FFN_DACT_GELU) {
      float h[32];
      if (mine) ffn_load32(a.h + row * a.N + f0 + c, left, h);
      tmem_ld_wait();
      if (mine) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = h[e];
          h[e] = __uint_as_float(r0[e]) *
                 (0.5f * (1.0f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x));
        }
        ffn_store32(a.out + row * a.N + f0 + c, left, a.wide, h);
      }
    } else {
      tmem_ld_wait();
      if (mine) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r0[e]);
        if (MODE == FFN_UP_GELU) {
          if (a.h != nullptr) ffn_store32(a.h + row * a.N + f0 + c, left, r0);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.5f * v[e] * (1.0f + erff(v[e] * 0.70710678118654752f));
        }
        ffn_store32(a.out + row * a.N + f0 + c, left, a.wide, v);
      }
    }
  }
}

// A tile of the schedule.  rows x features: tiles of a group lie together, its row tiles innermost (they share the
// weight tile); weight gradients: every group has the same tiles, whether it has rows or not.
struct FfnTile {
  int group, row0, rows, f0, m0, k_steps;
};
template <int MODE>
__device__ __forceinline__ FfnTile ffn_tile(const FfnArgs& a, const int* s_off, const int* s_items, int item) {
  FfnTile t;
  if (MODE == FFN_DWEIGHT) {
    const int nt = (a.N + 255) / 256, mt = (a.M + 127) / 128;
    t.group = item / (nt * mt);
    const int r = item - t.group * nt * mt;
    t.f0 = (r / mt) * 256;
    t.m0 = (r % mt) * 128;
    t.row0 = s_off[t.group];
    t.rows = s_off[t.group + 1] - t.row0;
    t.k_steps = (t.rows + 63) / 64;
  } else {
    int lo = 0, hi = a.G - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_items[mid] <= item) lo = mid; else hi = mid - 1;
    }
    const int first = s_off[lo], cnt = s_off[lo + 1] - first;
    const int mt = (cnt + 127) / 128;
    const int r = item - s_items[lo];
    t.group = lo;
    t.f0 = (r / mt) * a.feat;
    t.m0 = (r % mt) * 128;
    t.row0 = first + t.m0;
    t.rows = min(128, cnt - t.m0);
    t.k_steps = (a.K + 63) / 64;
  }
  return t;
}

template <int MODE>
__global__ void __launch_bounds__(192, 1)
ffn_kernel(const __grid_constant__ CUtensorMap tm_a32, const __grid_constant__ CUtensorMap tm_a64,
           const __grid_constant__ CUtensorMap tm_a128, const __grid_constant__ CUtensorMap tm_b, const FfnArgs a) {
  constexpr bool kBRows = MODE == FFN_UP_SWIGLU || MODE == FFN_UP_GELU || MODE == FFN_DOWN;   // B is K-major
  constexpr int STAGES = kFfnStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[STAGES];
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t acc_full_bar[kAccStages];
  __shared__ __align__(8) uint64_t acc_empty_bar[kAccStages];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ int s_off[kFfnMaxGroups + 1], s_items[kFfnMaxGroups + 1];

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int feats = MODE == FFN_UP_SWIGLU ? a.N / 2 : a.N;
  const int n_tiles = (feats + a.feat - 1) / a.feat;

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
      int cnt = g > 0 && g <= a.G ? (v - before + 127) / 128 * n_tiles : 0;       // tiles of group g - 1
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
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < kAccStages; ++s) {
      mbar_init(&acc_full_bar[s], 1);
      mbar_init(&acc_empty_bar[s], 4);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_b);
    tma_prefetch_desc(&tm_a128);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_smem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_smem;
  volatile int* abortp = &abort_flag;
  const int total = MODE == FFN_DWEIGHT ? a.G * n_tiles * ((a.M + 127) / 128) : s_items[a.G];

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      for (int item = blockIdx.x; item < total && !*abortp; item += gridDim.x) {
        const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
        const CUtensorMap* tma = &tm_a128;
        uint32_t tx = kFfnStageBytes;
        if (MODE != FFN_DWEIGHT) {
          tma = t.rows <= 32 ? &tm_a32 : (t.rows <= 64 ? &tm_a64 : &tm_a128);
          tx = kFfnBBytes + (t.rows <= 32 ? 32u : (t.rows <= 64 ? 64u : 128u)) * 128u;
        }
        for (int kb = 0; kb < t.k_steps; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abortp, a.limit_ns)) {
            record_timeout(a.status, WAIT_MBAR_EMPTY, item, kb);
            abort_flag = 1;
            break;
          }
          uint8_t* sa = smem + stage * kFfnStageBytes;
          uint8_t* sb = sa + kFfnABytes;
          uint64_t* bar = &full_bar[stage];
          mbar_expect_tx(bar, tx);
          if (MODE == FFN_DWEIGHT) {
            const int k0 = t.row0 + kb * 64;
#pragma unroll
            for (int i = 0; i < 2; ++i) tma_load_2d(sa + i * kFfnBlockBytes, tma, bar, t.m0 + 64 * i, k0);
#pragma unroll
            for (int i = 0; i < 4; ++i) tma_load_2d(sb + i * kFfnBlockBytes, &tm_b, bar, t.f0 + 64 * i, k0);
          } else {
            tma_load_2d(sa, tma, bar, kb * 64, t.row0);
            if (kBRows) {
              tma_load_3d(sb, &tm_b, bar, kb * 64, t.f0, t.group);
              tma_load_3d(sb + kFfnABytes, &tm_b, bar, kb * 64, t.f0 + a.up_offset, t.group);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) tma_load_3d(sb + i * kFfnBlockBytes, &tm_b, bar, t.f0 + 64 * i, kb * 64, t.group);
            }
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (*abortp) {                                     // given up: the block stays until its loads have landed
        int never = 0;
        for (long long i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
          mbar_wait_bounded(&full_bar[i % STAGES], (uint32_t)(i / STAGES) & 1u, &never, a.limit_ns);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (the warp stays together, lane 0 issues)
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    uint32_t idesc = make_idesc_bf16(128u, 256u);
    if (MODE == FFN_DWEIGHT) idesc |= 1u << 15;          // A is MN-major
    if (!kBRows) idesc |= 1u << 16;                      // B is MN-major
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
      const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
      if (t.k_steps == 0) continue;                      // a weight gradient without rows
      bool ok = mbar_wait_bounded(&acc_empty_bar[acc], acc_phase ^ 1, abortp, a.limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) {
          record_timeout(a.status, WAIT_TMEM_EMPTY, item, acc);
          abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      const uint32_t d0 = tmem_base + acc * 256;
      for (int kb = 0; kb < t.k_steps; ++kb) {
        ok = mbar_wait_bounded(&full_bar[stage], phase, abortp, a.limit_ns);
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) {
            record_timeout(a.status, WAIT_MBAR_FULL, item, kb);
            abort_flag = 1;
          }
          ok = false;
          break;
        }
        uint8_t* st = smem + stage * kFfnStageBytes;
        int steps = 4;
        if (MODE == FFN_DWEIGHT) {
          const int valid = t.rows - kb * 64;
          if (valid < 64) {
            steps = (valid + 15) / 16;
            const int bad = steps * 16 - valid;          // rows of other experts that an instruction would read
            for (int i = lane; i < bad * 48; i += 32) {
              const int r = valid + i / 48, q = i % 48;  // 6 blocks x 8 vectors; the swizzle stays inside a row
              *reinterpret_cast<uint4*>(st + (q >> 3) * kFfnBlockBytes + r * 128 + (q & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async();
            __syncwarp();
          }
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t sa = smem_u32(st), sb = sa + kFfnABytes;
          const uint64_t ad = MODE == FFN_DWEIGHT ? make_mnmajor_sw128_desc(sa) : make_kmajor_sw128_desc(sa);
          const uint64_t bd = kBRows ? make_kmajor_sw128_desc(sb) : make_mnmajor_sw128_desc(sb);
          constexpr uint64_t da = MODE == FFN_DWEIGHT ? 128 : 2, db = kBRows ? 2 : 128;      // 16 K further, 16-byte units
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (MODE != FFN_DWEIGHT || k < steps) umma_bf16(d0, ad + da * k, bd + db * k, idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit(&empty_bar[stage]);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0) umma_commit(&acc_full_bar[acc]);
      __syncwarp();
      if (++acc == kAccStages) { acc = 0; acc_phase ^= 1; }
    }
    if (*abortp && lane == 0) {                          // given up: nothing of this block's is in flight when TMEM is freed
      int never = 0;
      umma_commit(&drain_bar);
      mbar_wait_bounded(&drain_bar, 0, &never, a.limit_ns);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue (4 warps)
    const int quad = warp & 3;                           // the TMEM lanes this warp may read
    if (MODE == FFN_DOWN || MODE == FFN_DROWS) {
      // rows behind the last expert's: zero
      const int ew = (blockIdx.x * 4 + (warp - 2));
      for (long long r = s_off[a.G] + ew; r < a.n; r += 4ll * gridDim.x)
        for (int c = lane * 8; c < a.N; c += 256) *reinterpret_cast<uint4*>(a.out + r * a.N + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    int acc = 0;
    uint32_t acc_phase = 0;
    const int r = quad * 32 + lane;
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
      const FfnTile t = ffn_tile<MODE>(a, s_off, s_items, item);
      if (MODE == FFN_DWEIGHT && t.k_steps == 0) {
        const int w = min(256, a.N - t.f0), rows = min(128, a.M - t.m0);
        for (int i = warp - 2; i < rows; i += 4)
          if (lane * 8 < w)
            *reinterpret_cast<uint4*>(a.out + ((long long)t.group * a.M + t.m0 + i) * a.N + t.f0 + lane * 8) = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      int got = 1;
      if (lane == 0) {
        got = mbar_wait_bounded(&acc_full_bar[acc], acc_phase, abortp, a.limit_ns) ? 1 : 0;
        if (!got && !*abortp) {
          record_timeout(a.status, WAIT_TMEM_FULL, item, acc);
          abort_flag = 1;
        }
      }
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) break;
      tc_fence_after();
      const int rows = MODE == FFN_DWEIGHT ? a.M - t.m0 : t.rows;
      if (quad * 32 < rows) {
        const long long row = MODE == FFN_DWEIGHT ? (long long)t.group * a.M + t.m0 + r : (long long)t.row0 + r;
        ffn_epilogue<MODE>(a, tmem_base + acc * 256 + ((uint32_t)(quad * 32) << 16), r < rows, row, t.f0);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty_bar[acc]);
      if (++acc == kAccStages) { acc = 0; acc_phase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace zepp
