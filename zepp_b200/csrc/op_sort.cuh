// Token rows sorted by expert and back.
//
//   sort:    copy i = t * K + k of a token goes to row  position[i] = offsets[g] + #{j < i : group(j) = g},  g = group(i);
//            rows[position[i]] = x[t];   offsets[g] = #{j : group(j) < g}.  Copies without a group have position -1.
//   unsort:  y[t] = sum_k w[t, k] * rows[position[t, k]]         (without weights: the gradient of the sort)
//   its gradient:  drows[position[t, k]] = w[t, k] * dy[t],   dw[t, k] = <dy[t], rows[position[t, k]]>
//
// The order is that of a stable sort by group, and every sum runs over k in order, so equal inputs give equal bits.
// Everything is bound by the bytes of the rows: the sort reads a row once and writes its K copies, the gradient of the
// unsort reads dy once and makes both of its results from one pass over the rows.  Measured with 8192 tokens x 8 copies of
// 4096 bf16: sort 4 + 120 us (5.0 TB/s, nearly all writes; a fill of memory reaches 3.9), unsort 102 us (5.9 TB/s), its
// gradient 185 us (6.2 TB/s).
#pragma once
#include "op_common.cuh"

namespace zepp {

constexpr int kSortThreads = 512;
constexpr int kSortMaxGroups = 2048;
// Up to this many copies every block counts all of them itself: one launch.  Against a launch that counts beforehand (128
// experts, rows of 2048 bf16): 4.1 us against 8.2 for 256 copies, 13.4 against 15.9 for 8192, 22 either way for 16384, 43
// against 38 for 32768.
constexpr int kSortDirect = 8192;
constexpr int kSortChunks = 64;         // above: parts of the copies that are counted beforehand

struct SortArgs {
  const int* ids;          // [T * K]
  const int* group_of;     // [n_ids] group of an id, or nullptr: the id itself
  int n_ids, G;
  long long T;
  int K;
  int tokens_per_block;
  int chunk;               // copies per counted part (0: nothing was counted)
  const int* counts;       // [chunks, G]
  const unsigned char* x;
  unsigned char* rows;
  long long row_bytes;
  int* offsets;            // [G + 1]
  int* position;           // [T * K]
};

__device__ __forceinline__ int sort_group(const SortArgs& a, long long i) {
  const int id = a.ids[i];
  if (id < 0 || id >= a.n_ids) return -1;
  const int g = a.group_of != nullptr ? a.group_of[id] : id;
  return g >= 0 && g < a.G ? g : -1;
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a, int* counts) {
  extern __shared__ int sort_hist[];
  for (int g = threadIdx.x; g < a.G; g += kSortThreads) sort_hist[g] = 0;
  __syncthreads();
  const long long n = a.T * a.K, lo = (long long)blockIdx.x * a.chunk;
  const long long hi = lo + a.chunk < n ? lo + a.chunk : n;
  for (long long i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const int g = sort_group(a, i);
    if (g >= 0) atomicAdd(&sort_hist[g], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.G; g += kSortThreads) counts[(long long)blockIdx.x * a.G + g] = sort_hist[g];
}

// V: the widest access that every row's address allows.  A block places the copies of its tokens, up to kSortThreads at a
// time (a thread counts the copies of its group before its own among them), then copies the tokens' rows.
template <typename V>
__global__ void __launch_bounds__(kSortThreads) sort_rows_kernel(const SortArgs a, int chunks) {
  extern __shared__ int sort_hist[];                   // next[G]: first free row of each group for this block's copies
  __shared__ int s_group[kSortThreads], s_pos[kSortThreads], s_warp[kSortThreads / 32];
  int* next = sort_hist;
  int* total = sort_hist + a.G;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long n = a.T * a.K;
  const long long t0 = (long long)blockIdx.x * a.tokens_per_block;
  const long long t1 = t0 + a.tokens_per_block < a.T ? t0 + a.tokens_per_block : a.T;
  const long long i0 = (t0 < a.T ? t0 : a.T) * a.K;
  const int part = a.chunk > 0 ? (int)(i0 / a.chunk) : 0;

  // copies of each group in all, and before this block's first one
  for (int g = tid; g < a.G; g += kSortThreads) {
    int before = 0, all = 0;
    for (int c = 0; c < chunks; ++c) {
      const int v = a.counts[(long long)c * a.G + g];
      if (c < part) before += v;
      all += v;
    }
    next[g] = before;
    total[g] = all;
  }
  __syncthreads();
  if (a.chunk > 0) {
    for (long long i = (long long)part * a.chunk + tid; i < i0; i += kSortThreads) {
      const int g = sort_group(a, i);
      if (g >= 0) atomicAdd(&next[g], 1);
    }
  } else {
    for (long long i = tid; i < n; i += kSortThreads) {
      const int g = sort_group(a, i);
      if (g >= 0) {
        atomicAdd(&total[g], 1);
        if (i < i0) atomicAdd(&next[g], 1);
      }
    }
  }
  __syncthreads();
  // rows before each group
  int carry = 0;
  for (int g0 = 0; g0 < a.G; g0 += kSortThreads) {
    const int g = g0 + tid;
    const int v = g < a.G ? total[g] : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < kSortThreads / 32; ++w) {
      if (w < warp) base += s_warp[w];
      carry += s_warp[w];
    }
    if (g < a.G) {
      next[g] += base + incl - v;
      if (blockIdx.x == 0) a.offsets[g] = base + incl - v;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) a.offsets[a.G] = carry;

  const int per = kSortThreads / a.K;                  // whole tokens placed at a time
  const long long vecs = a.row_bytes / (long long)sizeof(V);
  for (long long tb = t0; tb < t1; tb += per) {
    const int tokens = (int)(tb + per < t1 ? per : t1 - tb);
    const int m = tokens * a.K;
    const int g = tid < m ? sort_group(a, tb * a.K + tid) : -1;
    s_group[tid] = g;
    __syncthreads();
    int pos = -1;
    if (g >= 0) {
      pos = next[g];
      for (int j = 0; j < tid; ++j) pos += s_group[j] == g ? 1 : 0;
    }
    s_pos[tid] = pos;
    if (tid < m) a.position[tb * a.K + tid] = pos;
    __syncthreads();
    if (g >= 0) atomicMax(&next[g], pos + 1);
    // the rows: 32 neighbouring vectors of a token per warp and step, four steps' loads in flight
    const int lines = (int)((vecs + 31) / 32);
    for (int u0 = warp; u0 < tokens * lines; u0 += 4 * (kSortThreads / 32)) {
      V val[4];
      int t[4], v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int u = u0 + q * (kSortThreads / 32);
        t[q] = u / lines;
        v[q] = u < tokens * lines ? (u - t[q] * lines) * 32 + lane : (int)vecs;
        if (v[q] < vecs) val[q] = reinterpret_cast<const V*>(a.x + (tb + t[q]) * a.row_bytes)[v[q]];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (v[q] < vecs)
          for (int k = 0; k < a.K; ++k) {
            const int p = s_pos[t[q] * a.K + k];
            if (p >= 0) reinterpret_cast<V*>(a.rows + (long long)p * a.row_bytes)[v[q]] = val[q];
          }
    }
    __syncthreads();
  }
  // rows behind the last group hold zeros
  for (long long p = carry + (long long)blockIdx.x; p < n; p += gridDim.x)
    for (long long v = tid; v < vecs; v += kSortThreads) reinterpret_cast<V*>(a.rows + p * a.row_bytes)[v] = V{};
}

constexpr int kUnsortThreads = 256;
constexpr int kUnsortGradThreads = 128;

struct UnsortArgs {
  const void* rows;        // [N, H]
  long long T, N;
  int K;
  long long H;
  const int* position;     // [T, K]
  const float* weights;    // [T, K] or nullptr: 1
  void* y;                 // [T, H]
  // gradient
  const void* dy;          // [T, H]
  void* drows;             // [N, H] or nullptr
  float* dweights;         // [T, K] or nullptr
  const int* n_rows;       // device: rows that have a copy (those behind it get a zero gradient)
};

__device__ __forceinline__ int unsort_position(const UnsortArgs& a, long long i) {
  const int p = a.position[i];
  return p < a.N ? p : -1;
}

// A thread adds up U vectors of E elements (kUnsortThreads vectors apart) of a token's row, KU rows at a time in flight;
// blockIdx.x = token, blockIdx.y = part of the row.
template <typename T, int E, int U, int KU>
__global__ void __launch_bounds__(kUnsortThreads) unsort_kernel(const UnsortArgs a) {
  typedef Pack<T, E> V;
  const long long t = blockIdx.x;
  const int vecs = (int)(a.H / E);
  const int v0 = blockIdx.y * (kUnsortThreads * U) + threadIdx.x;
  float acc[U][E];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[u][e] = 0.0f;
  for (int k0 = 0; k0 < a.K; k0 += KU) {
    V r[KU][U];
    float w[KU];
    int p[KU];
#pragma unroll
    for (int q = 0; q < KU; ++q) {
      const int k = k0 + q;
      p[q] = k < a.K ? unsort_position(a, t * a.K + k) : -1;
      w[q] = k < a.K && a.weights != nullptr ? a.weights[t * a.K + k] : 1.0f;
    }
#pragma unroll
    for (int q = 0; q < KU; ++q)
      if (p[q] >= 0) {
        const V* src = reinterpret_cast<const V*>(static_cast<const T*>(a.rows) + (long long)p[q] * a.H);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + u * kUnsortThreads < vecs) r[q][u] = src[v0 + u * kUnsortThreads];
      }
#pragma unroll
    for (int q = 0; q < KU; ++q)
      if (p[q] >= 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[u][e] = fmaf(w[q], to_f32<T>(r[q][u].v[e]), acc[u][e]);
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v0 + u * kUnsortThreads < vecs) {
      V out;
#pragma unroll
      for (int e = 0; e < E; ++e) out.v[e] = from_f32<T>(acc[u][e]);
      reinterpret_cast<V*>(static_cast<T*>(a.y) + t * a.H)[v0 + u * kUnsortThreads] = out;
    }
}

// `wpt` warps of a block own a token: dy is read once for eight copies, each row once.  With one warp per token nothing in
// the block waits for anything else.
template <typename T, int E>
__global__ void __launch_bounds__(kUnsortGradThreads) unsort_grad_kernel(const UnsortArgs a, int wpt) {
  typedef Pack<T, E> V;
  constexpr int KB = 8;
  __shared__ float s_dot[2][kUnsortGradThreads / 32][KB];
  const int vecs = (int)(a.H / E);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_block = kUnsortGradThreads / 32 / wpt;
  const int sub = warp % wpt, first = warp - sub;        // this warp among its token's, and the first of them
  int flip = 0;
  // a block's warps go round together (the barrier below), those behind the last token without one
  for (long long t0 = (long long)blockIdx.x * per_block; t0 < a.T; t0 += (long long)gridDim.x * per_block) {
    const long long t = t0 + warp / wpt;
    const bool real = t < a.T;
    const V* dy = reinterpret_cast<const V*>(static_cast<const T*>(a.dy) + (real ? t : 0) * a.H);
    for (int k0 = 0; k0 < a.K; k0 += KB) {
      int p[KB];
      float w[KB], dot[KB];
#pragma unroll
      for (int q = 0; q < KB; ++q) {
        const int k = k0 + q;
        p[q] = real && k < a.K ? unsort_position(a, t * a.K + k) : -1;
        w[q] = real && k < a.K && a.weights != nullptr ? a.weights[t * a.K + k] : 1.0f;
        dot[q] = 0.0f;
      }
      for (int v = sub * 32 + lane; real && v < vecs; v += wpt * 32) {
        const V d = dy[v];
        if (a.dweights != nullptr) {
          V r[KB];
#pragma unroll
          for (int q = 0; q < KB; ++q)
            if (p[q] >= 0) r[q] = reinterpret_cast<const V*>(static_cast<const T*>(a.rows) + (long long)p[q] * a.H)[v];
#pragma unroll
          for (int q = 0; q < KB; ++q)
            if (p[q] >= 0) {
#pragma unroll
              for (int e = 0; e < E; ++e) dot[q] = fmaf(to_f32<T>(d.v[e]), to_f32<T>(r[q].v[e]), dot[q]);
            }
        }
        if (a.drows != nullptr) {
#pragma unroll
          for (int q = 0; q < KB; ++q)
            if (p[q] >= 0) {
              V o;
#pragma unroll
              for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(w[q] * to_f32<T>(d.v[e]));
              reinterpret_cast<V*>(static_cast<T*>(a.drows) + (long long)p[q] * a.H)[v] = o;
            }
        }
      }
      if (a.dweights != nullptr) {
        float mine = 0.0f;                               // lane q: the sum for copy k0 + q
#pragma unroll
        for (int q = 0; q < KB; ++q) {
          const float s = warp_sum(dot[q]);
          if (lane == q) mine = p[q] >= 0 ? s : 0.0f;
        }
        if (wpt > 1) {
          if (lane < KB) s_dot[flip][warp][lane] = mine;
          __syncthreads();
          if (sub == 0 && lane < KB)
            for (int i = 1; i < wpt; ++i) mine += s_dot[flip][first + i][lane];
          flip ^= 1;                                     // the other half is free: its readers passed this barrier
        }
        if (sub == 0 && lane < KB && real && k0 + lane < a.K) a.dweights[t * a.K + k0 + lane] = mine;
      }
    }
  }
  if (a.drows != nullptr) {
    long long begin = *a.n_rows;
    if (begin < 0) begin = 0;
    for (long long p = begin + blockIdx.x; p < a.N; p += gridDim.x)
      for (int v = threadIdx.x; v < vecs; v += kUnsortGradThreads) reinterpret_cast<V*>(static_cast<T*>(a.drows) + p * a.H)[v] = V{};
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The gradient once more, for long rows of 16-bit elements in large numbers: one persistent block per SM, a warp that fetches
// pieces of the rows into a ring of shared-memory stages with bulk copies, eight warps that work on them.  A stage holds one
// piece (kPieceBytes) of dy and of up to eight copies' rows, so nearly 200 KB are in flight on every SM whatever the
// registers allow, where the kernel above waits for its loads: 190 us against 235 (8192 tokens x 8 copies of 4096 bf16).
// Steps of a token: (eight copies, piece) with the piece inner, so that a sum over the row stays in registers.
constexpr int kPieceBytes = 4096;
constexpr int kPieceThreads = kPieceBytes / 16;         // consumers: a 16-byte vector each
constexpr int kBulkThreads = 32 + kPieceThreads;
constexpr int kBulkStageBytes = 9 * kPieceBytes;        // eight copies and dy
constexpr int kBulkStages = 5;
constexpr unsigned long long kBulkDrainNs = 2000000000ull;      // limit of each wait for copies after a role gave up

struct BulkArgs {
  UnsortArgs u;
  int pieces, chunks;         // of a row; of its copies, eight at a time
  unsigned long long* status;
  unsigned long long limit_ns;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kBulkThreads, 1) unsort_grad_bulk_kernel(const BulkArgs b) {
  constexpr int E = 16 / (int)sizeof(T);
  typedef Pack<T, E> V;
  const UnsortArgs& a = b.u;
  extern __shared__ __align__(128) unsigned char bulk_ring[];
  __shared__ __align__(8) uint64_t full[kBulkStages], empty[kBulkStages];
  __shared__ int s_pos[kBulkStages][8];
  __shared__ float s_w[kBulkStages][8];
  __shared__ float s_dot[2][kPieceThreads / 32][8];
  __shared__ int abort_flag;
  volatile int* abortp = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kBulkStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kPieceThreads / 32);
    }
    fence_barrier_init();
  }
  __syncthreads();
  const int per_token = b.pieces * b.chunks;
  // gridDim.x <= T; rows of 4 KB and more: far fewer than 2^31 fit the memory
  const int mine = ((int)a.T - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int total = mine * per_token;
  const long long row_bytes = a.H * (long long)sizeof(T);
  int issued = 0;                                              // warp 0: stages whose copies it has started

  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    // Positions and weights of four steps at a time (lane: step lane / 8, copy lane % 8), four steps ahead: they are the
    // first link of every chain of loads, and one step ahead each stage still waited for most of their latency.
    int token = blockIdx.x, step = 0, stage = 0;
    uint32_t phase = 0;
    int p_next = -1, p_four = -1;
    float w_next = 1.0f, w_four = 1.0f;
    auto fetch = [&](int i) {
      i += lane >> 3;
      p_next = -1;
      w_next = 1.0f;
      if (i < total) {
        const int k = i % per_token / b.pieces * 8 + (lane & 7);
        const long long at = (long long)((int)blockIdx.x + i / per_token * (int)gridDim.x) * a.K + k;
        if (k < a.K) {
          p_next = unsort_position(a, at);
          if (a.weights != nullptr) w_next = a.weights[at];
        }
      }
    };
    fetch(0);
    for (int i = 0; i < total; ++i) {
      if ((i & 3) == 0) {
        p_four = p_next;
        w_four = w_next;
        fetch(i + 4);
      }
      const int from = (i & 3) * 8 + (lane & 7);
      const int p_lane = __shfl_sync(0xffffffffu, p_four, from);
      const int now_p = lane < 8 ? p_lane : -1;
      const float now_w = __shfl_sync(0xffffffffu, w_four, from);
      const long long t = token;
      const uint32_t at = (uint32_t)(step % b.pieces) * kPieceBytes;
      const uint32_t bytes = (uint32_t)min((long long)kPieceBytes, row_bytes - at);
      if (++step == per_token) { step = 0; token += gridDim.x; }
      const bool ok = mbar_wait_bounded(&empty[stage], phase ^ 1, abortp, b.limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) {
          record_timeout(b.status, WAIT_MBAR_EMPTY, t, i);
          abort_flag = 1;
        }
        break;
      }
      if (lane < 8) {
        s_pos[stage][lane] = now_p;
        s_w[stage][lane] = now_w;
      }
      const bool rows = a.dweights != nullptr;
      const uint32_t copies = rows ? __popc(__ballot_sync(0xffffffffu, now_p >= 0)) : 0u;
      __syncwarp();
      if (lane == 0) mbar_expect_tx(&full[stage], (copies + 1u) * bytes);
      __syncwarp();
      unsigned char* st = bulk_ring + (size_t)stage * kBulkStageBytes;
      if (rows && now_p >= 0)
        bulk_load(st + lane * kPieceBytes, static_cast<const unsigned char*>(a.rows) + now_p * row_bytes + at, bytes, &full[stage]);
      if (lane == 8)
        bulk_load(st + 8 * kPieceBytes, static_cast<const unsigned char*>(a.dy) + t * row_bytes + at, bytes, &full[stage]);
      ++issued;
      if (++stage == kBulkStages) { stage = 0; phase ^= 1; }
    }
  } else {
    // ---------------------------------------------------------------- sums
    const int v = threadIdx.x - 32;
    int token = blockIdx.x, step = 0, stage = 0, flip = 0;
    uint32_t phase = 0;
    float acc[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
    for (int i = 0; i < total; ++i) {
      const int piece = step % b.pieces, chunk = step / b.pieces;
      const long long t = token;
      const long long at = (long long)piece * kPieceBytes + v * 16;
      const bool in = at < row_bytes;
      const bool ok = mbar_wait_bounded(&full[stage], phase, abortp, b.limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !*abortp) record_timeout(b.status, WAIT_MBAR_FULL, t, i);
        abort_flag = 1;
        asm volatile("bar.arrive 1, %0;" ::"n"(kPieceThreads) : "memory");      // nobody is left waiting below
        break;
      }
      const unsigned char* st = bulk_ring + (size_t)stage * kBulkStageBytes + v * 16;
      if (in) {
        const V d = *reinterpret_cast<const V*>(st + 8 * kPieceBytes);
        float f[E];
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = to_f32<T>(d.v[e]);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int p = s_pos[stage][q];
          if (p >= 0) {
            if (a.dweights != nullptr) {
              const V r = *reinterpret_cast<const V*>(st + q * kPieceBytes);
#pragma unroll
              for (int e = 0; e < E; ++e) acc[q] = fmaf(f[e], to_f32<T>(r.v[e]), acc[q]);
            }
            if (a.drows != nullptr) {
              const float w = s_w[stage][q];
              V o;
#pragma unroll
              for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(w * f[e]);
              *reinterpret_cast<V*>(static_cast<unsigned char*>(a.drows) + p * row_bytes + at) = o;
            }
          }
        }
      }
      const int p_of_lane = lane < 8 ? s_pos[stage][lane] : -1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      if (++stage == kBulkStages) { stage = 0; phase ^= 1; }
      if (piece == b.pieces - 1 && a.dweights != nullptr) {    // eight copies of a token are done
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float s = warp_sum(acc[q]);
          if (lane == q) s_dot[flip][warp - 1][q] = s;
          acc[q] = 0.0f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kPieceThreads) : "memory");
        if (__any_sync(0xffffffffu, *abortp)) {                // a warp that gave up has left: go too, and count for the next round
          asm volatile("bar.arrive 1, %0;" ::"n"(kPieceThreads) : "memory");
          break;
        }
        if (warp == 1 && lane < 8 && chunk * 8 + lane < a.K) {
          float s = 0.0f;
          for (int w = 0; w < kPieceThreads / 32; ++w) s += s_dot[flip][w][lane];
          a.dweights[t * a.K + chunk * 8 + lane] = p_of_lane >= 0 ? s : 0.0f;
        }
        flip ^= 1;                                             // the other half is free: its readers passed this barrier
      }
      if (++step == per_token) { step = 0; token += gridDim.x; }
    }
    if (a.drows != nullptr) {
      long long begin = *a.n_rows;
      if (begin < 0) begin = 0;
      for (long long p = begin + blockIdx.x; p < a.N; p += gridDim.x)
        for (long long at = v * 16; at < row_bytes; at += kPieceBytes)
          *reinterpret_cast<V*>(static_cast<unsigned char*>(a.drows) + p * row_bytes + at) = V{};
    }
  }
  __syncthreads();
  if (warp == 0 && *abortp) {                                  // a role gave up: the block stays until its copies have landed
    int never = 0;
    for (int i = issued > kBulkStages ? issued - kBulkStages : 0; i < issued; ++i)
      mbar_wait_bounded(&full[i % kBulkStages], (uint32_t)(i / kBulkStages) & 1u, &never, kBulkDrainNs);
  }
}

}  // namespace zepp
