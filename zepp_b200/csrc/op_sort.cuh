// Token rows sorted by expert and back.
//
//   sort:    copy i = t * K + k of a token goes to row  position[i] = offsets[g] + #{j < i : group(j) = g},  g = group(i);
//            rows[position[i]] = x[t];   offsets[g] = #{j : group(j) < g}.  Copies without a group have position -1.
//   unsort:  y[t] = sum_k w[t, k] * rows[position[t, k]]         (without weights: the gradient of the sort)
//   its gradient:  drows[position[t, k]] = w[t, k] * dy[t],   dw[t, k] = <dy[t], rows[position[t, k]]>
//
// The order is that of a stable sort by group, and every sum runs over k in order, so equal inputs give equal bits.
// Everything is bound by the bytes of the rows: the sort reads a row once and writes its K copies, the gradient of the
// unsort reads dy once and makes both of its results from one pass over the rows.
#pragma once
#include "op_common.cuh"

namespace zepp {

constexpr int kSortThreads = 512;
constexpr int kSortMaxGroups = 2048;
constexpr int kSortDirect = 8192;       // up to this many copies every block counts all of them itself: one launch
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
    // the rows: 32 neighbouring vectors of a token per warp and step
    const int lines = (int)((vecs + 31) / 32);
    for (int u = warp; u < tokens * lines; u += kSortThreads / 32) {
      const int t = u / lines;
      const int v = (u - t * lines) * 32 + lane;
      if (v < vecs) {
        const V val = reinterpret_cast<const V*>(a.x + (tb + t) * a.row_bytes)[v];
        for (int k = 0; k < a.K; ++k) {
          const int p = s_pos[t * a.K + k];
          if (p >= 0) reinterpret_cast<V*>(a.rows + (long long)p * a.row_bytes)[v] = val;
        }
      }
    }
    __syncthreads();
  }
  // rows behind the last group hold zeros
  for (long long p = carry + (long long)blockIdx.x; p < n; p += gridDim.x)
    for (long long v = tid; v < vecs; v += kSortThreads) reinterpret_cast<V*>(a.rows + p * a.row_bytes)[v] = V{};
}

constexpr int kUnsortThreads = 256;

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

// E elements of a row per thread and step; blockIdx.x = token, blockIdx.y = part of the row
template <typename T, int E>
__global__ void __launch_bounds__(kUnsortThreads) unsort_kernel(const UnsortArgs a) {
  typedef Pack<T, E> V;
  const long long t = blockIdx.x;
  const long long vecs = a.H / E;
  const long long v = (long long)blockIdx.y * kUnsortThreads + threadIdx.x;
  if (v >= vecs) return;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int k0 = 0; k0 < a.K; k0 += 4) {                  // four rows in flight
    V r[4];
    float w[4];
    bool there[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = k0 + q;
      const int p = k < a.K ? unsort_position(a, t * a.K + k) : -1;
      there[q] = p >= 0;
      if (there[q]) {
        w[q] = a.weights != nullptr ? a.weights[t * a.K + k] : 1.0f;
        r[q] = reinterpret_cast<const V*>(static_cast<const T*>(a.rows) + (long long)p * a.H)[v];
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (there[q]) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w[q], to_f32<T>(r[q].v[e]), acc[e]);
      }
  }
  V out;
#pragma unroll
  for (int e = 0; e < E; ++e) out.v[e] = from_f32<T>(acc[e]);
  reinterpret_cast<V*>(static_cast<T*>(a.y) + t * a.H)[v] = out;
}

// a block owns a token: dy is read once for eight copies, each row once
template <typename T, int E>
__global__ void __launch_bounds__(kUnsortThreads) unsort_grad_kernel(const UnsortArgs a) {
  typedef Pack<T, E> V;
  constexpr int KB = 8;
  __shared__ float s_dot[kUnsortThreads / 32][KB];
  const long long vecs = a.H / E;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x) {
    const V* dy = reinterpret_cast<const V*>(static_cast<const T*>(a.dy) + t * a.H);
    for (int k0 = 0; k0 < a.K; k0 += KB) {
      int p[KB];
      float w[KB], dot[KB];
#pragma unroll
      for (int q = 0; q < KB; ++q) {
        const int k = k0 + q;
        p[q] = k < a.K ? unsort_position(a, t * a.K + k) : -1;
        w[q] = p[q] >= 0 && a.weights != nullptr ? a.weights[t * a.K + k] : 1.0f;
        dot[q] = 0.0f;
      }
      for (long long v = tid; v < vecs; v += blockDim.x) {
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
#pragma unroll
        for (int q = 0; q < KB; ++q) {
          const float s = warp_sum(dot[q]);
          if (lane == 0) s_dot[warp][q] = s;
        }
        __syncthreads();
        if (tid < KB && k0 + tid < a.K) {
          float s = 0.0f;
          for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += s_dot[i][tid];
          a.dweights[t * a.K + k0 + tid] = unsort_position(a, t * a.K + k0 + tid) >= 0 ? s : 0.0f;
        }
        __syncthreads();
      }
    }
  }
  if (a.drows != nullptr) {
    long long first = *a.n_rows;
    if (first < 0) first = 0;
    for (long long p = first + blockIdx.x; p < a.N; p += gridDim.x)
      for (long long v = tid; v < vecs; v += blockDim.x) reinterpret_cast<V*>(static_cast<T*>(a.drows) + p * a.H)[v] = V{};
  }
}

}  // namespace zepp
