// The 2-norm over all elements of many tensors, and their scaling to a largest norm:
//
//   n = sqrt(sum x^2),   x <- round(x * c),   c = min(1, max_norm / (n + 1e-6))
//
// Two launches: every block sums its chunks' squares into one 64-bit partial; every block of the second launch adds the
// partials in the same fixed order (so all blocks agree on n, and equal inputs give equal bits) and scales its chunks,
// last chunk first, while the end of what the first launch read is still in L2.  Bound by HBM: one read, and one read and
// one write where the norm is over the limit; with c = 1 nothing is touched.  Inside a chunk a thread adds at most
// 64 squares in 32 bits, then carries on in 64; a chunk sum that left the range in which that is exact enough (values
// beyond 1e19 or below 1e-16) is formed again in 64 bits.  Measured on 604 M bf16 elements: norm 175 us (6.9 TB/s), scaling
// 405 us (6.0 TB/s).
#pragma once
#include "op_common.cuh"

namespace zepp {

constexpr int kNormThreads = 256;
constexpr int kNormVecs = 8;                                   // 16-byte vectors a thread has in flight
constexpr int kNormChunkBytes = kNormThreads * kNormVecs * 16;  // 32 KB
constexpr int kNormMaxBlocks = 148 * 8;

// A tensor's elements as 16-byte vectors from the vector that holds its first element: `head` elements of that one
// lie before it.  The table travels as a kernel argument (it lives in the constant bank; nothing has to outlive the call).
template <int CAP>
struct NormTable {
  unsigned long long base[CAP];    // address of the first vector
  long long end[CAP];              // head + number of elements
  int chunk0[CAP + 1];             // chunks before the tensor
  unsigned char head[CAP], type[CAP];
  int count;
};

// this thread's vectors of chunk `c` of a tensor; elements outside it read as zero
template <typename T>
__device__ __forceinline__ void norm_load(const T* base, long long head, long long end, long long first, uint4 (&v)[kNormVecs]) {
  constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
  for (int q = 0; q < kNormVecs; ++q) {
    const long long e0 = first + (long long)(q * kNormThreads + threadIdx.x) * E;
    if (e0 >= head && e0 + E <= end) {
      v[q] = *reinterpret_cast<const uint4*>(base + e0);
    } else {
      v[q] = make_uint4(0u, 0u, 0u, 0u);
      T* e = reinterpret_cast<T*>(&v[q]);
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (e0 + i >= head && e0 + i < end) e[i] = base[e0 + i];
    }
  }
}

// this thread's elements of a chunk once more, in 64 bits
template <typename T>
__device__ __noinline__ double norm_chunk_wide(const T* base, long long head, long long end, long long first) {
  constexpr int E = 16 / (int)sizeof(T);
  double s = 0.0;
  for (int q = 0; q < kNormVecs; ++q) {
    const long long e0 = first + (long long)(q * kNormThreads + threadIdx.x) * E;
    for (int i = 0; i < E; ++i)
      if (e0 + i >= head && e0 + i < end) {
        const double x = (double)to_f32<T>(base[e0 + i]);
        s = fma(x, x, s);
      }
  }
  return s;
}

template <typename T>
__device__ __forceinline__ double norm_chunk_sum(const T* base, long long head, long long end, long long first) {
  constexpr int E = 16 / (int)sizeof(T);
  uint4 v[kNormVecs];
  norm_load<T>(base, head, end, first, v);
  float s = 0.0f;
  unsigned any = 0;
#pragma unroll
  for (int q = 0; q < kNormVecs; ++q) {
    const T* e = reinterpret_cast<const T*>(&v[q]);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) { const float x = to_f32<T>(e[i]); sq = fmaf(x, x, sq); }
    s += sq;
    any |= v[q].x | v[q].y | v[q].z | v[q].w;
  }
  if (any != 0u && !(s > 1e-30f && s < INFINITY)) return norm_chunk_wide<T>(base, head, end, first);
  return (double)s;
}

template <typename T>
__device__ __forceinline__ void norm_scale(T* base, long long head, long long end, long long first, float c) {
  constexpr int E = 16 / (int)sizeof(T);
  uint4 v[kNormVecs];
  norm_load<T>(base, head, end, first, v);
#pragma unroll
  for (int q = 0; q < kNormVecs; ++q) {
    const long long e0 = first + (long long)(q * kNormThreads + threadIdx.x) * E;
    T* e = reinterpret_cast<T*>(&v[q]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = from_f32<T>(to_f32<T>(e[i]) * c);
    if (e0 >= head && e0 + E <= end) {
      *reinterpret_cast<uint4*>(base + e0) = v[q];
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (e0 + i >= head && e0 + i < end) base[e0 + i] = e[i];
    }
  }
}

// The same with a factor below the normal numbers of fp32 (a norm beyond 1e38 of the limit), which would hold fewer bits of it
// the smaller it is.
template <typename T>
__device__ __noinline__ void norm_scale_wide(T* base, long long head, long long end, long long first, double c) {
  constexpr int E = 16 / (int)sizeof(T);
  for (int q = 0; q < kNormVecs; ++q) {
    const long long e0 = first + (long long)(q * kNormThreads + threadIdx.x) * E;
    for (int i = 0; i < E; ++i)
      if (e0 + i >= head && e0 + i < end) base[e0 + i] = from_f32<T>((float)((double)to_f32<T>(base[e0 + i]) * c));
  }
}

template <int CAP>
__device__ __forceinline__ int norm_tensor_of(const NormTable<CAP>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk0[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// sum over the block, valid in every thread
__device__ __forceinline__ double norm_block_sum(double v) {
  __shared__ double part[kNormThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kNormThreads / 32; ++i) s += part[i];
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(kNormThreads) norm_partials_kernel(const __grid_constant__ NormTable<CAP> t, double* partials) {
  double sum = 0.0;
  for (int c = blockIdx.x; c < t.chunk0[t.count]; c += gridDim.x) {
    const int k = norm_tensor_of(t, c);
    const long long bytes = (long long)(c - t.chunk0[k]) * kNormChunkBytes;
    if (t.type[k] == OP_F32)
      sum += norm_chunk_sum<float>(reinterpret_cast<const float*>(t.base[k]), t.head[k], t.end[k], bytes / 4);
    else if (t.type[k] == OP_BF16)
      sum += norm_chunk_sum<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(t.base[k]), t.head[k], t.end[k], bytes / 2);
    else
      sum += norm_chunk_sum<__half>(reinterpret_cast<const __half*>(t.base[k]), t.head[k], t.end[k], bytes / 2);
  }
  sum = norm_block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_total(const double* partials, int n) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kNormThreads) v += partials[i];
  return sqrt(norm_block_sum(v));
}

__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(const double* partials, int n, float* out) {
  const double total = norm_total(partials, n);
  if (threadIdx.x == 0) *out = (float)total;
}

template <int CAP>
__global__ void __launch_bounds__(kNormThreads)
norm_scale_kernel(const __grid_constant__ NormTable<CAP> t, const double* partials, int n, double max_norm, float* out) {
  const double total = norm_total(partials, n);
  if (blockIdx.x == 0 && threadIdx.x == 0 && out != nullptr) *out = (float)total;
  // without a limit nothing changes, elements that are infinite neither
  const double ratio = max_norm == INFINITY && total == INFINITY ? 1.0 : max_norm / (total + 1e-6);
  const float c = (float)(ratio > 1.0 ? 1.0 : ratio);      // NaN stays NaN
  if (c == 1.0f) return;
  if (ratio > 0.0 && ratio < 1.17549435e-38) {
    for (int i = blockIdx.x; i < t.chunk0[t.count]; i += gridDim.x) {
      const int k = norm_tensor_of(t, i);
      const long long bytes = (long long)(i - t.chunk0[k]) * kNormChunkBytes;
      if (t.type[k] == OP_F32)
        norm_scale_wide<float>(reinterpret_cast<float*>(t.base[k]), t.head[k], t.end[k], bytes / 4, ratio);
      else if (t.type[k] == OP_BF16)
        norm_scale_wide<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(t.base[k]), t.head[k], t.end[k], bytes / 2, ratio);
      else
        norm_scale_wide<__half>(reinterpret_cast<__half*>(t.base[k]), t.head[k], t.end[k], bytes / 2, ratio);
    }
    return;
  }
  for (int i = blockIdx.x; i < t.chunk0[t.count]; i += gridDim.x) {
    const int chunk = t.chunk0[t.count] - 1 - i;
    const int k = norm_tensor_of(t, chunk);
    const long long bytes = (long long)(chunk - t.chunk0[k]) * kNormChunkBytes;
    if (t.type[k] == OP_F32)
      norm_scale<float>(reinterpret_cast<float*>(t.base[k]), t.head[k], t.end[k], bytes / 4, c);
    else if (t.type[k] == OP_BF16)
      norm_scale<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(t.base[k]), t.head[k], t.end[k], bytes / 2, c);
    else
      norm_scale<__half>(reinterpret_cast<__half*>(t.base[k]), t.head[k], t.end[k], bytes / 2, c);
  }
}

}  // namespace zepp
