// The gate: top-k experts of each token and their weights from the router's logits, and the gradient of the weights.
//
//   softmax:  p = exp(l - max l) / sum exp(l - max l);   w_j = scale * p_{i_j},  renormalised: scale * p_{i_j} / sum_c p_{i_c}
//   sigmoid:  s = 1 / (1 + exp(-l));                     w_j = scale * s_{i_j},  renormalised: scale * s_{i_j} / (sum_c s_{i_c} + 1e-20)
//
// i_1 .. i_k are the experts with the largest logits (softmax and sigmoid are monotone, so no rounding of theirs decides
// between two experts), or with the largest s + bias where a balancing bias is given; equal values go to the lowest
// index.  A logit of -inf or NaN is never chosen; a row with fewer than k others has id -1 and weight 0 in the last
// places, and a NaN anywhere in a row makes its weights NaN.
//
// A warp owns a row and holds it in registers, so the logits are read once: element (j / 4) * 128 + lane * 4 + j % 4 for
// register j, four neighbours per access.  The (k + 1)-th largest of the 32 lanes' largest keys (order-preserving
// integers, redux.sync) is a bound that hardly more than k keys reach; those few are put together, one per lane, and each
// counts the ones before it.  That is about 20 instructions per place, where k rounds of a maximum over all registers took
// 200 (16381 rows of 384 bf16 logits with a bias: 25 us against 45 us).  A row with more than 32 keys at the bound goes
// through 64 bits: of normal logits none up to k = 14, 0.4 % with 16, 8 % with 18, 41 % with 20, 83 % with 22 and all with 28;
// and rows of equal logits.  The same 16381 rows take 23 us with k = 8, 24 with 12, 34 with 16, 75 with 20, 104 with 22
// and 140 with 32; with equal logits and k = 8, 44.
// 990 instructions a row; the schedulers issue in 65 % of their cycles, and a warp waits longest for results of fixed latency
// (31 % of its time), for the logits (14 %) and for shared memory, shuffles and reductions (12 %).
#pragma once
#include "op_common.cuh"

namespace zepp {

constexpr int kGateWarps = 4;
constexpr int kGateMaxExperts = 1024;
constexpr int kGateMaxK = 32;            // lane j of the row's warp keeps the j-th choice

struct GateArgs {
  const void* logits;     // [T, G]
  long long T;
  int G, k;
  int sigmoid, renormalize;
  const float* bias;      // [G] or nullptr
  float scale;
  int* ids;               // [T, k]
  float* weights;         // [T, k]
  // gradient
  const float* dweights;  // [T, k]
  void* dlogits;          // [T, G]
  int vec;                // rows can be accessed four elements at a time
};

__device__ __forceinline__ unsigned gate_key(float v) {      // larger key <=> larger value; 0: not to be chosen
  v += 0.0f;                                                 // -0 and +0 are equal
  const unsigned b = __float_as_uint(v);
  return v > -INFINITY ? ((b >> 31) ? ~b : (b | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float gate_value(unsigned key) {
  return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}
// The element that register j of a lane holds: four neighbours, 128 elements further the next four.  Up to 64 experts
// (NPL = 4) the lanes take every 32nd element instead, so that each has some.
template <int NPL>
__device__ __forceinline__ int gate_index(int G, int lane, int j) {
  if (NPL == 4 && G <= 64) return j * 32 + lane;
  return (j >> 2) * 128 + lane * 4 + (j & 3);
}

template <typename T, int NPL>
__device__ __forceinline__ void gate_load(const T* row, int G, int lane, bool vec, float (&v)[NPL], float fill) {
  if (vec && G > 64) {
#pragma unroll
    for (int q = 0; q < NPL / 4; ++q) {
      const int i = gate_index<NPL>(G, lane, 4 * q);
      Pack<T, 4> p;
      if (i < G) p = *reinterpret_cast<const Pack<T, 4>*>(row + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = i < G ? to_f32<T>(p.v[e]) : fill;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int i = gate_index<NPL>(G, lane, j);
      v[j] = i < G ? to_f32<T>(row[i]) : fill;
    }
  }
}

__device__ __forceinline__ float sigmoid_f32(float l) { return 1.0f / (1.0f + expf(-l)); }

// 1 / (1 + exp(-l)) + bias in 64 bits
__device__ __noinline__ double gate_score_f64(float l, float bias) { return 1.0 / (1.0 + exp(-(double)l)) + (double)bias; }

// The choice by the scores in 64 bits, straight from the row: for rows with too many equal values to sort them in one warp.
// Lane j < k returns its choice, -1 where none is left.
template <typename T, int NPL>
__device__ __noinline__ int gate_choose_f64(const T* row, const float* bias, int G, int k, int lane) {
  double key[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int i = gate_index<NPL>(G, lane, j);
    key[j] = -INFINITY;
    if (i < G) {
      const float l = to_f32<T>(row[i]);
      if (l > -INFINITY) {
        const double v = bias != nullptr ? gate_score_f64(l, bias[i]) : (double)l;
        if (v > -INFINITY) key[j] = v;                 // false for NaN
      }
    }
  }
  int mine = -1;
  for (int r = 0; r < k; ++r) {
    double best = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (key[j] > best) { best = key[j]; at = gate_index<NPL>(G, lane, j); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oa = __shfl_xor_sync(0xffffffffu, at, o);
      if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
    }
    if (!(best > -INFINITY)) break;
    if (lane == r) mine = at;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (gate_index<NPL>(G, lane, j) == at) key[j] = -INFINITY;
  }
  return mine;
}

template <typename T, int NPL>
__global__ void __launch_bounds__(32 * kGateWarps) gate_kernel(const GateArgs a) {
  __shared__ uint2 s_cand[kGateWarps][32];           // (key, index) of the row's candidates
  __shared__ uint2 s_order[kGateWarps][34];          // the first k + 1 of them in order
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int G = a.G;
  const long long row = (long long)blockIdx.x * kGateWarps + warp;
  if (row >= a.T) return;
  const T* src = static_cast<const T*>(a.logits) + row * a.G;
  float l[NPL];
  gate_load<T, NPL>(src, a.G, lane, a.vec, l, -INFINITY);
  unsigned key[NPL];
  unsigned best = 0;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    nan |= l[j] != l[j];
    float v = l[j];
    if (a.bias != nullptr) {
      const int i = gate_index<NPL>(G, lane, j);
      v = l[j] > -INFINITY ? __fdividef(1.0f, 1.0f + __expf(-l[j])) + a.bias[i < a.G ? i : 0] : -INFINITY;
    }
    key[j] = gate_key(v);
    best = max(best, key[j]);
  }
  nan = __any_sync(0xffffffffu, nan);

  // A bound that at least k + 1 keys reach (if the row has so many): the (k + 1)-th largest of the lanes' largest keys.
  // Equal ones leave together, which only lowers it.
  const unsigned top = __reduce_max_sync(0xffffffffu, best);
  unsigned bound = top;
  for (int r = 0; r < a.k; ++r) {
    if (best == bound) best = 0;
    bound = __reduce_max_sync(0xffffffffu, best);
  }
  if (bound == 0) bound = 1;                         // fewer lanes than that: every key that can be chosen
  // A 32-bit score is off by at most 1.6e-6 s (1 - s) <= 4e-7 for the exponential (its argument is rounded, |l| <= 16 where
  // s (1 - s) matters), 1.2e-7 for the quotient and half a step of s + bias: two of them may be in the wrong order where
  // they are less than `slack` apart.  What is that little below the bound is a candidate too.
  auto slack = [](float v) { return 2e-6f + 2.4e-7f * fabsf(v); };
  if (a.bias != nullptr && bound > 1) {
    const float v = gate_value(bound);
    bound = max(gate_key(v - slack(v)), 1u);
  }
  int cnt = 0;
#pragma unroll
  for (int j = 0; j < NPL; ++j) cnt += key[j] >= bound ? 1 : 0;
  int at = cnt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += u;
  }
  const int n = __shfl_sync(0xffffffffu, at, 31);
  int mine = -1;                                     // lane j < k: the j-th choice
  bool again = n > 32;
  if (!again) {
    at -= cnt;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (key[j] >= bound) s_cand[warp][at++] = make_uint2(key[j], (unsigned)gate_index<NPL>(G, lane, j));
    if (lane < a.k + 1) s_order[warp][lane] = make_uint2(0u, 0xffffffffu);
    if (lane == 0) s_order[warp][a.k] = make_uint2(0u, 0xffffffffu);
    __syncwarp();
    const uint2 me = s_cand[warp][lane];             // beyond n: never used
    int rank = 0;
    for (int c = 0; c < n; ++c) {
      const uint2 o = s_cand[warp][c];
      rank += o.x > me.x || (o.x == me.x && o.y < me.y) ? 1 : 0;
    }
    if (lane < n && rank <= a.k) s_order[warp][rank] = me;
    __syncwarp();
    const uint2 chosen = s_order[warp][lane < a.k ? lane : a.k];
    if (lane < a.k) mine = (int)chosen.y;
    if (a.bias != nullptr) {
      const uint2 next = s_order[warp][lane < a.k ? lane + 1 : a.k];
      const float v = gate_value(chosen.x);
      if (__any_sync(0xffffffffu, lane < a.k && next.x != 0u && v - gate_value(next.x) <= slack(v))) {
        // in doubt: the candidates once more, by their scores in 64 bits
        const bool real = lane < n;
        const double score = real ? gate_score_f64(to_f32<T>(src[me.y]), a.bias[me.y]) : 0.0;
        rank = 0;
        for (int c = 0; c < n; ++c) {
          const double o = __shfl_sync(0xffffffffu, score, c);
          const unsigned i = __shfl_sync(0xffffffffu, me.y, c);
          rank += o > score || (o == score && i < me.y) ? 1 : 0;
        }
        __syncwarp();
        if (real && rank < a.k) s_order[warp][rank] = me;
        __syncwarp();
        if (lane < a.k) mine = (int)s_order[warp][lane].y;
      }
    }
  }
  if (again) mine = gate_choose_f64<T, NPL>(src, a.bias, a.G, a.k, lane);

  const float lc = mine >= 0 ? to_f32<T>(src[mine]) : 0.0f;
  float w = 0.0f;
  if (a.sigmoid) {
    w = mine >= 0 ? sigmoid_f32(lc) : 0.0f;
    if (a.renormalize) w /= warp_sum(w) + 1e-20f;
  } else {
    const float mx = top ? gate_value(top) : 0.0f;           // NaN is left out of it: the row is marked below
    w = mine >= 0 ? expf(lc - mx) : 0.0f;
    float sum;
    if (a.renormalize) {
      sum = warp_sum(w);
    } else {
      sum = 0.0f;                  // __expf is off by units of 2 + 1.16 |x|: the more, the less the summand counts
#pragma unroll
      for (int j = 0; j < NPL; ++j) sum += __expf(l[j] - mx);
      sum = warp_sum(sum);
    }
    if (mine >= 0) w /= sum;
  }
  w *= a.scale;
  if (nan) w = __int_as_float(0x7fffffff);
  if (lane < a.k) {
    a.ids[row * a.k + lane] = mine;
    a.weights[row * a.k + lane] = w;
  }
}

// With q_c = scale * dw_c of the chosen experts c:
//   softmax, all experts:   dl_g = p_g * (q_g [g chosen] - sum_c q_c p_c)
//   renormalised, t = sum_c v_c, v = p or s:  dv_c = (q_c - sum_e q_e v_e / t) / t;  dl_c = dv_c v_c (softmax), dv_c s_c (1 - s_c)
//   sigmoid, not renormalised:  dl_c = q_c s_c (1 - s_c)
// Only the first has a value for every expert; the others write zeros there and read the chosen logits alone.  Measured:
// 16381 x 384 bf16, sigmoid, 8.8 us (the bytes take 2.1); 8192 x 128 fp32, softmax over all, 6.3 us (1.3).
template <typename T, int NPL>
__global__ void __launch_bounds__(32 * kGateWarps) gate_grad_kernel(const GateArgs a) {
  extern __shared__ __align__(16) unsigned char gate_rows[];       // kGateWarps rows of G elements, 16-byte multiples
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int G = a.G;
  const long long row = (long long)blockIdx.x * kGateWarps + warp;
  if (row >= a.T) return;
  const T* src = static_cast<const T*>(a.logits) + row * a.G;
  T* dst = static_cast<T*>(a.dlogits) + row * a.G;
  int id = -1;
  float q = 0.0f, w = 0.0f;
  if (lane < a.k) {
    id = a.ids[row * a.k + lane];
    w = a.weights[row * a.k + lane];
    if (id >= a.G) id = -1;
    if (id >= 0) q = a.scale * a.dweights[row * a.k + lane];
  }
  const float lc = id >= 0 ? to_f32<T>(src[id]) : -INFINITY;
  float mine;                                                     // dl of this lane's chosen expert
  float p[NPL];
  if (!a.sigmoid && !a.renormalize) {
    gate_load<T, NPL>(src, a.G, lane, a.vec, p, -INFINITY);
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) mx = fmaxf(mx, p[j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx == -INFINITY) mx = 0.0f;                               // every expert masked: exp(-inf) = 0 below
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) { p[j] = expf(p[j] - mx); sum += p[j]; }
    sum = warp_sum(sum);
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    const float pc = id >= 0 ? expf(lc - mx) * inv : 0.0f;
    const float dot = warp_sum(q * pc);
#pragma unroll
    for (int j = 0; j < NPL; ++j) p[j] *= -inv * dot;
    mine = pc * (q - dot);
  } else {
    float v, slope;
    if (a.sigmoid) {
      v = id >= 0 ? sigmoid_f32(lc) : 0.0f;
      slope = id >= 0 ? v * sigmoid_f32(-lc) : 0.0f;
    } else {
      float mx = lc;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      v = id >= 0 ? expf(lc - mx) : 0.0f;
      slope = v;
    }
    float d = q;
    if (a.renormalize) {
      const float t = warp_sum(v) + (a.sigmoid ? 1e-20f : 0.0f);
      const float dot = warp_sum(q * v);
      if (t > 0.0f) d = (q - dot / t) / t;
    }
    mine = id >= 0 ? d * slope : 0.0f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) p[j] = 0.0f;
  }
  if (w != w) mine = w;                                           // a row that held NaN
  // the row is put together in shared memory, so that it leaves in whole vectors with the chosen values in their places
  T* st = reinterpret_cast<T*>(gate_rows) + (size_t)warp * ((a.G + 7) / 8 * 8);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int i = gate_index<NPL>(G, lane, j);
    if (i < a.G) st[i] = from_f32<T>(p[j]);
  }
  __syncwarp();
  if (id >= 0) st[id] = from_f32<T>(mine);
  __syncwarp();
  if (a.vec) {
    for (int i = lane * 4; i < a.G; i += 128)
      *reinterpret_cast<Pack<T, 4>*>(dst + i) = *reinterpret_cast<const Pack<T, 4>*>(st + i);
  } else {
    for (int i = lane; i < a.G; i += 32) dst[i] = st[i];
  }
}

}  // namespace zepp
