// Host side of the operators around the layer (zepp_op_* in include/zepp_b200.h): checks, tensor maps and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <initializer_list>
#include <mutex>

#include "../../include/zepp_b200.h"
#include "host.cuh"
#include "op_ffn.cuh"
#include "op_gate.cuh"
#include "op_norm.cuh"
#include "op_sort.cuh"

using namespace zepp;

#define OP_LAUNCHED()                                                                                      \
  do {                                                                                                     \
    cudaError_t _e = cudaGetLastError();                                                                   \
    if (_e != cudaSuccess) return fail("kernel launch failed: %s (%s:%d)", cudaGetErrorString(_e), __FILE__, __LINE__); \
  } while (0)

// status words of the operators' bounded waits, one block per device that loads the library
__device__ unsigned long long g_op_status[ST_WORDS];
// how long each of them waits (zepp_op_set_wait_limit_ns)
std::atomic<unsigned long long> g_op_wait_ns{2000000000ull};

namespace {

constexpr int kMaxDevices = 64;
struct OpDevice {
  bool ready = false;
  int sms = 0;
  unsigned long long* status = nullptr;
};
OpDevice g_dev[kMaxDevices];
std::mutex g_dev_mutex;

// dynamic shared memory of the products: tables of G groups (behind at most 512 bytes of static shared memory), stages on
// 1024-byte boundaries, staging of the epilogue warps
size_t ffn_smem_bytes(int G, int stages) {
  return (512 + 2 * sizeof(int) * (size_t)(G + 1) + 1023) / 1024 * 1024 + (size_t)stages * kFfnStageBytes + kFfnEpiWarps * kFfnStagingBytes;
}
constexpr int kFfnSmemLimit = 227 * 1024 - 512;

template <int MODE>
cudaError_t ffn_smem() {
  return cudaFuncSetAttribute(ffn_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFfnSmemLimit);
}

template <typename T>
cudaError_t bulk_smem() {
  return cudaFuncSetAttribute(unsort_grad_bulk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkStages * kBulkStageBytes);
}

// the current device's record; its first use sets kernel attributes and looks up the status block
int op_device(OpDevice** out) {
  int dev = 0;
  CU_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail("device ordinal %d out of range", dev);
  // binds the device's context to the calling thread: a thread that has made no launch yet (autograd's) has none, and the
  // driver's tensor-map encoder does not look for one
  CU_OK(cudaSetDevice(dev));
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  OpDevice& d = g_dev[dev];
  if (!d.ready) {
    int major = 0;
    CU_OK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    if (major != 10) return fail("libzepp_b200 needs an sm_100 device (found major %d)", major);
    CU_OK(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
    void* p = nullptr;
    CU_OK(cudaGetSymbolAddress(&p, g_op_status));
    d.status = static_cast<unsigned long long*>(p);
    CU_OK(ffn_smem<FFN_UP_SWIGLU>());
    CU_OK(ffn_smem<FFN_UP_GELU>());
    CU_OK(ffn_smem<FFN_DOWN>());
    CU_OK(ffn_smem<FFN_DACT_SWIGLU>());
    CU_OK(ffn_smem<FFN_DACT_GELU>());
    CU_OK(ffn_smem<FFN_DROWS>());
    CU_OK(ffn_smem<FFN_DWEIGHT>());
    CU_OK(bulk_smem<__nv_bfloat16>());
    CU_OK(bulk_smem<__half>());
    d.ready = true;
  }
  *out = &d;
  return 0;
}

int elem_bytes(int dtype) { return dtype == OP_F32 ? 4 : 2; }
// none of the pointers that a call cannot do without is null
bool given(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (p == nullptr) return false;
  return true;
}
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

extern "C" int zepp_op_set_wait_limit_ns(int64_t ns) {
  if (ns < 0 || ns > 3600000000000ll) return fail("wait limit: 0..3600 s (got %lld ns)", (long long)ns);
  g_op_wait_ns = (unsigned long long)ns;
  return 0;
}

extern "C" int zepp_op_status(void* stream, uint64_t out[8]) {
  OpDevice* d;
  if (int rc = op_device(&d)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CU_OK(cudaDeviceSynchronize());                  // kernels of every stream record into this block
  CU_OK(cudaMemcpyAsync(out, d->status, 8 * sizeof(uint64_t), cudaMemcpyDeviceToHost, s));
  CU_OK(cudaStreamSynchronize(s));
  if (out[ST_ERROR] != 0) {                        // without one, there is nothing to clear that a kernel could be writing
    CU_OK(cudaMemsetAsync(d->status, 0, 8 * sizeof(uint64_t), s));
    CU_OK(cudaStreamSynchronize(s));
  }
  return 0;
}

// ---------------------------------------------------------------------------------------------
// gate
// ---------------------------------------------------------------------------------------------
static int gate_check(const char* what, int dtype, int64_t T, int G, int k, int sigmoid) {
  if (dtype < OP_F32 || dtype > OP_F16) return fail("%s: unknown element type %d", what, dtype);
  if (T < 0 || T > (1ll << 31)) return fail("%s: %lld tokens", what, (long long)T);
  if (G < 1 || G > kGateMaxExperts) return fail("%s: 1..%d experts (got %d)", what, kGateMaxExperts, G);
  if (k < 1 || k > kGateMaxK || k > G) return fail("%s: top-k of 1..min(%d, experts) (got %d of %d)", what, kGateMaxK, k, G);
  if (sigmoid < 0 || sigmoid > 1) return fail("%s: unknown score %d", what, sigmoid);
  return 0;
}

template <typename T>
static void gate_launch(const GateArgs& a, bool grad, cudaStream_t s) {
  const dim3 grid((unsigned)((a.T + kGateWarps - 1) / kGateWarps));
  const size_t sm = grad ? (size_t)kGateWarps * ((a.G + 7) / 8 * 8) * sizeof(T) : 0;
#define GATE(NPL)                                                                             \
  do {                                                                                        \
    if (grad) gate_grad_kernel<T, NPL><<<grid, 32 * kGateWarps, sm, s>>>(a);                  \
    else gate_kernel<T, NPL><<<grid, 32 * kGateWarps, 0, s>>>(a);                             \
  } while (0)
  if (a.G <= 128) GATE(4);
  else if (a.G <= 256) GATE(8);
  else if (a.G <= 384) GATE(12);
  else if (a.G <= 512) GATE(16);
  else GATE(32);
#undef GATE
}

static int gate_run(GateArgs& a, int dtype, bool grad, void* stream) {
  if (a.T == 0) return 0;
  const size_t e = elem_bytes(dtype);
  a.vec = a.G % 4 == 0 && aligned(a.logits, 4 * e) && (!grad || aligned(a.dlogits, 4 * e));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == OP_F32) gate_launch<float>(a, grad, s);
  else if (dtype == OP_BF16) gate_launch<__nv_bfloat16>(a, grad, s);
  else gate_launch<__half>(a, grad, s);
  OP_LAUNCHED();
  return 0;
}

extern "C" int zepp_op_gate(const void* logits, int dtype, int64_t T, int G, int k, int sigmoid, int renormalize,
                            const float* bias, float scale, int32_t* ids, float* weights, void* stream) {
  if (int rc = gate_check("gate", dtype, T, G, k, sigmoid)) return rc;
  if (bias != nullptr && !sigmoid) return fail("gate: a balancing bias goes with sigmoid scores");
  if (T > 0 && !given({logits, ids, weights})) return fail("gate: null pointer");
  GateArgs a{};
  a.logits = logits; a.T = T; a.G = G; a.k = k; a.sigmoid = sigmoid; a.renormalize = renormalize; a.bias = bias; a.scale = scale;
  a.ids = ids; a.weights = weights;
  return gate_run(a, dtype, false, stream);
}

extern "C" int zepp_op_gate_grad(const void* logits, int dtype, int64_t T, int G, int k, int sigmoid, int renormalize,
                                 float scale, const int32_t* ids, const float* weights, const float* dweights,
                                 void* dlogits, void* stream) {
  if (int rc = gate_check("gate_grad", dtype, T, G, k, sigmoid)) return rc;
  if (T > 0 && !given({logits, ids, weights, dweights, dlogits})) return fail("gate_grad: null pointer");
  GateArgs a{};
  a.logits = logits; a.T = T; a.G = G; a.k = k; a.sigmoid = sigmoid; a.renormalize = renormalize; a.scale = scale;
  a.ids = const_cast<int32_t*>(ids); a.weights = const_cast<float*>(weights);
  a.dweights = dweights; a.dlogits = dlogits;
  return gate_run(a, dtype, true, stream);
}

// ---------------------------------------------------------------------------------------------
// sort by expert and back
// ---------------------------------------------------------------------------------------------
static int sort_check(const char* what, int dtype, int64_t T, int K, int64_t H) {
  if (dtype < OP_F32 || dtype > OP_F16) return fail("%s: unknown element type %d", what, dtype);
  if (K < 1 || K > 64) return fail("%s: top-k of 1..64 (got %d)", what, K);
  if (T < 0 || T >= (1ll << 31) || T * K >= (1ll << 31)) return fail("%s: %lld tokens x %d copies do not fit 32-bit row numbers", what, (long long)T, K);
  if (H < 1 || H > (1 << 20)) return fail("%s: rows of 1..%d elements (got %lld)", what, 1 << 20, (long long)H);
  return 0;
}
static int sort_chunk(int64_t n) { return n <= kSortDirect ? 0 : (int)((n + kSortChunks - 1) / kSortChunks); }

extern "C" size_t zepp_op_sort_ws_ints(int64_t T, int K, int G) {
  return sort_chunk(T * K) == 0 ? 0 : (size_t)kSortChunks * G;
}

extern "C" int zepp_op_sort(const void* x, int dtype, int64_t T, int K, int64_t H, const int32_t* ids,
                            const int32_t* group_of, int n_ids, int G, int32_t* ws, void* rows, int32_t* offsets,
                            int32_t* position, void* stream) {
  if (int rc = sort_check("sort", dtype, T, K, H)) return rc;
  if (G < 1 || G > kSortMaxGroups) return fail("sort: 1..%d experts (got %d)", kSortMaxGroups, G);
  if (offsets == nullptr || (T > 0 && !given({x, ids, rows, position}))) return fail("sort: null pointer");
  OpDevice* d;
  if (int rc = op_device(&d)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  SortArgs a{};
  a.ids = ids; a.group_of = group_of; a.n_ids = group_of != nullptr ? n_ids : G; a.G = G; a.T = T; a.K = K;
  a.x = static_cast<const unsigned char*>(x); a.rows = static_cast<unsigned char*>(rows); a.row_bytes = H * elem_bytes(dtype);
  a.offsets = offsets; a.position = position;
  a.chunk = sort_chunk(T * K);
  a.counts = ws;
  int chunks = 0;
  if (a.chunk > 0) {
    if (ws == nullptr) return fail("sort: %lld copies need a workspace", (long long)(T * K));
    chunks = (int)((T * K + a.chunk - 1) / a.chunk);
    sort_count_kernel<<<chunks, kSortThreads, G * sizeof(int), s>>>(a, ws);
    OP_LAUNCHED();
  }
  const int64_t most = 2ll * d->sms;       // two blocks of 512 threads fill an SM's copy bandwidth
  const int64_t blocks = T < 1 ? 1 : (T < most ? T : most);
  a.tokens_per_block = (int)((T + blocks - 1) / blocks);
  const size_t sm = 2 * (size_t)G * sizeof(int);
  if (a.row_bytes % 16 == 0 && aligned(x, 16) && aligned(rows, 16))
    sort_rows_kernel<uint4><<<(unsigned)blocks, kSortThreads, sm, s>>>(a, chunks);
  else if (a.row_bytes % 4 == 0 && aligned(x, 4) && aligned(rows, 4))
    sort_rows_kernel<uint32_t><<<(unsigned)blocks, kSortThreads, sm, s>>>(a, chunks);
  else
    sort_rows_kernel<uint16_t><<<(unsigned)blocks, kSortThreads, sm, s>>>(a, chunks);
  OP_LAUNCHED();
  return 0;
}

template <typename T, int E>
static void unsort_launch(const UnsortArgs& a, bool grad, int sms, cudaStream_t s) {
  const long long vecs = a.H / E;
  if (grad) {
    // A warp per token once that fills the machine (16 warps on every SM) and rows have up to eight vectors for a lane; else
    // as many as a block has, as long as each has a vector for every lane.  Rows of 28 KB fp32 (2368 tokens x 8 copies), 4
    // warps against 1: 183 us against 200, and the weights' gradient is off by 1.5e-7 of its norm against 2.8e-7, because
    // fewer products are added one after the other; of 4012 bytes (1531 x 6): 30 us against 34; with one or two copies
    // of 8 KB it is 3 to 6 % slower.
    int wpt = 1;
    while (wpt < kUnsortGradThreads / 32 && vecs > 32 * wpt && (a.T * wpt < 16ll * sms || vecs > 256 * wpt)) wpt *= 2;
    const long long tokens = kUnsortGradThreads / 32 / wpt;
    const long long blocks = (a.T + tokens - 1) / tokens;
    unsort_grad_kernel<T, E><<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), kUnsortGradThreads, 0, s>>>(a, wpt);
  } else if (E > 1) {
    const dim3 grid((unsigned)a.T, (unsigned)((vecs + kUnsortThreads - 1) / kUnsortThreads));
    unsort_kernel<T, E, 1, 4><<<grid, kUnsortThreads, 0, s>>>(a);
  } else {       // single elements: four per thread and row
    const dim3 grid((unsigned)a.T, (unsigned)((vecs + 4 * kUnsortThreads - 1) / (4 * kUnsortThreads)));
    unsort_kernel<T, E, E == 1 ? 4 : 1, 8><<<grid, kUnsortThreads, 0, s>>>(a);
  }
}
// The gradient through the ring of shared-memory stages, where that is faster.  Measured against the kernel above, which it
// replaces then (us, 128 experts, T tokens x 8 copies, rows from HBM):
//   bf16, rows of 2 KB:  T 592 10.4 / 10.2, T 9472 100 / 80        of 4 KB:  T 592 12.5 / 15.9, T 9472 110 / 150
//         rows of 8 KB:  T 148 8.5 / 12.3 (one copy, T 300: 8.0 / 7.2), T 592 19.8 / 26.3, T 9472 243 / 282
//   fp32, rows of 4 KB:  T 592 11.5 / 9.7, T 9472 128 / 109        of 8 KB:  T 592 18.8 / 16.6, T 9472 239 / 214
// (half as many elements in the same bytes: nothing is left to win).  Without the weights' gradient the two are within 15 %.
template <typename T>
static bool unsort_grad_bulk(const UnsortArgs& a, const OpDevice* d, cudaStream_t s) {
  const long long row_bytes = a.H * (long long)sizeof(T);
  if (row_bytes < kPieceBytes || a.T < 4ll * d->sms) return false;
  BulkArgs b{};
  b.u = a;
  b.pieces = (int)((row_bytes + kPieceBytes - 1) / kPieceBytes);
  b.chunks = (a.K + 7) / 8;
  b.status = d->status;
  b.limit_ns = g_op_wait_ns;
  unsort_grad_bulk_kernel<T><<<d->sms, kBulkThreads, kBulkStages * kBulkStageBytes, s>>>(b);
  return true;
}
template <typename T>
static void unsort_type(const UnsortArgs& a, bool grad, const OpDevice* d, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool wide = a.H % E == 0 && aligned(a.rows, 16) && aligned(a.y, 16) && aligned(a.dy, 16) && aligned(a.drows, 16);
  if constexpr (sizeof(T) == 2)
    if (wide && grad && unsort_grad_bulk<T>(a, d, s)) return;
  if (wide) unsort_launch<T, E>(a, grad, d->sms, s);
  else unsort_launch<T, 1>(a, grad, d->sms, s);
}
static int unsort_run(const UnsortArgs& a, int dtype, bool grad, void* stream) {
  OpDevice* d;
  if (int rc = op_device(&d)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == OP_F32) unsort_type<float>(a, grad, d, s);
  else if (dtype == OP_BF16) unsort_type<__nv_bfloat16>(a, grad, d, s);
  else unsort_type<__half>(a, grad, d, s);
  OP_LAUNCHED();
  return 0;
}

extern "C" int zepp_op_unsort(const void* rows, int dtype, int64_t T, int K, int64_t H, const int32_t* position,
                              const float* weights, void* y, void* stream) {
  if (int rc = sort_check("unsort", dtype, T, K, H)) return rc;
  if (T == 0) return 0;
  if (!given({rows, position, y})) return fail("unsort: null pointer");
  UnsortArgs a{};
  a.rows = rows; a.T = T; a.N = T * K; a.K = K; a.H = H; a.position = position; a.weights = weights; a.y = y;
  return unsort_run(a, dtype, false, stream);
}

extern "C" int zepp_op_unsort_grad(const void* dy, const void* rows, int dtype, int64_t T, int K, int64_t H, int G,
                                   const int32_t* offsets, const int32_t* position, const float* weights, void* drows,
                                   float* dweights, void* stream) {
  if (int rc = sort_check("unsort_grad", dtype, T, K, H)) return rc;
  if (G < 1) return fail("unsort_grad: no experts");
  if (T == 0 || (drows == nullptr && dweights == nullptr)) return 0;
  if (!given({dy, offsets, position})) return fail("unsort_grad: null pointer");
  if (dweights != nullptr && rows == nullptr) return fail("unsort_grad: the weights' gradient needs the rows");
  UnsortArgs a{};
  a.dy = dy; a.rows = rows; a.T = T; a.N = T * K; a.K = K; a.H = H; a.position = position; a.weights = weights;
  a.drows = drows; a.dweights = dweights; a.n_rows = offsets + G;
  return unsort_run(a, dtype, true, stream);
}

// ---------------------------------------------------------------------------------------------
// the experts' products
// ---------------------------------------------------------------------------------------------
// bf16 [outer, rows, cols] (row-major, outer = 1: two dimensions), box of 64 columns x box_rows, 128-byte swizzle, zeros outside
static int ffn_map(CUtensorMap* m, const void* base, uint64_t cols, uint64_t rows, uint64_t outer, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail("cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {cols, rows, outer};
  cuuint64_t strides[2] = {cols * 2, cols * rows * 2};
  cuuint32_t box[3] = {64, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, outer > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail("cuTensorMapEncodeTiled failed with %d (%llu x %llu x %llu, box %u)", (int)r, (unsigned long long)outer,
                (unsigned long long)rows, (unsigned long long)cols, box_rows);
  return 0;
}

struct FfnCall {
  const int32_t* offsets;
  int64_t n;
  int G, H, I, act;            // act: 0 gelu, 1 swiglu, as in zepp_layer_cfg
  OpDevice* dev;
  cudaStream_t stream;
  int f1() const { return act ? 2 * I : I; }
};

static int ffn_check(const char* what, int64_t n, int G, int H, int I, int act, std::initializer_list<const void*> ptrs) {
  if (act < 0 || act > 1) return fail("%s: unknown activation %d", what, act);
  if (G < 1 || G > kFfnMaxGroups) return fail("%s: 1..%d experts (got %d)", what, kFfnMaxGroups, G);
  if (H < 8 || I < 8 || H % 8 || I % 8 || H > (1 << 20) || I > (1 << 19))
    return fail("%s: hidden and ffn_hidden must be multiples of 8 (got %d, %d)", what, H, I);
  if (n < 0 || n >= (1ll << 31)) return fail("%s: %lld rows", what, (long long)n);
  const int widest = H > 2 * I ? H : 2 * I;
  if ((n / 128 + G) * (widest / 128 + 1) >= (1ll << 31) || (int64_t)G * (widest / 128 + 1) * (widest / 128 + 1) >= (1ll << 31))
    return fail("%s: too many tiles", what);
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return fail("%s: tensors must start on 16-byte boundaries", what);
  return 0;
}

// one launch of the products' kernel over at most `tiles` tiles
template <int MODE>
static int ffn_launch(const FfnCall& c, int64_t tiles, const CUtensorMap& f, const CUtensorMap& r32, const CUtensorMap& r128, FfnArgs& a) {
  a.offsets = c.offsets; a.G = c.G; a.n = c.n;
  a.stages = kFfnMaxStages;
  while (ffn_smem_bytes(c.G, a.stages) > (size_t)kFfnSmemLimit) --a.stages;      // the tables of 192 groups and more take one's place
  a.status = c.dev->status;
  a.limit_ns = g_op_wait_ns;
  const int pairs = c.dev->sms / 2;
  ffn_kernel<MODE><<<(unsigned)(tiles < pairs ? tiles : pairs) * 2, kFfnThreads, ffn_smem_bytes(c.G, a.stages), c.stream>>>(f, r32, r128, a);
  OP_LAUNCHED();
  return 0;
}

// K-major rows [n, K] times the weights [G, wr, wc]; N: features of the result (of each half, where it has two)
template <int MODE>
static int ffn_rows_launch(const FfnCall& c, const void* rows, int K, const void* w, int wr, int wc, int N, void* out, void* h) {
  constexpr bool kWhole = MODE == FFN_UP_GELU || MODE == FFN_DOWN;       // 128 weight rows in one box
  CUtensorMap r32, r128, f;
  if (int rc = ffn_map(&r32, rows, K, c.n, 0, 32)) return rc;
  if (int rc = ffn_map(&r128, rows, K, c.n, 0, 128)) return rc;
  if (int rc = ffn_map(&f, w, wc, wr, c.G, kWhole ? 128 : 64)) return rc;
  FfnArgs a{};
  a.K = K; a.N = N;
  a.feat = MODE == FFN_UP_SWIGLU ? 128 : 256;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.h = static_cast<float*>(h);
  const int64_t tiles = (c.n / kFfnRows + (c.n < c.G ? c.n : c.G)) * ((N + a.feat - 1) / a.feat);
  return ffn_launch<MODE>(c, tiles, f, r32, r128, a);
}

// dW [G, M, N] = p_e^T q_e over the rows of each expert
static int ffn_weight_launch(const FfnCall& c, const void* p, int M, const void* q, int N, void* out) {
  CUtensorMap mp, mq;
  if (int rc = ffn_map(&mp, p, M, c.n, 0, 64)) return rc;
  if (int rc = ffn_map(&mq, q, N, c.n, 0, 64)) return rc;
  FfnArgs a{};
  a.M = M; a.N = N; a.feat = 256;
  a.out = static_cast<__nv_bfloat16*>(out);
  const int64_t tiles = (int64_t)c.G * ((M + 255) / 256) * ((N + kFfnRows - 1) / kFfnRows);
  return ffn_launch<FFN_DWEIGHT>(c, tiles, mp, mq, mq, a);
}

extern "C" int zepp_op_expert_ffn(const void* rows, int64_t n, const int32_t* offsets, int G, int H, int I, int act,
                                  const void* w1, const void* w2, void* a_out, void* h_out, void* y, void* stream) {
  if (int rc = ffn_check("expert_ffn", n, G, H, I, act, {rows, w1, w2, a_out, h_out, y})) return rc;
  if (n == 0) return 0;
  if (!given({rows, offsets, w1, w2, a_out, y})) return fail("expert_ffn: null pointer");
  FfnCall c{offsets, n, G, H, I, act, nullptr, static_cast<cudaStream_t>(stream)};
  if (int rc = op_device(&c.dev)) return rc;
  if (act) {
    if (int rc = ffn_rows_launch<FFN_UP_SWIGLU>(c, rows, H, w1, 2 * I, H, I, a_out, h_out)) return rc;
  } else {
    if (int rc = ffn_rows_launch<FFN_UP_GELU>(c, rows, H, w1, I, H, I, a_out, h_out)) return rc;
  }
  return ffn_rows_launch<FFN_DOWN>(c, a_out, I, w2, H, I, H, y, nullptr);
}

extern "C" int zepp_op_expert_ffn_grad(const void* dy, const void* rows, int64_t n, const int32_t* offsets, int G, int H,
                                       int I, int act, const void* w1, const void* w2, const void* a, const void* h,
                                       void* dh_ws, void* drows, void* dw1, void* dw2, void* stream) {
  if (int rc = ffn_check("expert_ffn_grad", n, G, H, I, act, {dy, rows, w1, w2, a, h, dh_ws, drows, dw1, dw2})) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FfnCall c{offsets, n, G, H, I, act, nullptr, s};
  if (n == 0) {
    if (dw1 != nullptr) CU_OK(cudaMemsetAsync(dw1, 0, (size_t)G * c.f1() * H * 2, s));
    if (dw2 != nullptr) CU_OK(cudaMemsetAsync(dw2, 0, (size_t)G * H * I * 2, s));
    return 0;
  }
  if (!given({dy, rows, offsets, w1, w2, a, h}) || ((drows != nullptr || dw1 != nullptr) && dh_ws == nullptr))
    return fail("expert_ffn_grad: null pointer");
  if (int rc = op_device(&c.dev)) return rc;
  if (drows != nullptr || dw1 != nullptr) {
    if (act) {
      if (int rc = ffn_rows_launch<FFN_DACT_SWIGLU>(c, dy, H, w2, H, I, I, dh_ws, const_cast<void*>(h))) return rc;
    } else {
      if (int rc = ffn_rows_launch<FFN_DACT_GELU>(c, dy, H, w2, H, I, I, dh_ws, const_cast<void*>(h))) return rc;
    }
  }
  if (dw2 != nullptr)
    if (int rc = ffn_weight_launch(c, dy, H, a, I, dw2)) return rc;
  if (drows != nullptr)
    if (int rc = ffn_rows_launch<FFN_DROWS>(c, dh_ws, c.f1(), w1, c.f1(), H, H, drows, nullptr)) return rc;
  if (dw1 != nullptr)
    if (int rc = ffn_weight_launch(c, dh_ws, c.f1(), rows, H, dw1)) return rc;
  return 0;
}

// ---------------------------------------------------------------------------------------------
// norm of many tensors, scaling to a largest norm
// ---------------------------------------------------------------------------------------------
extern "C" size_t zepp_op_grad_norm_ws_bytes(int count) {
  // one block of partials for each launch of up to 1024 tensors
  return (size_t)((count + 1023) / 1024 + 1) * kNormMaxBlocks * sizeof(double);
}

// the table of tensors [lo, hi) and its chunks; empty tensors are left out
template <int CAP>
static int norm_table(NormTable<CAP>& t, void* const* ptrs, const int64_t* sizes, const uint8_t* dtypes, int lo, int hi) {
  t.count = 0;
  long long chunks = 0;
  for (int i = lo; i < hi; ++i) {
    if (sizes[i] == 0) continue;
    const int e = elem_bytes(dtypes[i]);
    const uintptr_t p = reinterpret_cast<uintptr_t>(ptrs[i]);
    const int k = t.count++;
    t.base[k] = p / 16 * 16;
    t.head[k] = (unsigned char)(p % 16 / e);
    t.end[k] = t.head[k] + sizes[i];
    t.type[k] = dtypes[i];
    t.chunk0[k] = (int)chunks;
    chunks += (t.end[k] * e + kNormChunkBytes - 1) / kNormChunkBytes;
    if (chunks >= (1ll << 31)) return fail("grad_norm: too many elements in one call");
  }
  t.chunk0[t.count] = (int)chunks;
  return 0;
}

template <int CAP>
static int norm_run(void* const* ptrs, const int64_t* sizes, const uint8_t* dtypes, int count, double max_norm, float* out,
                    double* ws, OpDevice* d, cudaStream_t s) {
  static thread_local NormTable<CAP> t;      // up to 20 KB: not on the caller's stack
  int n = 0;                                 // partials so far
  int held = -1;                             // where the tensors in the table begin
  const int resident = 4 * d->sms;
  for (int lo = 0; lo < count; lo += CAP) {
    if (int rc = norm_table(t, ptrs, sizes, dtypes, lo, lo + CAP < count ? lo + CAP : count)) return rc;
    held = lo;
    const int chunks = t.chunk0[t.count];
    if (chunks == 0) continue;
    const int blocks = chunks < resident ? chunks : resident;
    norm_partials_kernel<CAP><<<blocks, kNormThreads, 0, s>>>(t, ws + n);
    OP_LAUNCHED();
    n += blocks;
  }
  if (max_norm < 0 || n == 0) {
    norm_finish_kernel<<<1, kNormThreads, 0, s>>>(ws, n, out);
    OP_LAUNCHED();
    return 0;
  }
  bool first = true;
  for (int lo = (count - 1) / CAP * CAP; lo >= 0; lo -= CAP) {
    if (lo != held)
      if (int rc = norm_table(t, ptrs, sizes, dtypes, lo, lo + CAP < count ? lo + CAP : count)) return rc;
    held = lo;
    const int chunks = t.chunk0[t.count];
    if (chunks == 0) continue;
    norm_scale_kernel<CAP><<<chunks < resident ? chunks : resident, kNormThreads, 0, s>>>(t, ws, n, max_norm, first ? out : nullptr);
    OP_LAUNCHED();
    first = false;
  }
  return 0;
}

extern "C" int zepp_op_grad_norm(void* const* ptrs, const int64_t* sizes, const uint8_t* dtypes, int count, double max_norm,
                                 float* norm, void* ws, void* stream) {
  if (count < 0) return fail("grad_norm: %d tensors", count);
  if (!given({norm, ws}) || (count > 0 && !given({ptrs, sizes, dtypes}))) return fail("grad_norm: null pointer");
  for (int i = 0; i < count; ++i) {
    if (dtypes[i] > OP_F16) return fail("grad_norm: unknown element type %d of tensor %d", dtypes[i], i);
    if (sizes[i] < 0 || sizes[i] >= (1ll << 45)) return fail("grad_norm: %lld elements in tensor %d", (long long)sizes[i], i);
    if (sizes[i] > 0 && ptrs[i] == nullptr) return fail("grad_norm: tensor %d is a null pointer", i);
    if (sizes[i] > 0 && !aligned(ptrs[i], elem_bytes(dtypes[i]))) return fail("grad_norm: tensor %d is not aligned to its elements", i);
  }
  OpDevice* d;
  if (int rc = op_device(&d)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the table is copied with every launch: 0.7, 5.6 or 22 KB
  if (count <= 32) return norm_run<32>(ptrs, sizes, dtypes, count, max_norm, norm, static_cast<double*>(ws), d, s);
  if (count <= 256) return norm_run<256>(ptrs, sizes, dtypes, count, max_norm, norm, static_cast<double*>(ws), d, s);
  return norm_run<1024>(ptrs, sizes, dtypes, count, max_norm, norm, static_cast<double*>(ws), d, s);
}
