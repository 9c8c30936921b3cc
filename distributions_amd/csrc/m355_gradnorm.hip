// 2-norm over a list of tensors and clipping by it (include/m355_dist.h).  The list travels in the kernel arguments, up
// to kListMax tensors a launch: nothing is uploaded, nothing is kept between calls, and a captured graph holds its own
// copy.  The tensors of a launch are cut into chunks of kChunkVecs 16-byte accesses per thread that never cross a tensor;
// workgroups take chunks in turn.  Squares are added in float64 (a float32 square overflows at 1.8e19, and the float64
// fused multiply-adds cost a tenth of the memory time); one partial sum per workgroup, added in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "m355_error.h"
#include "m355_logits_io.h"

namespace m355 {

constexpr int kListMax = 128;     // 3712 bytes of kernel arguments
constexpr int kListThreads = 256;
constexpr int kChunkVecs = 8;     // 16-byte accesses in flight per thread
constexpr int kNormBlocks = 2048;  // workgroups per launch of the norm: partial sums

struct TensorList {
  int count, chunks;
  const void* in[kListMax];
  void* out[kListMax];
  long long n[kListMax];
  int first[kListMax];  // index of the tensor's first chunk
  unsigned char dtype[kListMax];
};

template <class T> constexpr long long kChunkElems = (long long)kListThreads * kChunkVecs * kPer<T>;

M355_DEV int tensor_of(const TensorList& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <class T> M355_DEV double sum_squares(const void* in, long long n, long long base) {
  const typename T::store* p = static_cast<const typename T::store*>(in);
  constexpr int N = kPer<T>;
  raw_t<T> raw[kChunkVecs];
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j) {
    const long long v = base + (j * kListThreads + (int)threadIdx.x) * N;
    if (v < n) raw[j] = load_row<T>(p, v, n, 0);
  }
  double acc = 0.0;
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j) {
    const long long v = base + (j * kListThreads + (int)threadIdx.x) * N;
    if (v >= n) continue;
    typename T::comp t[N];
    unpack<T>(raw[j], t);
#pragma unroll
    for (int e = 0; e < N; ++e) acc = __builtin_fma((double)t[e], (double)t[e], acc);
  }
  return acc;
}

template <class T> M355_DEV void scale_chunk(const void* in, void* out, long long n, long long base, double f) {
  const typename T::store* p = static_cast<const typename T::store*>(in);
  constexpr int N = kPer<T>;
  raw_t<T> raw[kChunkVecs];
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j) {
    const long long v = base + (j * kListThreads + (int)threadIdx.x) * N;
    if (v < n) raw[j] = load_row<T>(p, v, n, 0);
  }
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j) {
    const long long v = base + (j * kListThreads + (int)threadIdx.x) * N;
    if (v >= n) continue;
    typename T::comp t[N];
    unpack<T>(raw[j], t);
    // the product in float64, rounded to float32 on the way to a 16-bit type (twice rounded: off by at most 2^-25 more)
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = (typename T::comp)((double)t[e] * f);
    store_row<T>(static_cast<typename T::store*>(out), v, n, t);
  }
}

__global__ __launch_bounds__(kListThreads) void k_norm_partials(const TensorList l, double* __restrict__ partials) {
  double acc = 0.0;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const long long i = c - l.first[t];
    switch (l.dtype[t]) {
      case M355_F64: acc += sum_squares<F64>(l.in[t], l.n[t], i * kChunkElems<F64>); break;
      case M355_F32: acc += sum_squares<F32>(l.in[t], l.n[t], i * kChunkElems<F32>); break;
      case M355_F16: acc += sum_squares<F16>(l.in[t], l.n[t], i * kChunkElems<F16>); break;
      default: acc += sum_squares<BF16>(l.in[t], l.n[t], i * kChunkElems<BF16>); break;
    }
  }
  acc = block_reduce_sum(acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// Sum of the partials over a workgroup of kListThreads, in the same order wherever it is taken; valid in thread 0
M355_DEV double sum_partials(const double* __restrict__ partials, int count) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < count; i += kListThreads) acc += partials[i];
  return block_reduce_sum(acc);
}

M355_DEV void store_norm(void* norm, int dtype, double v) {
  if (!norm) return;
  if (dtype == M355_F64) *static_cast<double*>(norm) = v;
  else *static_cast<float*>(norm) = (float)v;
}

__global__ __launch_bounds__(kListThreads) void k_norm_final(const double* __restrict__ partials, int count,
                                                             double* __restrict__ sumsq, void* __restrict__ norm,
                                                             int norm_dtype) {
  const double s = sum_partials(partials, count);
  if (threadIdx.x == 0) {
    if (sumsq) *sumsq = s;
    store_norm(norm, norm_dtype, ::sqrt(s));
  }
}

// Every workgroup adds the partials itself (a few reads from L2), so that norm and scale need no launch in between.
__global__ __launch_bounds__(kListThreads) void k_norm_scale(const TensorList l, const double* __restrict__ partials,
                                                             int count, double max_norm, void* __restrict__ norm,
                                                             int norm_dtype) {
  __shared__ double shared_sum;
  const double s = sum_partials(partials, count);
  if (threadIdx.x == 0) {
    shared_sum = s;
    if (blockIdx.x == 0) store_norm(norm, norm_dtype, ::sqrt(s));
  }
  __syncthreads();
  const double n = ::sqrt(shared_sum);
  const bool clips = n > max_norm && n < kInf;
  const double f = clips ? max_norm / n : 1.0;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    if (!clips && l.in[t] == l.out[t]) continue;
    const long long i = c - l.first[t];
    switch (l.dtype[t]) {
      case M355_F64: scale_chunk<F64>(l.in[t], l.out[t], l.n[t], i * kChunkElems<F64>, f); break;
      case M355_F32: scale_chunk<F32>(l.in[t], l.out[t], l.n[t], i * kChunkElems<F32>, f); break;
      case M355_F16: scale_chunk<F16>(l.in[t], l.out[t], l.n[t], i * kChunkElems<F16>, f); break;
      default: scale_chunk<BF16>(l.in[t], l.out[t], l.n[t], i * kChunkElems<BF16>, f); break;
    }
  }
}

}  // namespace m355

namespace {
using m355::fail;
using m355::kListMax;
using m355::TensorList;

int launched() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? M355_OK : fail(M355_ERR_LAUNCH, "HIP launch failed: %s", hipGetErrorString(e));
}

size_t item_size(int dtype) { return dtype == M355_F64 ? 8 : dtype == M355_F32 ? 4 : 2; }

long long chunk_elems(int dtype) {
  return (long long)m355::kListThreads * m355::kChunkVecs * (16 / (long long)item_size(dtype));
}

int check_list(int64_t count, const m355_tensor* t, bool out) {
  if (count < 0 || (count && !t)) return fail(M355_ERR_INVALID, "bad list of tensors");
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].dtype != M355_F64 && t[i].dtype != M355_F32 && t[i].dtype != M355_F16 && t[i].dtype != M355_BF16)
      return fail(M355_ERR_INVALID, "tensor %lld: float64, float32, float16 or bfloat16", (long long)i);
    if (t[i].n < 0 || t[i].n > INT64_C(1) << 42) return fail(M355_ERR_INVALID, "tensor %lld: bad size", (long long)i);
    if (t[i].n && (!t[i].ptr || (out && !t[i].out))) return fail(M355_ERR_INVALID, "NULL pointer argument");
  }
  return 0;
}

// No output may overlap another output or an input other than its own.
int check_overlap(int64_t count, const m355_tensor* t) {
  struct Range {
    uintptr_t lo, hi;
    bool out;
  };
  std::vector<Range> r;
  r.reserve(2 * (size_t)count);
  for (int64_t i = 0; i < count; ++i) {
    if (!t[i].n) continue;
    const uintptr_t bytes = (uintptr_t)t[i].n * item_size(t[i].dtype), o = (uintptr_t)t[i].out, p = (uintptr_t)t[i].ptr;
    r.push_back({o, o + bytes, true});
    if (o != p) r.push_back({p, p + bytes, false});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t any = 0, outs = 0;  // ends of what began before
  for (const Range& x : r) {
    if (x.lo < (x.out ? any : outs))
      return fail(M355_ERR_INVALID, "an output overlaps another tensor (or a tensor is listed twice with outputs in place)");
    any = std::max(any, x.hi);
    if (x.out) outs = std::max(outs, x.hi);
  }
  return 0;
}

// Calls f(list) for launch-sized pieces of the tensors that are not empty.
template <class F> void each_launch(int64_t count, const m355_tensor* t, F f) {
  TensorList l;
  l.count = 0;
  l.chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const long long ce = chunk_elems(t[i].dtype);
    long long at = 0;
    while (at < t[i].n) {  // a launch counts its chunks in 31 bits: a tensor that would not fit goes on in the next one
      if (l.count == kListMax || l.chunks >= (1 << 30)) {
        f(l);
        l.count = l.chunks = 0;
      }
      const long long room = (1ll << 30) - l.chunks;
      const long long n = std::min((long long)t[i].n - at, room * ce);
      const size_t off = (size_t)at * item_size(t[i].dtype);
      l.in[l.count] = static_cast<const char*>(t[i].ptr) + off;
      l.out[l.count] = t[i].out ? static_cast<char*>(t[i].out) + off : nullptr;
      l.n[l.count] = n;
      l.first[l.count] = l.chunks;
      l.dtype[l.count] = (unsigned char)t[i].dtype;
      l.chunks += (int)((n + ce - 1) / ce);
      ++l.count;
      at += n;
    }
  }
  if (l.count) f(l);
}

// launches of a list: what the workspace is sized for (each tensor may be continued in one more launch)
int64_t launches_of(int64_t count) { return (count + kListMax - 1) / kListMax + 1; }

int partial_sums(int64_t count, const m355_tensor* t, double* ws, size_t ws_bytes, hipStream_t s, int* nparts) {
  const size_t room = ws_bytes / sizeof(double);
  size_t at = 0;
  bool fits = true;
  each_launch(count, t, [&](const TensorList& l) {
    const int grid = l.chunks < m355::kNormBlocks ? l.chunks : m355::kNormBlocks;
    if (!fits || at + grid >= room) {  // one double stays free for the joined sum
      fits = false;
      return;
    }
    hipLaunchKernelGGL(m355::k_norm_partials, dim3(grid), dim3(m355::kListThreads), 0, s, l, ws + at);
    at += grid;
  });
  *nparts = (int)at;
  return fits ? 0 : fail(M355_ERR_WORKSPACE, "workspace too small");
}
}  // namespace

extern "C" size_t m355_global_norm_workspace_bytes(int64_t count) {
  return (size_t)launches_of(count > 0 ? count : 0) * m355::kNormBlocks * sizeof(double);
}

extern "C" int m355_global_norm(int64_t count, const m355_tensor* tensors, double* sumsq, void* norm, int norm_dtype,
                                void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_list(count, tensors, false);
  if (rc) return rc;
  if (norm_dtype != M355_F64 && norm_dtype != M355_F32) return fail(M355_ERR_INVALID, "the norm is float64 or float32");
  if (!workspace) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if (workspace_bytes < m355_global_norm_workspace_bytes(count)) return fail(M355_ERR_WORKSPACE, "workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* ws = static_cast<double*>(workspace);
  int nparts = 0;
  if ((rc = partial_sums(count, tensors, ws, workspace_bytes, s, &nparts))) return rc;
  hipLaunchKernelGGL(m355::k_norm_final, dim3(1), dim3(m355::kListThreads), 0, s, ws, nparts, sumsq, norm, norm_dtype);
  return launched();
}

extern "C" int m355_clip_global_norm(int64_t count, const m355_tensor* tensors, double max_norm, const double* sumsq,
                                     void* norm, int norm_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_list(count, tensors, true);
  if (rc) return rc;
  if (!(max_norm >= 0.0)) return fail(M355_ERR_INVALID, "max_norm must be >= 0");
  if (norm_dtype != M355_F64 && norm_dtype != M355_F32) return fail(M355_ERR_INVALID, "the norm is float64 or float32");
  if (!sumsq && !workspace) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if (!sumsq && workspace_bytes < m355_global_norm_workspace_bytes(count))
    return fail(M355_ERR_WORKSPACE, "workspace too small");
  try {
    if ((rc = check_overlap(count, tensors))) return rc;
  } catch (const std::bad_alloc&) {
    return fail(M355_ERR_INVALID, "out of host memory");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* ws = static_cast<double*>(workspace);
  const double* parts = sumsq;
  int nparts = 1;
  if (!sumsq) {
    if ((rc = partial_sums(count, tensors, ws, workspace_bytes, s, &nparts))) return rc;
    parts = ws;
    if (nparts > m355::kNormBlocks) {  // several launches: one workgroup adds their partials, not every workgroup of the scale
      hipLaunchKernelGGL(m355::k_norm_final, dim3(1), dim3(m355::kListThreads), 0, s, ws, nparts, ws + nparts, nullptr,
                         M355_F64);
      parts = ws + nparts;
      nparts = 1;
    }
  }
  bool first = true;
  each_launch(count, tensors, [&](const TensorList& l) {
    const int grid = l.chunks < 8192 ? l.chunks : 8192;
    hipLaunchKernelGGL(m355::k_norm_scale, dim3(grid), dim3(m355::kListThreads), 0, s, l, parts, nparts, max_norm,
                       first ? norm : nullptr, norm_dtype);
    first = false;
  });
  if (first)  // nothing to scale: the norm alone
    hipLaunchKernelGGL(m355::k_norm_final, dim3(1), dim3(m355::kListThreads), 0, s, parts, nparts, nullptr, norm, norm_dtype);
  return launched();
}
