// 2-norm over a list of tensors and clipping by it (include/m355_dist.h).  The list travels in the kernel arguments, up
// to kListMax tensors of one type a launch: nothing is uploaded, nothing is kept between calls, and a captured graph holds
// its own copy.  The tensors of a launch are cut into chunks of kChunkVecs 16-byte accesses per thread that never cross a
// tensor.  Squares are added in float64 (a float32 square overflows at 1.8e19, and the float64 multiply-adds cost a fifth of
// the memory time); one partial sum per workgroup, added in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "m355_error.h"
#include "m355_logits_io.h"

namespace m355 {

constexpr int kListMax = 128;     // 3712 bytes of kernel arguments
constexpr int kListThreads = 256;
constexpr int kChunkVecs = 4;     // 16-byte accesses in flight per thread
constexpr int kNormBlocks = 2048;  // workgroups per launch of the norm: partial sums
constexpr int kFinalThreads = 1024;

struct TensorList {
  int count, chunks;
  const void* in[kListMax];
  void* out[kListMax];
  long long n[kListMax];
  int first[kListMax];  // index of the tensor's first chunk
};

template <class T> constexpr long long kChunkElems = (long long)kListThreads * kChunkVecs * kPer<T>;

// the tensor a chunk belongs to: the last one that begins at or before it (scalar loads of kernel arguments)
M355_DEV int tensor_of(const TensorList& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A thread's pieces of a chunk: full 16-byte accesses, and the tensor's last n % kPer elements singly by the first threads of
// its last chunk.
template <class T> struct Chunk {
  const typename T::store* p;
  long long at, left;  // element of the thread's first piece; elements of the tensor from there on
  int thread;  // of the chunk's kListThreads
  M355_DEV Chunk(const TensorList& l, int t, int c, int thread_)
      : p(static_cast<const typename T::store*>(l.in[t])),
        at((c - l.first[t]) * kChunkElems<T> + thread_ * kPer<T>),
        left(l.n[t] - at),
        thread(thread_) {}
  M355_DEV bool whole(int j) const { return left >= ((long long)j * kListThreads + 1) * kPer<T>; }
  // the element of the tensor's tail that is this thread's, or -1
  M355_DEV long long tail(const TensorList& l, int t, int c) const {
    const long long n = l.n[t], full = n / kPer<T> * kPer<T>;
    const bool last = (c - l.first[t] + 1) * kChunkElems<T> >= n;
    return last && full + thread < n ? full + thread : -1;
  }
};

// A thread's share of the squares of the chunks [lo, hi): the tensor is searched once and then followed, and the next chunk's
// loads are under way while one chunk's squares are added.
template <class T> M355_DEV double sum_run(const TensorList& l, int lo, int hi, int thread) {
  constexpr int N = kPer<T>;
  raw_t<T> none;
  none.x = none.y = none.z = none.w = 0;
  raw_t<T> raw[2][kChunkVecs];
  double acc[2] = {0.0, 0.0};
  int t = lo < hi ? tensor_of(l, lo) : 0;
  auto fetch = [&](int c, raw_t<T>(&r)[kChunkVecs]) {
    while (t + 1 < l.count && l.first[t + 1] <= c) ++t;
    const Chunk<T> k(l, t, c, thread);
#pragma unroll
    for (int j = 0; j < kChunkVecs; ++j) r[j] = k.whole(j) ? load_raw<T>(k.p + k.at + (long long)j * kListThreads * N) : none;
    const long long e = k.tail(l, t, c);
    if (e >= 0) {
      const double v = (double)k.p[e];
      acc[0] = __builtin_fma(v, v, acc[0]);
    }
  };
  auto add = [&](const raw_t<T>(&r)[kChunkVecs]) {
#pragma unroll
    for (int j = 0; j < kChunkVecs; ++j) {
      typename T::comp v[N];
      unpack<T>(r[j], v);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e & 1] = __builtin_fma((double)v[e], (double)v[e], acc[e & 1]);
    }
  };
  if (lo < hi) fetch(lo, raw[0]);
  for (int c = lo; c < hi; c += 2) {
    if (c + 1 < hi) fetch(c + 1, raw[1]);
    add(raw[0]);
    if (c + 1 >= hi) break;
    if (c + 2 < hi) fetch(c + 2, raw[0]);
    add(raw[1]);
  }
  return acc[0] + acc[1];
}

// The chunks of a launch in equal runs, one a workgroup.  Bound by HBM: 5.6e8 bytes of bf16 in 96-99 us, 5.7-5.9 TB/s.
template <class T> __global__ __launch_bounds__(kListThreads) void k_norm_partials(const TensorList l, double* __restrict__ partials) {
  const int lo = (int)((long long)l.chunks * blockIdx.x / gridDim.x), hi = (int)((long long)l.chunks * (blockIdx.x + 1) / gridDim.x);
  const double s = block_reduce_sum(sum_run<T>(l, lo, hi, threadIdx.x));
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Sum over a workgroup of kFinalThreads; valid in thread 0
M355_DEV double sum_wide(double v) {
  __shared__ double red[kFinalThreads / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0)
#pragma unroll
    for (int w = 1; w < kFinalThreads / 64; ++w) v += red[w];
  return v;
}

M355_DEV void store_norm(void* norm, int dtype, double v) {
  if (!norm) return;
  if (dtype == M355_F64) *static_cast<double*>(norm) = v;
  else *static_cast<float*>(norm) = (float)v;
}

// The factor of the clipping, 1 where nothing is clipped: up to max_norm, and where the norm is not finite as it goes out (the
// sum of squares of float32 gradients may have a root that float32 does not hold).
M355_DEV double clip_factor(double n, double max_norm, int norm_dtype) {
  const bool finite = norm_dtype == M355_F64 ? n < kInf : (float)n < (float)kInf;
  return n > max_norm && finite ? max_norm / n : 1.0;
}

// Joins the partial sums: the sum of squares, the norm, and the factor of the clipping
__global__ __launch_bounds__(kFinalThreads) void k_norm_final(const double* __restrict__ partials, int count,
                                                              double* __restrict__ sumsq, void* __restrict__ norm,
                                                              int norm_dtype, double max_norm, double* __restrict__ factor) {
  double acc = 0.0;
  for (int base = threadIdx.x; base < count; base += 4 * kFinalThreads) {
    double v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = base + j * kFinalThreads < count ? partials[base + j * kFinalThreads] : 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc += v[j];
  }
  const double s = sum_wide(acc);
  if (threadIdx.x == 0) {
    const double n = ::sqrt(s);
    if (sumsq) *sumsq = s;
    store_norm(norm, norm_dtype, n);
    if (factor) *factor = clip_factor(n, max_norm, norm_dtype);
  }
}

template <class T> M355_DEV void scale_chunk(const TensorList& l, int t, int c, const Chunk<T>& k, double f) {
  constexpr int N = kPer<T>;
  typedef typename T::comp comp;
  typename T::store* out = static_cast<typename T::store*>(l.out[t]);
  raw_t<T> raw[kChunkVecs];
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j)
    if (k.whole(j)) raw[j] = load_raw_nt<T>(k.p + k.at + (long long)j * kListThreads * N);
  const long long e = k.tail(l, t, c);
  if (e >= 0) out[e] = (typename T::store)(comp)((double)k.p[e] * f);
#pragma unroll
  for (int j = 0; j < kChunkVecs; ++j) {
    if (!k.whole(j)) continue;
    comp v[N];
    unpack<T>(raw[j], v);
    // the product in float64, rounded to float32 on the way to a 16-bit type (which is off by at most 2^-24 more)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (comp)((double)v[i] * f);
    store_raw_nt<T>(out + k.at + (long long)j * kListThreads * N, pack<T>(v));
  }
}

// One workgroup per chunk.  The list comes with its last tensors first: they are what the Infinity Cache still holds of the
// pass that formed the norm.  5.64e8 bytes of bf16 read and written in 170-190 us, 5.9-6.7 TB/s, as a copy.
template <class T> __global__ __launch_bounds__(kListThreads) void k_norm_scale(const TensorList l, const double* __restrict__ factor) {
  const double f = *factor;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    if (f == 1.0 && l.in[t] == l.out[t]) continue;  // in place and not clipped
    scale_chunk<T>(l, t, c, Chunk<T>(l, t, c, threadIdx.x), f);
  }
}

// A short list (one type, one launch, kSmallChunks chunks at most) in one workgroup, norm and scale: the launches that the
// general path needs cost more than the work (24 float32 tensors of 6 * 10^4 elements: a call of 20 against 23 us).
constexpr int kSmallChunks = 32;
template <class T>
__global__ __launch_bounds__(kFinalThreads) void k_norm_small(const TensorList l, double* __restrict__ sumsq,
                                                              void* __restrict__ norm, int norm_dtype, double max_norm,
                                                              bool scales) {
  constexpr int kGroups = kFinalThreads / kListThreads;
  __shared__ double shared_sum;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / kListThreads), thread = threadIdx.x % kListThreads;
  const int lo = l.chunks * group / kGroups, hi = l.chunks * (group + 1) / kGroups;
  double acc = sum_run<T>(l, lo, hi, thread);
  acc = sum_wide(acc);
  if (threadIdx.x == 0) {
    shared_sum = acc;
    if (sumsq) *sumsq = acc;
    store_norm(norm, norm_dtype, ::sqrt(acc));
  }
  if (!scales) return;
  __syncthreads();
  const double f = clip_factor(::sqrt(shared_sum), max_norm, norm_dtype);
  for (int c = lo; c < hi; ++c) {
    const int t = tensor_of(l, c);
    if (f == 1.0 && l.in[t] == l.out[t]) continue;
    scale_chunk<T>(l, t, c, Chunk<T>(l, t, c, thread), f);
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

int check_list(int64_t count, const m355_tensor* t, bool out) {
  if (count < 0 || (count && !t)) return fail(M355_ERR_INVALID, "bad list of tensors");
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].dtype != M355_F64 && t[i].dtype != M355_F32 && t[i].dtype != M355_F16 && t[i].dtype != M355_BF16)
      return fail(M355_ERR_INVALID, "tensor %lld: float64, float32, float16 or bfloat16", (long long)i);
    if (t[i].n < 0 || t[i].n > INT64_C(1) << 40) return fail(M355_ERR_INVALID, "tensor %lld: bad size", (long long)i);
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

template <class F> void by_dtype(int dtype, F f) {
  switch (dtype) {
    case M355_F64: return f(m355::F64());
    case M355_F32: return f(m355::F32());
    case M355_F16: return f(m355::F16());
    default: return f(m355::BF16());
  }
}

// Calls f(type, list) for launch-sized pieces of the tensors that are not empty, type by type; backwards: the last first.
template <class F> void each_launch(int64_t count, const m355_tensor* t, bool backwards, F f) {
  const int types[4] = {M355_F64, M355_F32, M355_F16, M355_BF16};
  bool has[5] = {};
  for (int64_t i = 0; i < count; ++i)
    if (t[i].n) has[t[i].dtype] = true;
  for (int step = 0; step < 4; ++step) {
    const int dtype = types[backwards ? 3 - step : step];
    if (!has[dtype]) continue;
    by_dtype(dtype, [&](auto type) {
      TensorList l;
      l.count = l.chunks = 0;
      const long long ce = m355::kChunkElems<decltype(type)>;
      for (int64_t at = 0; at < count; ++at) {
        const m355_tensor& x = t[backwards ? count - 1 - at : at];
        if (x.dtype != dtype || !x.n) continue;
        const int chunks = (int)((x.n + ce - 1) / ce);  // at most 2^30 (check_list)
        if (l.count == kListMax || l.chunks > INT32_MAX - chunks) {
          f(type, l);
          l.count = l.chunks = 0;
        }
        l.in[l.count] = x.ptr;
        l.out[l.count] = x.out;
        l.n[l.count] = x.n;
        l.first[l.count] = l.chunks;
        l.chunks += chunks;
        ++l.count;
      }
      if (l.count) f(type, l);
    });
  }
}

// launches of a list at most: full ones, one begun per type, and what a launch's chunk count (31 bits) cuts off
int64_t launches_of(int64_t count) { return count / kListMax + 4; }

// Runs f(type, list) if the whole list is short enough for one workgroup.
template <class F> bool if_small(int64_t count, const m355_tensor* t, F f) {
  int lists = 0;
  int64_t elems = 0;
  for (int64_t i = 0; i < count; ++i) elems += t[i].n;
  if (count > kListMax || elems > INT64_C(1) << 20) return false;
  bool small = true;
  each_launch(count, t, false, [&](auto, const TensorList& l) { small = small && ++lists == 1 && l.chunks <= m355::kSmallChunks; });
  if (!small || !lists) return false;
  each_launch(count, t, false, f);
  return true;
}

int partial_sums(int64_t count, const m355_tensor* t, double* ws, size_t ws_bytes, hipStream_t s, int* nparts) {
  const size_t room = ws_bytes / sizeof(double) - 1;  // one double stays free for the factor
  size_t at = 0;
  bool fits = true;
  each_launch(count, t, false, [&](auto type, const TensorList& l) {
    const int grid = l.chunks < m355::kNormBlocks ? l.chunks : m355::kNormBlocks;
    if (!fits || at + grid > room) {
      fits = false;
      return;
    }
    hipLaunchKernelGGL((m355::k_norm_partials<decltype(type)>), dim3(grid), dim3(m355::kListThreads), 0, s, l, ws + at);
    at += grid;
  });
  *nparts = (int)at;
  return fits ? 0 : fail(M355_ERR_WORKSPACE, "workspace too small");
}
}  // namespace

extern "C" size_t m355_global_norm_workspace_bytes(int64_t count) {
  return ((size_t)launches_of(count > 0 ? count : 0) * m355::kNormBlocks + 1) * sizeof(double);
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
  if (if_small(count, tensors, [&](auto type, const TensorList& l) {
        hipLaunchKernelGGL((m355::k_norm_small<decltype(type)>), dim3(1), dim3(m355::kFinalThreads), 0, s, l, sumsq, norm,
                           norm_dtype, 0.0, false);
      }))
    return launched();
  int nparts = 0;
  if ((rc = partial_sums(count, tensors, ws, workspace_bytes, s, &nparts))) return rc;
  hipLaunchKernelGGL(m355::k_norm_final, dim3(1), dim3(m355::kFinalThreads), 0, s, ws, nparts, sumsq, norm, norm_dtype,
                     0.0, static_cast<double*>(nullptr));
  return launched();
}

extern "C" int m355_clip_global_norm(int64_t count, const m355_tensor* tensors, double max_norm, const double* sumsq,
                                     void* norm, int norm_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_list(count, tensors, true);
  if (rc) return rc;
  if (!(max_norm >= 0.0)) return fail(M355_ERR_INVALID, "max_norm must be >= 0");
  if (norm_dtype != M355_F64 && norm_dtype != M355_F32) return fail(M355_ERR_INVALID, "the norm is float64 or float32");
  if (!workspace) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if (workspace_bytes < m355_global_norm_workspace_bytes(count)) return fail(M355_ERR_WORKSPACE, "workspace too small");
  try {
    if ((rc = check_overlap(count, tensors))) return rc;
  } catch (const std::bad_alloc&) {
    return fail(M355_ERR_INVALID, "out of host memory");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* ws = static_cast<double*>(workspace);
  if (!sumsq && if_small(count, tensors, [&](auto type, const TensorList& l) {
        hipLaunchKernelGGL((m355::k_norm_small<decltype(type)>), dim3(1), dim3(m355::kFinalThreads), 0, s, l,
                           static_cast<double*>(nullptr), norm, norm_dtype, max_norm, true);
      }))
    return launched();
  int nparts = 0;
  if (!sumsq && (rc = partial_sums(count, tensors, ws, workspace_bytes, s, &nparts))) return rc;
  double* factor = ws + nparts;
  hipLaunchKernelGGL(m355::k_norm_final, dim3(1), dim3(m355::kFinalThreads), 0, s, sumsq ? sumsq : ws, sumsq ? 1 : nparts,
                     static_cast<double*>(nullptr), norm, norm_dtype, max_norm, factor);
  each_launch(count, tensors, true, [&](auto type, const TensorList& l) {
    hipLaunchKernelGGL((m355::k_norm_scale<decltype(type)>), dim3(l.chunks < (1 << 23) ? l.chunks : 1 << 23),
                       dim3(m355::kListThreads), 0, s, l, factor);
  });
  return launched();
}
