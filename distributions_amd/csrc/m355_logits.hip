// Categorical given by logits: adjustment before drawing or scoring (penalties, bias, temperature, mask) with its
// gradient, log-density and the gradient of the weighted sum of log-densities.  Formulas: include/m355_dist.h.
#include <hip/hip_runtime.h>

#include "m355_error.h"
#include "m355_logits_io.h"

namespace m355 {

// ------------------------------------------------------------------------------------------------ adjust
struct AdjustArgs {
  long long rows, k;
  const void* src;  // the logits (forward) or g (gradient)
  long long src_ld;
  const void* x;  // gradient: the logits, for the sign of the penalised ones
  long long x_ld;
  void* dst;  // NULL: not wanted (gradient)
  long long dst_ld;
  void* dbias;  // gradient: per-element gradient of the bias (rows x k), or NULL
  const void* history;
  long long history_ld;
  int history_len, history_dtype;
  const long long *lengths, *prompts;
  DevOperand rep, pres, freq, temp;
  const void* bias;
  long long bias_ld;
  int bias_dtype;
  int mask_kind;
  const void* mask;
  long long mask_ld;
};

// Whether category v is allowed
M355_DEV bool allowed(const AdjustArgs& a, long long row, long long v) {
  if (a.mask_kind == M355_MASK_NONE) return true;
  if (a.mask_kind == M355_MASK_BITS) return (static_cast<const unsigned*>(a.mask)[row * a.mask_ld + (v >> 5)] >> (v & 31)) & 1;
  return static_cast<const unsigned char*>(a.mask)[row * a.mask_ld + v] != 0;
}
// The mask of a whole piece (v is a multiple of kPer, v + kPer <= k): the raw bytes resp. the word, then its kPer flags
template <class T> struct MaskPiece {
  typename std::conditional<kPer<T> == 8, unsigned long long, unsigned>::type bytes;
  // `rel` categories behind category `base` of the row; row and base are the same for the whole workgroup, so that the
  // address is a scalar plus a 32-bit offset
  M355_DEV void load(const AdjustArgs& a, long long row, long long base, unsigned rel) {
    bytes = ~(decltype(bytes))0;
    if (a.mask_kind == M355_MASK_BYTES) {
      const unsigned char* m = static_cast<const unsigned char*>(a.mask) + row * a.mask_ld + base;
      __builtin_memcpy(&bytes, m + rel, kPer<T>);
    } else if (a.mask_kind == M355_MASK_BITS) {
      const unsigned* m = static_cast<const unsigned*>(a.mask) + row * a.mask_ld + (base >> 5);
      const unsigned at = (unsigned)(base & 31) + rel;
      bytes = m[at >> 5] >> (at & 31);
    }
  }
  M355_DEV bool operator()(const AdjustArgs& a, int e) const {
    return a.mask_kind == M355_MASK_BYTES ? ((bytes >> (8 * e)) & 0xff) != 0 : ((bytes >> e) & 1) != 0;
  }
};

// kPer values of the bias, of type B: the logits' own, or float32 next to 16-bit logits (two loads)
template <class T, class B> struct BiasPiece {
  static constexpr int kLoads = kPer<T> / kPer<B>;
  raw_t<B> raw[kLoads];
  M355_DEV void load(const AdjustArgs& a, long long row, long long base, unsigned rel) {
    const typename B::store* b = static_cast<const typename B::store*>(a.bias) + row * a.bias_ld + base;
#pragma unroll
    for (int h = 0; h < kLoads; ++h) raw[h] = load_raw<B>(b + (rel + h * kPer<B>));
  }
  M355_DEV void add_to(typename T::comp (&s)[kPer<T>]) const {
#pragma unroll
    for (int h = 0; h < kLoads; ++h) {
      typename B::comp b[kPer<B>];
      unpack<B>(raw[h], b);
#pragma unroll
      for (int e = 0; e < kPer<B>; ++e) s[h * kPer<B> + e] += b[e];
    }
  }
};
template <class T> struct BiasPiece<T, void> {
  M355_DEV void load(const AdjustArgs&, long long, long long, unsigned) {}
  M355_DEV void add_to(typename T::comp (&)[kPer<T>]) const {}
};

// Quotients by a row's argument d (temperature, repetition) are products with its reciprocal: one rounding more than a
// division per element, which would cost more than the rest of the body.  That needs a reciprocal that is a normal number:
// |d| in [2^-126, 2^126] (float64: 2^-1022, 2^1022).
template <class C> M355_DEV C reciprocal(const DevOperand& o, long long row) { return (C)1 / (C)row_operand(o, row); }
template <class C> M355_DEV bool normal(C inv) {
  constexpr C lo = (C)(sizeof(C) == 8 ? 0x1p-1022 : 0x1p-126);
  return __builtin_fabs(inv) >= lo && __builtin_fabs(inv) <= 1 / lo;
}
M355_DEV float ldexp_c(float v, int e) { return __builtin_ldexpf(v, e); }
M355_DEV double ldexp_c(double v, int e) { return __builtin_ldexp(v, e); }
// Products with d and 1 / d for any d = m 2^e: the power of two first, by the exponent, and m such that this overflows only
// where the result does.  For |d| in the range above the same values as the short way; 0, infinities and NaN as in s * d, s / d.
template <class C> struct Factor {
  C mul, inv;
  int up = 0, down = 0;
  M355_DEV explicit Factor(double d) : mul((C)d), inv((C)1 / (C)d) {
    if (normal(inv)) return;
    const double m = __builtin_amdgcn_frexp_mant(d);
    const int e = __builtin_amdgcn_frexp_exp(d);
    mul = (C)(2 * m), inv = (C)1 / (C)m;
    up = e - 1, down = -e;
  }
  M355_DEV C times(C s) const { return ldexp_c(s, up) * mul; }
  M355_DEV C over(C s) const { return ldexp_c(s, down) * inv; }
};
// s / argument of the row; inv: its reciprocal
template <class C, int N> M355_DEV void divide(C (&s)[N], const DevOperand& o, long long row, C inv) {
  if (__builtin_expect(normal(inv), true)) {
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] *= inv;
    return;
  }
  const Factor<C> f(row_operand(o, row));
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = f.over(s[e]);
}

struct AdjustGrid {
  long long items;
  int chunks, per;    // a row is cut into `chunks` of `per` pieces (of kPer categories)
  bool rows_by_xcd;  // see item_of
};
// (row, chunk) of a work item.  Workgroups are dealt to the eight XCDs in turn; with many rows all chunks of a row go to one
// of them, so that the row's history and mask words are fetched into one L2 and not into eight.
M355_DEV bool item_of(const AdjustArgs& a, const AdjustGrid& g, long long item, long long& row, int& chunk) {
  if (g.rows_by_xcd) {
    const long long local = item >> 3;
    row = local / g.chunks * 8 + (item & 7);
    chunk = (int)(local % g.chunks);
  } else {
    row = item / g.chunks;
    chunk = (int)(item % g.chunks);
  }
  return row < a.rows;
}

// Occurrences of the categories [base, base + width) in the row's history, in LDS: twice the number among the generated ids,
// plus 1 if the prompt has it, in C-sized counters: 32 bits, or 16 where the history is short enough for them.  One
// atomic per id; additions of integers: their order does not matter.
template <class C> M355_DEV void count_one(unsigned* counts, unsigned at, bool generated) {
  if (sizeof(C) == 2) {
    if (generated) atomicAdd(&counts[at >> 1], 2u << (16 * (at & 1)));
    else atomicOr(&counts[at >> 1], 1u << (16 * (at & 1)));
  } else {
    if (generated) atomicAdd(&counts[at], 2u);
    else atomicOr(&counts[at], 1u);
  }
}
template <class C, class ID, int THREADS>
M355_DEV void count_history(const AdjustArgs& a, long long row, unsigned base, unsigned width, unsigned* counts) {
  constexpr int U = 4;  // ids in flight per thread: the loop is all latency
  const ID* h = static_cast<const ID*>(a.history) + row * a.history_ld;
  const unsigned most = (unsigned)a.history_len, tid = threadIdx.x;  // positions and ids in 32 bits: both are below 2^31
  // the first ids are fetched before the row's length is known; those behind it are dropped
  ID id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) id[u] = u * THREADS + tid < most ? h[u * THREADS + tid] : (ID)-1;
  const long long given = a.lengths ? a.lengths[row] : a.history_len, start = a.prompts ? a.prompts[row] : 0;
  const unsigned len = given < 0 ? 0u : given > a.history_len ? most : (unsigned)given;
  const unsigned prompt = start < 0 ? 0u : start > a.history_len ? most : (unsigned)start;
  for (unsigned first = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = first + u * THREADS + tid;
      // an id outside [0, k) lies behind the chunk: base + width is at most 2^31, and a negative one wraps past it
      const bool small = sizeof(ID) == 4 || (unsigned)((unsigned long long)(long long)id[u] >> 32) == 0;
      const unsigned at = (unsigned)id[u] - base;
      if (small && i < len && at < width) count_one<C>(counts, at, i >= prompt);
    }
    first += U * THREADS;
    if (first >= len) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = first + u * THREADS + tid;
      id[u] = i < len ? h[i] : (ID)-1;
    }
  }
}

// The penalties of a row; inv = 1 / rep (one rounding more): a division would be paid for by nearly every wavefront, because
// nearly every one has some id of the history among its elements (64 x 131072 bf16, 2048 ids: 16.0 us with it, 13.7 without)
template <class C> struct Penalties {
  C rep, inv, pres, freq;
  M355_DEV C factor(C x) const { return x > 0 ? inv : rep; }
  M355_DEV C counted(C s, unsigned count) const {
    const C q = s - (freq * (C)(count >> 1) + pres);
    return count >> 1 ? q : s;
  }
  M355_DEV C operator()(C s, unsigned count) const {
    const C p = s * factor(s);
    return counted(count ? p : s, count);
  }
};

// One workgroup per (row, chunk): everything the chunk needs from memory is fetched first, then, with a history (CNT: the
// type of its counters, or void), the ids that fall into the chunk are counted in LDS, then the pieces are worked off.  The
// k % kPer last categories of a row belong to the first threads of its last chunk.  Without a history bound by HBM (1024 x
// 65537 float32: 97 us, 5.5 TB/s, rows at odd addresses); with one by the chain ids -> counters -> barrier -> stores, and every
// chunk of a row looks at all of its ids: 256 x 100003 float32 with 4001 ids 45 us (4.6 TB/s), 64 x 131072 bf16 with 2048 ids
// 12.9 us.  A row with a temperature or a penalty that has no normal reciprocal goes element by element; where that was a branch
// in the unrolled loops, the others paid for it (64 x 131072: 12.3 against 11.7 us, fewer wavefronts a SIMD).
template <class T, int THREADS, int VPT, class CNT, class B, bool BWD>
__global__ __launch_bounds__(THREADS, 4) void k_logits_adjust(const AdjustArgs a, const AdjustGrid grid) {
  typedef typename T::comp comp;
  typedef typename T::store store;
  constexpr int N = kPer<T>;
  constexpr bool HIST = !std::is_void<CNT>::value;
  typedef typename std::conditional<HIST, CNT, unsigned>::type cnt;
  constexpr int kCounts = HIST ? (THREADS * VPT + 1) * N : 4;  // one piece more for the tail
  __shared__ uint4 count_store[(kCounts * sizeof(cnt) + 15) / 16];
  cnt* counts = reinterpret_cast<cnt*>(count_store);
  const int tid = threadIdx.x, nv = (int)(a.k / N);
  for (long long item = blockIdx.x; item < grid.items; item += gridDim.x) {
    long long row;
    int chunk;
    if (!item_of(a, grid, item, row, chunk)) continue;
    const int c0 = chunk * grid.per, c1 = c0 + grid.per < nv ? c0 + grid.per : nv;  // pieces of the chunk
    const long long base = (long long)c0 * N;
    const unsigned count_here = (unsigned)(c1 - c0);
    const unsigned width = chunk == grid.chunks - 1 ? (unsigned)(a.k - base) : count_here * N;  // categories of the chunk
    const store* src = static_cast<const store*>(a.src) + row * a.src_ld;
    raw_t<T> raw[VPT];
    MaskPiece<T> mask[VPT];
    BiasPiece<T, typename std::conditional<BWD, void, B>::type> bias[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const unsigned i = j * THREADS + tid;
      if (i >= count_here) continue;
      raw[j] = load_raw<T>(src + base + i * N);
      mask[j].load(a, row, base, i * N);
      bias[j].load(a, row, base, i * N);
    }
    // the row's arguments before the barriers: behind them their latency would stand alone
    const comp inv_t = reciprocal<comp>(a.temp, row);
    Penalties<comp> penalty = {1, 1, 0, 0};
    if constexpr (HIST) {
      penalty.rep = (comp)row_operand(a.rep, row);
      penalty.inv = (comp)1 / penalty.rep;
      penalty.pres = (comp)row_operand(a.pres, row);
      penalty.freq = (comp)row_operand(a.freq, row);
      for (int i = tid; i < (int)(sizeof(count_store) / 16); i += THREADS) count_store[i] = uint4{0, 0, 0, 0};
      __syncthreads();
      if (a.history_dtype == M355_I64) count_history<cnt, long long, THREADS>(a, row, (unsigned)base, width, reinterpret_cast<unsigned*>(counts));
      else count_history<cnt, int, THREADS>(a, row, (unsigned)base, width, reinterpret_cast<unsigned*>(counts));
      __syncthreads();
    }
    store* dst = static_cast<store*>(a.dst) + row * a.dst_ld;
    const store* x = static_cast<const store*>(a.x) + row * a.x_ld;
    // behind the barriers: the arguments' loads are not waited for before the ids are under way
    const bool fast = normal(inv_t) && normal(penalty.inv);
    const unsigned whole = fast ? count_here : 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const unsigned i = j * THREADS + tid, rel = i * N;
      if (i >= whole) continue;
      comp s[N];
      unpack<T>(raw[j], s);
      cnt count[N];
      bool any = false;  // most pieces have no id of the history
      if constexpr (HIST) {
        __builtin_memcpy(count, counts + rel, sizeof(count));
#pragma unroll
        for (int e = 0; e < N; ++e) any |= count[e] != 0;
      }
      if constexpr (!BWD) {
        if (any) {
#pragma unroll
          for (int e = 0; e < N; ++e) s[e] = penalty(s[e], count[e]);
        }
        bias[j].add_to(s);
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] *= inv_t;
        if (a.mask_kind != M355_MASK_NONE) {
#pragma unroll
          for (int e = 0; e < N; ++e) s[e] = mask[j](a, e) ? s[e] : (comp)-kInf;
        }
        store_raw_nt<T>(dst + base + rel, pack<T>(s));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = mask[j](a, e) ? s[e] * inv_t : (comp)0;
        if constexpr (!std::is_void<B>::value) {  // every row has its own bias: the gradient goes out as it is
#pragma unroll
          for (int h = 0; h < N; h += kPer<B>) {
            typename B::comp db[kPer<B>];
#pragma unroll
            for (int e = 0; e < kPer<B>; ++e) db[e] = (typename B::comp)s[h + e];
            store_raw_nt<B>(static_cast<typename B::store*>(a.dbias) + row * a.k + base + (rel + h), pack<B>(db));
          }
        }
        if (a.dst) {
          if (any) {
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (count[e]) s[e] *= penalty.factor((comp)x[base + (rel + e)]);
          }
          store_raw_nt<T>(dst + base + rel, pack<T>(s));
        }
      }
    }
    auto single = [&](unsigned rel, auto exact) {
      const unsigned count = HIST ? counts[rel] : 0;
      const long long v = base + rel;
      const comp t = (comp)src[v];
      const bool ok = allowed(a, row, v);
      auto over_t = [&](comp s) { return exact ? Factor<comp>(row_operand(a.temp, row)).over(s) : s * inv_t; };
      auto repeated = [&](comp s, comp z) {
        if constexpr (exact) {
          const Factor<comp> r(row_operand(a.rep, row));
          return z > 0 ? r.over(s) : r.times(s);
        }
        return s * penalty.factor(z);
      };
      if constexpr (!BWD) {
        comp s = HIST && count ? repeated(t, t) : t;
        if constexpr (HIST) s = penalty.counted(s, count);
        if constexpr (!std::is_void<B>::value) s += (comp) static_cast<const typename B::store*>(a.bias)[row * a.bias_ld + v];
        dst[v] = (store)(ok ? over_t(s) : (comp)-kInf);
      } else {
        const comp s = ok ? over_t(t) : (comp)0;
        if constexpr (!std::is_void<B>::value) static_cast<typename B::store*>(a.dbias)[row * a.k + v] = (typename B::store)s;
        if (a.dst) dst[v] = (store)(HIST && count ? repeated(s, (comp)x[v]) : s);
      }
    };
    if (__builtin_expect(fast, true)) {
      const unsigned rel = count_here * N + tid;
      if (rel < width) single(rel, std::false_type());
    } else {
      for (unsigned rel = tid; rel < width; rel += THREADS) single(rel, std::true_type());
    }
    if constexpr (HIST) __syncthreads();  // the next item clears the counts
  }
}

// Short rows without a history: a thread takes a piece, or the k % kPer last categories, of any row.
template <class T, class B, bool BWD> __global__ __launch_bounds__(256) void k_logits_adjust_short(const AdjustArgs a, int pieces) {
  typedef typename T::comp comp;
  typedef typename T::store store;
  constexpr int N = kPer<T>;
  const int nv = (int)(a.k / N), k = (int)a.k;
  const long long all = a.rows * pieces, step = (long long)gridDim.x * 256;
  for (long long p = (long long)blockIdx.x * 256 + threadIdx.x; p < all; p += step) {
    const long long row = all <= 0xffffffffll ? (unsigned)p / (unsigned)pieces : p / pieces;
    const int i = (int)(p - row * pieces);
    const store* src = static_cast<const store*>(a.src) + row * a.src_ld;
    const comp inv_t = reciprocal<comp>(a.temp, row);
    comp s[N], b[N];
    bool ok[N];
    if (i < nv) {
      unpack<T>(load_raw<T>(src + i * N), s);
      MaskPiece<T> mask;
      mask.load(a, row, 0, i * N);
#pragma unroll
      for (int e = 0; e < N; ++e) ok[e] = mask(a, e);
      BiasPiece<T, typename std::conditional<BWD, void, B>::type> bias;
      bias.load(a, row, 0, i * N);
      bias.add_to(s);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int v = i * N + e;
        if (v >= k) continue;
        s[e] = (comp)src[v];
        ok[e] = allowed(a, row, v);
        if constexpr (!BWD && !std::is_void<B>::value)
          s[e] += (comp) static_cast<const typename B::store*>(a.bias)[row * a.bias_ld + v];
      }
    }
    divide(s, a.temp, row, inv_t);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int v = i * N + e;
      if (v < k) b[e] = ok[e] ? s[e] : BWD ? (comp)0 : (comp)-kInf;
    }
    if constexpr (BWD && !std::is_void<B>::value) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i * N + e < k) static_cast<typename B::store*>(a.dbias)[row * a.k + i * N + e] = (typename B::store)b[e];
    }
    if (a.dst) {
      store* dst = static_cast<store*>(a.dst) + row * a.dst_ld + i * N;
      if (i < nv) {
        *reinterpret_cast<raw_t<T>*>(dst) = pack<T>(b);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i * N + e < k) dst[e] = (store)b[e];
      }
    }
  }
}

// Gradient of a bias that all rows share.  A workgroup of G groups of CT threads takes CT * kPer columns and a block of rows;
// a thread owns kPer columns and every G-th row of the block, so that the column sums stay in its registers (float64) and
// kSumRows rows are in flight; the groups are joined in LDS, the row blocks by k_logits_cols_final, all in a fixed order.
// Without a history the gradient of the logits is written on the way.  4096 x 32768 bf16 with a mask: 123 us, 5.5 TB/s.
constexpr int kSumThreads = 512, kSumRows = 4;

template <class T, int CT, bool WRITE>
__global__ __launch_bounds__(kSumThreads) void k_logits_adjust_cols(const AdjustArgs a, int chunks,
                                                                                 int row_blocks, double* __restrict__ partials) {
  constexpr int N = kPer<T>;
  constexpr int G = kSumThreads / CT;
  typedef typename T::comp comp;
  typedef typename T::store store;
  __shared__ double joined[G - 1][N][CT];
  const int col = threadIdx.x % CT, group = threadIdx.x / CT;
  const int nv = (int)(a.k / N), tail = (int)(a.k - (long long)nv * N);
  const int chunk = blockIdx.x % chunks, rb = blockIdx.x / chunks;
  const int i = chunk * CT + col;  // the piece, or (from nv on) a single category of the tail
  const long long lo = a.rows * rb / row_blocks, hi = a.rows * (rb + 1) / row_blocks;
  double acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.0;
  bool all_normal = true;
  if (i < nv) {
    const long long v = (long long)i * N;
    for (long long first = lo + group; first < hi; first += G * kSumRows) {
      raw_t<T> raw[kSumRows];
      MaskPiece<T> mask[kSumRows];
      comp inv_t[kSumRows];
#pragma unroll
      for (int r = 0; r < kSumRows; ++r) {
        const long long row = first + r * G;
        if (row >= hi) continue;
        raw[r] = __builtin_nontemporal_load(reinterpret_cast<const raw_t<T>*>(static_cast<const store*>(a.src) + row * a.src_ld + v));
        mask[r].load(a, row, 0, (unsigned)v);
        inv_t[r] = reciprocal<comp>(a.temp, row);
        all_normal = all_normal && normal(inv_t[r]);
      }
#pragma unroll
      for (int r = 0; r < kSumRows; ++r) {
        const long long row = first + r * G;
        if (row >= hi) continue;
        comp s[N];
        unpack<T>(raw[r], s);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          s[e] = mask[r](a, e) ? s[e] * inv_t[r] : (comp)0;
          acc[e] += (double)s[e];
        }
        if constexpr (WRITE) store_raw_nt<T>(static_cast<store*>(a.dst) + row * a.dst_ld + v, pack<T>(s));
      }
    }
  }
  // Temperatures without a normal reciprocal: the thread's rows once more.  (A branch in the loop above keeps the rows' loads
  // from overlapping: 4096 x 32768 bf16 132 against 126 us; a look at the temperatures before it costs 1.2 us.)
  if (__builtin_expect(i < nv && !all_normal, false)) {
    const long long v = (long long)i * N;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0;
    for (long long row = lo + group; row < hi; row += G) {
      const Factor<comp> t(row_operand(a.temp, row));
      MaskPiece<T> mask;
      mask.load(a, row, 0, (unsigned)v);
      comp s[N];
      unpack<T>(load_raw<T>(static_cast<const store*>(a.src) + row * a.src_ld + v), s);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        s[e] = mask(a, e) ? t.over(s[e]) : (comp)0;
        acc[e] += (double)s[e];
      }
      if constexpr (WRITE) store_raw_nt<T>(static_cast<store*>(a.dst) + row * a.dst_ld + v, pack<T>(s));
    }
  }
  if (i >= nv && i - nv < tail) {
    const long long v = (long long)nv * N + (i - nv);
    for (long long row = lo + group; row < hi; row += G) {
      const comp g = (comp) static_cast<const store*>(a.src)[row * a.src_ld + v];
      const comp s = allowed(a, row, v) ? Factor<comp>(row_operand(a.temp, row)).over(g) : (comp)0;
      acc[0] += (double)s;
      if constexpr (WRITE) static_cast<store*>(a.dst)[row * a.dst_ld + v] = (store)s;
    }
  }
  if (group > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) joined[group - 1][e][col] = acc[e];
  }
  __syncthreads();
  if (group == 0) {
#pragma unroll 4
    for (int g = 0; g < G - 1; ++g)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += joined[g][e][col];
    double* out = partials + (long long)rb * a.k;
    if (i < nv) {
#pragma unroll
      for (int e = 0; e < N; ++e) out[(long long)i * N + e] = acc[e];
    } else if (i - nv < tail) {
      out[(long long)nv * N + (i - nv)] = acc[0];
    }
  }
}

// Sums the row blocks: 64 columns by 4 groups of row blocks a workgroup, joined in order
template <class T>
__global__ __launch_bounds__(256) void k_logits_cols_final(const double* __restrict__ partials, long long k, int row_blocks,
                                                           void* __restrict__ out, int odt) {
  __shared__ double joined[4][64];
  const int col = threadIdx.x & 63, group = threadIdx.x >> 6;
  const long long v = (long long)blockIdx.x * 64 + col;
  double s = 0.0;
  if (v < k) {
#pragma unroll 4
    for (int b = group; b < row_blocks; b += 4) s += partials[(long long)b * k + v];
  }
  joined[group][col] = s;
  __syncthreads();
  if (group != 0 || v >= k) return;
  s = ((joined[0][col] + joined[1][col]) + joined[2][col]) + joined[3][col];
  if (odt == T::kCode) static_cast<typename T::store*>(out)[v] = (typename T::store)s;
  else static_cast<float*>(out)[v] = (float)s;
}

// ----------------------------------------------------------------------------------------- log-density
// exp(d) for d <= 0 or NaN (d = z - maximum): 2^(d log2 e).  The roundings of d, of log2 e (0.23 of half a step) and of their
// product change the result by up to 2.3 * 2^-24 |d| of it, so the sum of a row by 2.3 * 2^-24 times the mean of |d| under the
// softmax (8 where 131071 logits lie 8 below the maximum); exp(0) is 1.  Results below 2^-126 are 0.  (One fused multiply-add
// from z to the exponent saves an operation per element and no time, and the maximum's own exp is then off 1 by the rounding of
// its product.)
M355_DEV float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * 1.44269502f); }
M355_DEV double exp_neg(double d) { return ::exp(d); }
M355_DEV float log_c(float v) { return ::logf(v); }
M355_DEV double log_c(double v) { return ::log(v); }

struct DensityArgs {
  long long rows, k;
  const void* z;
  long long z_ld;
  const void* x;
  int x_dtype;
  void* lp;  // rows values of the arithmetic type
  DevOperand weight;
  void* grad;  // NULL: value only
  long long grad_ld;
};

// The observation of a row as a category, or -1
M355_DEV long long observed(const DensityArgs& a, long long row) {
  if (a.x_dtype == M355_I64 || a.x_dtype == M355_I32) {
    const long long i = a.x_dtype == M355_I64 ? static_cast<const long long*>(a.x)[row]
                                              : (long long)static_cast<const int*>(a.x)[row];
    return i >= 0 && i < a.k ? i : -1;
  }
  const double v = load1(a.x, a.x_dtype, (unsigned long long)row);
  return v >= 0.0 && v < (double)a.k && v == floor_(v) ? (long long)v : -1;
}

M355_DEV float max_c(float a, float b) { return __builtin_fmaxf(a, b); }  // a NaN is left out: the sum holds it
M355_DEV double max_c(double a, double b) { return __builtin_fmax(a, b); }
template <class C> M355_DEV C finite_max(C m) { return m == (C)-kInf ? (C)0 : m; }

// (m, s) of two parts of a row: the running maximum and the sum of exp(z - m), with m taken as 0 where a part is all -inf
template <class C> M355_DEV void join(C& m, C& s, C m2, C s2) {
  const C mm = max_c(m, m2);
  const C b = finite_max(mm);
  s = s * exp_neg(m - b) + s2 * exp_neg(m2 - b);
  m = mm;
}

// log-density from the row's statistics; -inf for an observation that is no category and for a row that is all -inf
template <class C> M355_DEV C density(C zx, C m, C s, bool inside) {
  return !inside || s == (C)0 ? (C)-kInf : (zx - finite_max(m)) - log_c(s);
}

template <class C> M355_DEV C wave_max(C v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max_c(v, (C)__shfl_xor(v, o, 64));
  return v;
}
template <class C> M355_DEV C wave_sum(C v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += (C)__shfl_xor(v, o, 64);
  return v;
}

// The thread's piece of the j-th round of THREADS pieces: a uniform address plus a 32-bit offset that all rounds share
template <class T, int THREADS> M355_DEV const raw_t<T>* piece(const typename T::store* row, int j) {
  return reinterpret_cast<const raw_t<T>*>(reinterpret_cast<const char*>(row) + (size_t)j * (THREADS * 16) +
                                           (unsigned)threadIdx.x * 16u);
}
template <class T, int THREADS> M355_DEV raw_t<T>* piece(typename T::store* row, int j) {
  return reinterpret_cast<raw_t<T>*>(reinterpret_cast<char*>(row) + (size_t)j * (THREADS * 16) + (unsigned)threadIdx.x * 16u);
}

template <class T> M355_DEV raw_t<T> raw_lowest() {  // kPer times -inf
  typename T::comp t[kPer<T>];
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) t[e] = (typename T::comp)-kInf;
  return pack<T>(t);
}

// Keeps the compiler from carrying the unpacked elements of one pass over the registers into the next (twice the
// registers for 16-bit types, which then spill): to it the pieces may have changed.  No instruction.
template <class T> M355_DEV void repack(raw_t<T>& r) {
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  u4 v = {r.x, r.y, r.z, r.w};
  asm volatile("" : "+v"(v));
  r.x = v.x, r.y = v.y, r.z = v.z, r.w = v.w;
}

// Value and gradient, one row per workgroup: z[x] - m - log s and w ([v = x] - exp(z - m) / s), m the row's maximum, s its sum
// of exp(z - m).  The row is read once: its first NR * THREADS 16-byte pieces wait in registers,
// the next NL * THREADS in LDS, while maximum and sum are formed; what does not fit there is summed as it passes and read
// again for the gradient.  The k % kPer last elements belong to the first threads, one each.  In place (grad == z): a row is
// read before it is written, but for the pieces that are read again, which the same thread reads and writes.  Bound by HBM and
// by how far the phases (load, sum, store) of the workgroups of a CU overlap: 4096 x 131072 bf16, an eighth of the rows padding,
// 401 us (5.0 TB/s of what has to move, where a copy reaches 6.5), 1500 x 100003 float32 247 us.
template <class T, int THREADS, int NR, int NL, int WAVES, bool REST>
__global__ __launch_bounds__(THREADS, WAVES) void k_logits_grad(const DensityArgs a) {
  typedef typename T::comp comp;
  typedef typename T::store store;
  constexpr int N = kPer<T>;
  constexpr int W = THREADS / 64;
  constexpr bool kKeepExp = sizeof(comp) == sizeof(store);  // exp(z) has room where z was (16 bits would not hold it)
  constexpr int U = 4;  // loads in flight per thread of what passes by
  __shared__ comp red[2][W];
  __shared__ uint4 kept[NL ? NL * THREADS : 1];
  const int tid = threadIdx.x, nv = (int)(a.k / N), tail = (int)(a.k - (long long)nv * N);
  const raw_t<T> lowest = raw_lowest<T>();
  auto load = [&](const store* z, int j, int count) {
    return tid < count - j * THREADS ? __builtin_nontemporal_load(piece<T, THREADS>(z, j)) : lowest;
  };
  // the number of pieces anew for every pass: the comparisons with it are cheaper than 2 * NR scalar registers to keep them
  auto fresh = [](int count) {
    asm volatile("" : "+s"(count));
    return count;
  };
  auto to_lds = [&](int l, raw_t<T> r) { kept[l * THREADS + tid] = uint4{r.x, r.y, r.z, r.w}; };
  auto from_lds = [&](int l) {  // a thread reads what it wrote itself: no barrier
    const uint4 u = kept[l * THREADS + tid];
    raw_t<T> r;
    r.x = u.x, r.y = u.y, r.z = u.z, r.w = u.w;
    return r;
  };
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const store* z = static_cast<const store*>(a.z) + row * a.z_ld;
    store* g = static_cast<store*>(a.grad) + row * a.grad_ld;
    const double wd = row_operand(a.weight, row);
    const comp w = (comp)wd;
    const long long xi = observed(a, row);
    if (wd == 0.0 || xi < 0) {  // the gradient is 0 whatever the row holds: it is not read
      raw_t<T> none;
      none.x = none.y = none.z = none.w = 0;
      for (int i = tid; i < nv; i += THREADS) __builtin_nontemporal_store(none, reinterpret_cast<raw_t<T>*>(g + (long long)i * N));
      if (tid < tail) g[(long long)nv * N + tid] = (store)0;
      if (tid == 0) static_cast<comp*>(a.lp)[row] = (comp)-kInf;  // left out of the total where the weight is 0
      continue;
    }
    raw_t<T> raw[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) raw[j] = load(z, j, nv);
    const comp zx = (comp)z[xi];
    const comp last = tid < tail ? (comp)z[(long long)nv * N + tid] : (comp)-kInf;
#pragma unroll U
    for (int l = 0; l < NL; ++l) to_lds(l, load(z, NR + l, nv));
    comp m = last, s = 0;
    comp ms = (comp)-kInf;  // maximum of what passes by; s is its sum
    for (int base = (NR + NL) * THREADS + tid; REST && base < nv; base += U * THREADS) {
      raw_t<T> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = base + u * THREADS < nv ? load_raw<T>(z + (long long)(base + u * THREADS) * N) : lowest;
      comp mt = ms;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        comp t[N];
        unpack<T>(r[u], t);
#pragma unroll
        for (int e = 0; e < N; ++e) mt = max_c(mt, t[e]);
      }
      const comp b = finite_max(mt);
      s *= exp_neg(ms - b);
      ms = mt;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        comp t[N];
        repack<T>(r[u]);
        unpack<T>(r[u], t);
#pragma unroll
        for (int e = 0; e < N; ++e) s += exp_neg(t[e] - b);
      }
    }
    m = max_c(m, ms);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      comp t[N];
      unpack<T>(raw[j], t);
#pragma unroll
      for (int e = 0; e < N; ++e) m = max_c(m, t[e]);
    }
#pragma unroll 2
    for (int l = 0; l < NL; ++l) {
      comp t[N];
      unpack<T>(from_lds(l), t);
#pragma unroll
      for (int e = 0; e < N; ++e) m = max_c(m, t[e]);
    }
    m = wave_max(m);
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = max_c(m, red[0][i]);
    const comp b = finite_max(m);
    s = REST ? s * exp_neg(ms - b) + exp_neg(last - b) : exp_neg(last - b);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      comp t[N];
      repack<T>(raw[j]);
      unpack<T>(raw[j], t);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        t[e] = exp_neg(t[e] - b);
        s += t[e];
      }
      if constexpr (kKeepExp) raw[j] = pack<T>(t);
    }
#pragma unroll 2
    for (int l = 0; l < NL; ++l) {
      comp t[N];
      unpack<T>(from_lds(l), t);
#pragma unroll
      for (int e = 0; e < N; ++e) s += exp_neg(t[e] - b);
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) red[1][tid >> 6] = s;
    __syncthreads();  // red[0] is written again only behind this barrier, red[1] behind the next row's first
    s = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) s += red[1][i];
    if (tid == 0) static_cast<comp*>(a.lp)[row] = density(zx, m, s, true);
    const bool zero = s == (comp)0;  // all -inf: every exp(z) is 0
    const comp q = zero ? (comp)0 : -w / s;
    auto gradient = [&](raw_t<T> r) {
      comp t[N];
      unpack<T>(r, t);
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] = exp_neg(t[e] - b) * q;
      return pack<T>(t);
    };
    auto times = [](raw_t<T> r, comp f) {
      comp t[N];
      unpack<T>(r, t);
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] *= f;
      return pack<T>(t);
    };
    const int here = fresh(nv);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      if constexpr (!kKeepExp) repack<T>(raw[j]);
      if (tid < here - j * THREADS)
        __builtin_nontemporal_store(kKeepExp ? times(raw[j], q) : gradient(raw[j]), piece<T, THREADS>(g, j));
    }
#pragma unroll 2
    for (int l = 0; l < NL; ++l)
      if (tid < here - (NR + l) * THREADS) __builtin_nontemporal_store(gradient(from_lds(l)), piece<T, THREADS>(g, NR + l));
    for (int base = (NR + NL) * THREADS + tid; REST && base < nv; base += U * THREADS) {
      raw_t<T> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = base + u * THREADS < nv ? load_raw<T>(z + (long long)(base + u * THREADS) * N) : lowest;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (base + u * THREADS < nv)
          __builtin_nontemporal_store(gradient(r[u]), reinterpret_cast<raw_t<T>*>(g + (long long)(base + u * THREADS) * N));
    }
    if (tid < tail) g[(long long)nv * N + tid] = (store)(exp_neg(last - b) * q);
    if (!zero) {  // the observation's own element, by the thread that wrote it: after that store
      const long long vi = xi / N;
      if (vi < nv ? (int)(vi % THREADS) == tid : (int)(xi - (long long)nv * N) == tid) g[xi] = (store)(exp_neg(zx - b) * q + w);
    }
  }
}

// Short rows (k <= kShort * G): G lanes per row, at most kShort elements a lane, all in registers; a wavefront takes 64 / G
// rows, there is nothing to wait for but the loads.  10^6 rows of 10 float32: 19 us (value), 31 us (with the gradient).  (A
// workgroup of 256 threads per short row does little but start: 2 * 10^5 rows of 600 bf16 took 660 us that way, and take
// 117 us with a wavefront per row.)
constexpr int kShort = 8;
template <class T, int G, bool GRAD> __global__ __launch_bounds__(256) void k_logits_short(const DensityArgs a) {
  typedef typename T::comp comp;
  typedef typename T::store store;
  constexpr int kRows = 256 / G;
  const int l = threadIdx.x % G, k = (int)a.k;
  for (long long row = (long long)blockIdx.x * kRows + threadIdx.x / G; row < a.rows; row += (long long)gridDim.x * kRows) {
    const store* z = static_cast<const store*>(a.z) + row * a.z_ld;
    const long long xi = observed(a, row);
    const double wd = GRAD ? row_operand(a.weight, row) : 1.0;
    comp v[kShort];
#pragma unroll
    for (int j = 0; j < kShort; ++j) v[j] = j * G + l < k ? (comp)z[j * G + l] : (comp)-kInf;
    const comp zx = xi >= 0 ? (comp)z[xi] : (comp)0;
    comp m = v[0];
#pragma unroll
    for (int j = 1; j < kShort; ++j) m = max_c(m, v[j]);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = max_c(m, (comp)__shfl_xor(m, o, 64));
    const comp b = finite_max(m);
    comp s = 0;
#pragma unroll
    for (int j = 0; j < kShort; ++j) {
      v[j] = exp_neg(v[j] - b);
      s += v[j];
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) s += (comp)__shfl_xor(s, o, 64);
    if (l == 0) static_cast<comp*>(a.lp)[row] = density(zx, m, s, xi >= 0);
    if constexpr (GRAD) {
      store* g = static_cast<store*>(a.grad) + row * a.grad_ld;
      const bool zero = wd == 0.0 || xi < 0 || s == (comp)0;
      const comp w = (comp)wd, q = zero ? (comp)0 : -w / s;
#pragma unroll
      for (int j = 0; j < kShort; ++j)
        if (j * G + l < k) g[j * G + l] = (store)(zero ? (comp)0 : v[j] * q + (j * G + l == xi ? w : (comp)0));
    }
  }
}

// Value only: one row per workgroup, tiles of NR 16-byte loads per thread with a running maximum and sum.  Bound by HBM:
// 8192 x 32768 float16 in 85 us, 6.3 TB/s, a call among others (a launch that a profiler times by itself: 92-98 us).
template <class T, int THREADS, int NR>
__global__ __launch_bounds__(THREADS) void k_logits_value(const DensityArgs a) {
  constexpr int N = kPer<T>;
  constexpr int W = THREADS / 64;
  typedef typename T::comp comp;
  typedef typename T::store store;
  __shared__ comp red[2][W];
  const int tid = threadIdx.x, nv = (int)(a.k / N), tail = (int)(a.k - (long long)nv * N);
  const raw_t<T> lowest = raw_lowest<T>();
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const store* z = static_cast<const store*>(a.z) + row * a.z_ld;
    const long long xi = observed(a, row);
    const comp zx = xi >= 0 ? (comp)z[xi] : (comp)0;
    comp m = tid < tail ? (comp)z[(long long)nv * N + tid] : (comp)-kInf;
    comp s = exp_neg(m - finite_max(m));
    for (int base = 0; base < nv; base += NR * THREADS) {
      raw_t<T> raw[NR];
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const int i = base + j * THREADS + tid;
        raw[j] = i < nv ? load_raw_nt<T>(z + (long long)i * N) : lowest;
      }
      comp mt = m;
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        comp t[N];
        unpack<T>(raw[j], t);
#pragma unroll
        for (int e = 0; e < N; ++e) mt = max_c(mt, t[e]);
      }
      const comp b = finite_max(mt);
      s *= exp_neg(m - b);
      m = mt;
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        comp t[N];
        repack<T>(raw[j]);
        unpack<T>(raw[j], t);
#pragma unroll
        for (int e = 0; e < N; ++e) s += exp_neg(t[e] - b);
      }
    }
    comp mm = wave_max(m);
    s = wave_sum(s * exp_neg(m - finite_max(mm)));
    if ((tid & 63) == 0) {
      red[0][tid >> 6] = mm;
      red[1][tid >> 6] = s;
    }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int i = 1; i < W; ++i) join<comp>(mm, s, red[0][i], red[1][i]);
      static_cast<comp*>(a.lp)[row] = density(zx, mm, s, xi >= 0);
    }
    __syncthreads();
  }
}

// total = sum over rows of w * lp in a fixed order; a row of weight 0 is left out whatever its density.  Workgroup b of many
// sums its share of the rows into partials[b] (lp, weight given), a last one the partials (lp NULL).
constexpr int kTotalRows = 8192;  // rows from which more than one workgroup sums
constexpr int kTotalBlocks = 512;
template <class C>
__global__ __launch_bounds__(1024) void k_logits_total(const C* __restrict__ lp, DevOperand weight, long long rows,
                                                       double* __restrict__ partials, C* __restrict__ total) {
  __shared__ double red[16];
  const long long lo = rows * blockIdx.x / gridDim.x, hi = rows * (blockIdx.x + 1) / gridDim.x;
  double acc = 0.0;
  for (long long base = lo + threadIdx.x; base < hi; base += 4096) {
    double w[4], v[4];  // four rows' loads together: the launch is all latency
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = base + j * 1024;
      w[j] = r >= hi ? 0.0 : lp ? row_operand(weight, r) : 1.0;
      v[j] = r >= hi ? 0.0 : lp ? (double)lp[r] : partials[r];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (w[j] != 0.0) acc += w[j] * v[j];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_down(acc, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) acc += red[i];
    if (total) total[0] = (C)acc;
    else partials[blockIdx.x] = acc;
  }
}

// ---------------------------------------------------------------------------------------------- launches
constexpr long long kMaxGrid = 1ll << 21;  // workgroups (the launch counts threads in 32 bits); kernels walk on from there

template <class T, int THREADS, int VPT, class CNT, class B, bool BWD> void launch_adjust(const AdjustArgs& a, hipStream_t s) {
  const long long nv = a.k / kPer<T>;
  AdjustGrid g;
  g.chunks = (int)((nv + THREADS * VPT - 1) / (THREADS * VPT));
  if (g.chunks < 1) g.chunks = 1;
  g.per = (int)((nv + g.chunks - 1) / g.chunks);  // chunks of one size
  if (g.per > 0) g.chunks = (int)((nv + g.per - 1) / g.per);  // and none that is empty
  g.rows_by_xcd = a.rows >= 64;
  g.items = (g.rows_by_xcd ? (a.rows + 7) / 8 * 8 : a.rows) * g.chunks;
  hipLaunchKernelGGL((k_logits_adjust<T, THREADS, VPT, CNT, B, BWD>), dim3((unsigned)(g.items < kMaxGrid ? g.items : kMaxGrid)),
                     dim3(THREADS), 0, s, a, g);
}

template <class T, class B, bool BWD> void launch_adjust(const AdjustArgs& a, hipStream_t s) {
  // Four pieces per thread hide the latencies of a chunk behind each other; where that gives too few workgroups for 256
  // CUs, one piece each (1 x 32768 bf16, 300 ids: 4.4 against 5.4 us).  512 threads halve how often a history is scanned:
  // slower with a short one (512 x 131072 bf16, 500 ids: 77 against 71 us), 3 % faster with 8000 ids (256 x 65536: 41.0 against
  // 42.3 us), which is not worth a second form.
  const bool few = a.rows * (a.k / kPer<T>) < 256ll * 1024;
  if (!a.history && a.k / kPer<T> < 256) {  // a workgroup per row would be half empty
    const int pieces = (int)((a.k + kPer<T> - 1) / kPer<T>);
    const long long want = (a.rows * pieces + 255) / 256;
    hipLaunchKernelGGL((k_logits_adjust_short<T, B, BWD>), dim3((unsigned)(want < kMaxGrid ? want : kMaxGrid)), dim3(256), 0,
                       s, a, pieces);
    return;
  }
  if (!a.history) few ? launch_adjust<T, 256, 1, void, B, BWD>(a, s) : launch_adjust<T, 256, 4, void, B, BWD>(a, s);
  else if (a.history_len > 32767) launch_adjust<T, 256, 4, unsigned, B, BWD>(a, s);
  else if (few) launch_adjust<T, 256, 1, unsigned short, B, BWD>(a, s);
  else launch_adjust<T, 256, 4, unsigned short, B, BWD>(a, s);
}

// forward: with the bias, if there is one; gradient: with a bias' gradient that goes out per element
template <class T, bool BWD> void launch_adjust(const AdjustArgs& a, hipStream_t s) {
  if (!(BWD ? a.dbias : a.bias)) launch_adjust<T, void, BWD>(a, s);
  else if (a.bias_dtype == T::kCode) launch_adjust<T, T, BWD>(a, s);
  else if constexpr (kPer<T> == 8) launch_adjust<T, F32, BWD>(a, s);
}

// Shape of k_logits_adjust_cols: threads per group by the row's length, about four workgroups per CU, at least one round of
// rows in flight each
struct ColumnGrid {
  int ct, chunks, row_blocks;
};
template <class T> ColumnGrid column_grid(long long rows, long long k) {
  const long long columns = k / kPer<T> + k % kPer<T>;  // pieces, and categories of the tail
  ColumnGrid g;
  g.ct = columns <= 8 ? 8 : columns <= 32 ? 32 : 128;
  g.chunks = (int)((columns + g.ct - 1) / g.ct);
  long long rb = 1024 / g.chunks;
  const long long most = rows / (kSumThreads / g.ct * kSumRows);
  if (rb > most) rb = most;
  g.row_blocks = (int)(rb < 1 ? 1 : rb);
  return g;
}

template <class T> void launch_cols_final(const AdjustArgs& a, const double* ws, int row_blocks, void* dbias, hipStream_t s) {
  hipLaunchKernelGGL((k_logits_cols_final<T>), dim3((unsigned)((a.k + 63) / 64)), dim3(256), 0, s, ws, a.k, row_blocks, dbias,
                     a.bias_dtype);
}
template <class T> void launch_adjust_cols(const AdjustArgs& a, void* dbias, double* ws, hipStream_t s) {
  const ColumnGrid g = column_grid<T>(a.rows, a.k);
  const dim3 grid((unsigned)((long long)g.chunks * g.row_blocks)), block(kSumThreads);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a, g.chunks, g.row_blocks, ws); };
  if (g.ct == 8) a.dst ? launch(k_logits_adjust_cols<T, 8, true>) : launch(k_logits_adjust_cols<T, 8, false>);
  else if (g.ct == 32) a.dst ? launch(k_logits_adjust_cols<T, 32, true>) : launch(k_logits_adjust_cols<T, 32, false>);
  else a.dst ? launch(k_logits_adjust_cols<T, 128, true>) : launch(k_logits_adjust_cols<T, 128, false>);
  launch_cols_final<T>(a, ws, g.row_blocks, dbias, s);
}

template <class T, int THREADS, int NR, int NL, int WAVES, bool REST> void launch_grad(const DensityArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_logits_grad<T, THREADS, NR, NL, WAVES, REST>),
                     dim3((unsigned)(a.rows < kMaxGrid ? a.rows : kMaxGrid)), dim3(THREADS), 0, s, a);
}

template <class T, int G, bool GRAD> void launch_short(const DensityArgs& a, hipStream_t s) {
  const long long want = (a.rows * G + 255) / 256;
  hipLaunchKernelGGL((k_logits_short<T, G, GRAD>), dim3((unsigned)(want < kMaxGrid ? want : kMaxGrid)), dim3(256), 0, s, a);
}

// Lanes per short row; pieces per thread and threads per workgroup by the length of longer ones.  Gradient, measured for
// bf16 (reads and writes at 5.0-5.7 TB/s; a copy reaches 6.5): four pieces per thread beat eight of half the threads while a
// row fits 1024 threads (8192 x 32768: 194 against 208 us), then two workgroups of 512 threads a CU beat one of 1024 (4096 x
// 131072: 415 against 437-450 us) although they read half of the row twice; rows over 256 KiB take one workgroup a CU again
// (float32, 1500 x 100003: 256 against 277 us), as less of them is read twice.  Value: enough rows fill the chip with 256
// threads each, few rows take 1024 (8 x 50021 float32: 7 against 17 us).
template <class T, bool GRAD> void launch_density(const DensityArgs& a, hipStream_t s) {
  const long long nv = a.k / kPer<T>;
  if (a.k <= kShort * 4) return launch_short<T, 4, GRAD>(a, s);
  if (a.k <= kShort * 16) return launch_short<T, 16, GRAD>(a, s);
  if (a.k <= kShort * 64) return launch_short<T, 64, GRAD>(a, s);
  if constexpr (GRAD && sizeof(typename T::store) == 8) {  // float64 arithmetic takes registers from the row
    if (nv <= 64 * 4) launch_grad<T, 64, 4, 0, 4, false>(a, s);
    else if (nv <= 256 * 4) launch_grad<T, 256, 4, 0, 4, false>(a, s);
    else if (nv <= 512 * 4) launch_grad<T, 512, 4, 0, 4, false>(a, s);
    else if (nv <= 1024 * 4) launch_grad<T, 1024, 4, 0, 4, false>(a, s);
    else launch_grad<T, 1024, 6, 6, 4, true>(a, s);
  } else if constexpr (GRAD) {
    if (nv <= 64 * 4) launch_grad<T, 64, 4, 0, 4, false>(a, s);
    else if (nv <= 256 * 4) launch_grad<T, 256, 4, 0, 8, false>(a, s);
    else if (nv <= 512 * 4) launch_grad<T, 512, 4, 0, 4, false>(a, s);
    else if (nv <= 1024 * 4) launch_grad<T, 1024, 4, 0, 8, false>(a, s);
    else if (nv <= 512 * 16) launch_grad<T, 512, 16, 0, 4, false>(a, s);
    else if (nv <= 512 * 32) launch_grad<T, 512, 16, 0, 4, true>(a, s);
    else launch_grad<T, 1024, 8, 4, 4, true>(a, s);
  } else {
    const dim3 grid((unsigned)(a.rows < kMaxGrid ? a.rows : kMaxGrid));
    if (nv <= 64 * 4) hipLaunchKernelGGL((k_logits_value<T, 64, 4>), grid, dim3(64), 0, s, a);
    else if (nv <= 256 * 4) hipLaunchKernelGGL((k_logits_value<T, 256, 4>), grid, dim3(256), 0, s, a);
    else if (a.rows >= 1024) hipLaunchKernelGGL((k_logits_value<T, 256, 8>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_logits_value<T, 1024, 8>), grid, dim3(1024), 0, s, a);
  }
}

template <class F> int by_dtype(int dtype, F f) {
  switch (dtype) {
    case M355_F64: return f(F64());
    case M355_F32: return f(F32());
    case M355_F16: return f(F16());
    case M355_BF16: return f(BF16());
  }
  return fail(M355_ERR_INVALID, "logits are float64, float32, float16 or bfloat16 (dtype %d)", dtype);
}

}  // namespace m355

namespace {
using m355::fail;

int launched() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? M355_OK : fail(M355_ERR_LAUNCH, "HIP launch failed: %s", hipGetErrorString(e));
}

int check_rows(int64_t rows, int64_t k, int dtype) {
  if (rows < 0) return fail(M355_ERR_INVALID, "rows must be >= 0");
  if (k < 1 || k > INT32_MAX) return fail(M355_ERR_INVALID, "1 <= k < 2^31 categories, got %lld", (long long)k);
  return m355::by_dtype(dtype, [](auto) { return 0; });
}

int row_arg(const m355_operand& in, int64_t rows, m355::DevOperand& out, const char* what) {
  out.ptr = in.ptr;
  out.scalar = in.scalar;
  out.dtype = in.dtype;
  out.div = 1;
  out.mod = 1;
  if (!in.ptr) return 0;
  if (in.dtype != M355_F64 && in.dtype != M355_F32) return fail(M355_ERR_INVALID, "%s: float64 or float32", what);
  if (in.div < 1 || in.mod < 1) return fail(M355_ERR_INVALID, "%s: div and mod must be >= 1", what);
  out.div = (unsigned long long)in.div;
  out.mod = in.div >= rows ? 1 : (unsigned long long)in.mod;
  if (out.div == 1 && out.mod >= (unsigned long long)rows) out.mod = 0;  // one value per row: no division per access
  return 0;
}

int check_adjust(int64_t rows, int64_t k, int dtype, const m355_logit_adjust* d, m355::AdjustArgs& a) {
  if (!d) return fail(M355_ERR_INVALID, "NULL adjustment");
  a = m355::AdjustArgs();
  a.rows = rows;
  a.k = k;
  if (d->history_len < 0 || d->history_len > INT32_MAX || d->history_stride < 0)
    return fail(M355_ERR_INVALID, "0 <= history_len < 2^31, history_stride >= 0");
  if (d->history && d->history_len) {
    if (d->history_dtype != M355_I64 && d->history_dtype != M355_I32)
      return fail(M355_ERR_INVALID, "history ids are int64 or int32");
    a.history = d->history;
  }
  a.history_ld = d->history_stride;
  a.history_len = (int)d->history_len;
  a.history_dtype = d->history_dtype;
  a.lengths = reinterpret_cast<const long long*>(d->lengths);
  a.prompts = reinterpret_cast<const long long*>(d->prompt_lengths);
  if (d->bias && d->bias_dtype != dtype && !(d->bias_dtype == M355_F32 && (dtype == M355_F16 || dtype == M355_BF16)))
    return fail(M355_ERR_INVALID, "the bias has the dtype of the logits, or float32 with 16-bit logits");
  if (d->bias_stride < 0 || d->mask_stride < 0) return fail(M355_ERR_INVALID, "negative stride");
  a.bias = d->bias;
  a.bias_ld = d->bias_stride;
  a.bias_dtype = d->bias_dtype;
  if (d->mask_kind < M355_MASK_NONE || d->mask_kind > M355_MASK_BITS || (d->mask_kind && !d->mask))
    return fail(M355_ERR_INVALID, "bad mask");
  a.mask_kind = d->mask_kind;
  a.mask = d->mask;
  a.mask_ld = d->mask_stride;
  int rc;
  if ((rc = row_arg(d->repetition, rows, a.rep, "repetition")) || (rc = row_arg(d->presence, rows, a.pres, "presence")) ||
      (rc = row_arg(d->frequency, rows, a.freq, "frequency")) ||
      (rc = row_arg(d->temperature, rows, a.temp, "temperature")))
    return rc;
  return 0;
}

int check_density(int64_t rows, int64_t k, int dtype, const void* logits, int64_t stride, const void* x, int x_dtype,
                  m355::DensityArgs& a) {
  const int rc = check_rows(rows, k, dtype);
  if (rc) return rc;
  if (x_dtype != M355_I64 && x_dtype != M355_I32 && x_dtype != M355_F64 && x_dtype != M355_F32)
    return fail(M355_ERR_INVALID, "observations are int64, int32, float64 or float32");
  if (stride < 0) return fail(M355_ERR_INVALID, "negative stride");
  if (rows && (!logits || !x)) return fail(M355_ERR_INVALID, "NULL pointer argument");
  a = m355::DensityArgs();
  a.rows = rows;
  a.k = k;
  a.z = logits;
  a.z_ld = stride;
  a.x = x;
  a.x_dtype = x_dtype;
  return 0;
}
}  // namespace

extern "C" int m355_logits_adjust(int64_t rows, int64_t k, int dtype, const void* logits, int64_t logits_stride,
                                  const m355_logit_adjust* adjust, void* out, int64_t out_stride, void* stream) {
  using namespace m355;
  AdjustArgs a;
  int rc = check_rows(rows, k, dtype);
  if (!rc) rc = check_adjust(rows, k, dtype, adjust, a);
  if (rc) return rc;
  if (logits_stride < 0 || (rows > 1 && out_stride < k)) return fail(M355_ERR_INVALID, "bad row stride");
  if (rows == 0) return M355_OK;
  if (!logits || !out) return fail(M355_ERR_INVALID, "NULL pointer argument");
  a.src = logits;
  a.src_ld = logits_stride;
  a.dst = out;
  a.dst_ld = out_stride;
  by_dtype(dtype, [&](auto t) { return launch_adjust<decltype(t), false>(a, static_cast<hipStream_t>(stream)), 0; });
  return launched();
}

extern "C" size_t m355_logits_adjust_grad_workspace_bytes(int64_t rows, int64_t k, int dtype) {
  if (rows < 1 || k < 1 || k > INT32_MAX) return 0;
  int rb = 0;
  m355::by_dtype(dtype, [&](auto t) { return (rb = m355::column_grid<decltype(t)>(rows, k).row_blocks), 0; });
  return (size_t)rb * (size_t)k * sizeof(double);
}

extern "C" int m355_logits_adjust_grad(int64_t rows, int64_t k, int dtype, const void* g, int64_t g_stride,
                                       const void* logits, int64_t logits_stride, const m355_logit_adjust* adjust,
                                       void* dlogits, void* dbias, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  using namespace m355;
  AdjustArgs a;
  int rc = check_rows(rows, k, dtype);
  if (!rc) rc = check_adjust(rows, k, dtype, adjust, a);
  if (rc) return rc;
  if (g_stride < 0 || logits_stride < 0) return fail(M355_ERR_INVALID, "bad row stride");
  if (dbias && !a.bias) return fail(M355_ERR_INVALID, "dbias without a bias");
  const bool shared = dbias && a.bias_ld == 0;
  if (shared && k > (INT64_C(1) << 28)) return fail(M355_ERR_INVALID, "gradient of a shared bias: at most 2^28 categories");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {  // no row blocks: a workspace is neither asked for nor read, and the sums are 0
    if (!shared) return M355_OK;
    by_dtype(dtype, [&](auto t) { return launch_cols_final<decltype(t)>(a, nullptr, 0, dbias, s), 0; });
    return launched();
  }
  if (!g || (dlogits && a.history && !logits)) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if (shared && (!workspace || workspace_bytes < m355_logits_adjust_grad_workspace_bytes(rows, k, dtype)))
    return fail(M355_ERR_WORKSPACE, "workspace too small");
  a.src = g;
  a.src_ld = g_stride;
  a.x = logits;
  a.x_ld = logits_stride;
  a.dst = dlogits;
  a.dst_ld = k;
  a.dbias = shared ? nullptr : dbias;
  by_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (shared) {
      AdjustArgs c = a;
      if (a.history) c.dst = nullptr;  // the row kernel writes the gradient of the logits
      launch_adjust_cols<T>(c, dbias, static_cast<double*>(workspace), s);
    }
    if ((a.dst && (!shared || a.history)) || a.dbias) launch_adjust<T, true>(a, s);
    return 0;
  });
  return launched();
}

extern "C" size_t m355_logits_workspace_bytes(int64_t rows, int64_t k, int dtype) {
  (void)k;
  (void)dtype;
  return ((size_t)(rows > 0 ? rows : 0) + m355::kTotalBlocks) * sizeof(double);
}

extern "C" int m355_logits_logpdf(int64_t rows, int64_t k, int dtype, const void* logits, int64_t logits_stride,
                                  const void* x, int x_dtype, void* out, void* stream) {
  using namespace m355;
  DensityArgs a;
  const int rc = check_density(rows, k, dtype, logits, logits_stride, x, x_dtype, a);
  if (rc) return rc;
  if (rows == 0) return M355_OK;
  if (!out) return fail(M355_ERR_INVALID, "NULL pointer argument");
  a.lp = out;
  by_dtype(dtype, [&](auto t) { return launch_density<decltype(t), false>(a, static_cast<hipStream_t>(stream)), 0; });
  return launched();
}

extern "C" int m355_logits_sum_logpdf_grad(int64_t rows, int64_t k, int dtype, const void* logits, int64_t logits_stride,
                                           const void* x, int x_dtype, const m355_operand* weights, void* total,
                                           void* dlogits, int64_t dlogits_stride, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  using namespace m355;
  DensityArgs a;
  int rc = check_density(rows, k, dtype, logits, logits_stride, x, x_dtype, a);
  if (rc) return rc;
  if (!weights || !total) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if ((rc = row_arg(*weights, rows, a.weight, "weights"))) return rc;
  if (dlogits && rows > 1 && dlogits_stride < k) return fail(M355_ERR_INVALID, "bad row stride");
  if (!workspace) return fail(M355_ERR_INVALID, "NULL pointer argument");
  if (workspace_bytes < m355_logits_workspace_bytes(rows, k, dtype)) return fail(M355_ERR_WORKSPACE, "workspace too small");
  a.lp = workspace;
  a.grad = dlogits;
  a.grad_ld = dlogits_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename T::comp comp;
    if (rows && dlogits) launch_density<T, true>(a, s);
    else if (rows) launch_density<T, false>(a, s);
    const comp* lp = static_cast<const comp*>(a.lp);
    comp* out = static_cast<comp*>(total);
    double* partials = static_cast<double*>(workspace) + rows;  // behind the densities
    if (rows <= kTotalRows) {
      hipLaunchKernelGGL((k_logits_total<comp>), dim3(1), dim3(1024), 0, s, lp, a.weight, (long long)rows, partials, out);
    } else {
      const long long want = (rows + 4095) / 4096;
      const int blocks = (int)(want < kTotalBlocks ? want : kTotalBlocks);
      hipLaunchKernelGGL((k_logits_total<comp>), dim3(blocks), dim3(1024), 0, s, lp, a.weight, (long long)rows, partials,
                         static_cast<comp*>(nullptr));
      hipLaunchKernelGGL((k_logits_total<comp>), dim3(1), dim3(1024), 0, s, static_cast<const comp*>(nullptr), a.weight,
                         (long long)blocks, partials, out);
    }
    return 0;
  });
  return launched();
}
