// Loads, stores and arithmetic types shared by the kernels on logits (m355_logits.hip) and on lists of gradients
// (m355_gradnorm.hip): 16 bytes per lane of float64 / float32 / float16 / bfloat16 at any element alignment (global
// accesses of gfx950 need no more than the element's own), unpacked to the type the arithmetic is done in.
#pragma once
#include <hip/hip_runtime.h>

#include "m355_elemwise.h"

namespace m355 {

// raw: 16 bytes of which only the element's own alignment is assured; comp: the type of the arithmetic
struct F64 {
  typedef unsigned raw __attribute__((ext_vector_type(4), aligned(8)));
  typedef double store;
  typedef double comp;
  static constexpr int kCode = M355_F64;
};
struct F32 {
  typedef unsigned raw __attribute__((ext_vector_type(4), aligned(4)));
  typedef float store;
  typedef float comp;
  static constexpr int kCode = M355_F32;
};
struct F16 {
  typedef unsigned raw __attribute__((ext_vector_type(4), aligned(2)));
  typedef _Float16 store;
  typedef float comp;
  static constexpr int kCode = M355_F16;
};
struct BF16 {
  typedef unsigned raw __attribute__((ext_vector_type(4), aligned(2)));
  typedef __bf16 store;
  typedef float comp;
  static constexpr int kCode = M355_BF16;
};

template <class T> constexpr int kPer = 16 / (int)sizeof(typename T::store);  // elements of one 16-byte access

template <class T> using raw_t = typename T::raw;

template <class T> M355_DEV raw_t<T> load_raw(const typename T::store* p) {
  return *reinterpret_cast<const raw_t<T>*>(p);
}
template <class T> M355_DEV raw_t<T> load_raw_nt(const typename T::store* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const raw_t<T>*>(p));
}
template <class T> M355_DEV void store_raw_nt(typename T::store* p, raw_t<T> v) {
  __builtin_nontemporal_store(v, reinterpret_cast<raw_t<T>*>(p));
}

template <class T> M355_DEV void unpack(raw_t<T> r, typename T::comp (&v)[kPer<T>]) {
  typedef typename T::store vec __attribute__((ext_vector_type(kPer<T>)));
  const unsigned u[4] = {r.x, r.y, r.z, r.w};
  vec s;
  __builtin_memcpy(&s, u, 16);
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) v[e] = (typename T::comp)s[e];
}
template <class T> M355_DEV raw_t<T> pack(const typename T::comp (&v)[kPer<T>]) {
  typedef typename T::store vec __attribute__((ext_vector_type(kPer<T>)));
  vec s;
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) s[e] = (typename T::store)v[e];
  unsigned u[4];
  __builtin_memcpy(u, &s, 16);
  raw_t<T> r;
  r.x = u[0];
  r.y = u[1];
  r.z = u[2];
  r.w = u[3];
  return r;
}

// A per-row argument: scalar, or float64 / float32 array indexed by the row (mod == 0) or by (row / div) % mod
M355_DEV double row_operand(const DevOperand& o, long long row) {
  if (!o.ptr) return o.scalar;
  const unsigned long long i = o.mod == 0 ? row : o.mod == 1 ? 0 : ((unsigned long long)row / o.div) % o.mod;
  return o.dtype == M355_F32 ? (double)static_cast<const float*>(o.ptr)[i] : static_cast<const double*>(o.ptr)[i];
}

}  // namespace m355
