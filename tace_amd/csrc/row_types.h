// Element types and row addressing of the row operators (rows.hip, dropout.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tace_rows.h"

int tace_fail_msg(const char* msg);   // tace_hip.hip
int tace_check_launch(const char* what);

template <typename T>
struct RowSum { typedef float type; };   // sums of float and 16-bit rows
template <>
struct RowSum<double> { typedef double type; };
template <typename T>
using row_sum_t = typename RowSum<T>::type;

// V elements moved by one instruction (16 bytes, or one element)
template <typename T, int V>
struct RowVec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T>
struct RowVec<T, 1> { typedef T type; };
template <typename T, int V>
using row_vec_t = typename RowVec<T, V>::type;

template <typename T, int V>
__device__ __forceinline__ void row_widen(const row_vec_t<T, V>& v, row_sum_t<T>* a) {
  if constexpr (V == 1) {
    a[0] = (row_sum_t<T>)v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = (row_sum_t<T>)v[i];
  }
}

// one rounding, to nearest even
template <typename T, int V>
__device__ __forceinline__ row_vec_t<T, V> row_round(const row_sum_t<T>* a) {
  row_vec_t<T, V> v;
  if constexpr (V == 1) {
    v = (T)a[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)a[i];
  }
  return v;
}

// q / d for q * d < 2^32 (magic 0: d = 1)
struct RowDiv {
  unsigned d, magic;
  __device__ __forceinline__ unsigned div(unsigned q) const { return magic ? __umulhi(q, magic) : q; }
};
inline RowDiv row_div(unsigned d) {
  return {d, d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d)};
}

inline bool row_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// calls f with a zero of the row type; false for another code
template <typename F>
bool row_dispatch(int type, F&& f) {
  switch (type) {
    case TACE_ROW_F32: f(float()); return true;
    case TACE_ROW_F64: f(double()); return true;
    case TACE_ROW_BF16: f(__bf16()); return true;
    case TACE_ROW_F16: f(_Float16()); return true;
  }
  return false;
}
