// Element types and row addressing of the row operators (rows.hip, dropout.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// Calls f with the elements a move takes, as a constant: 16 bytes, else 8, that
// `fits` (an element count, bytes) allows, else one.
template <typename T, typename Fits, typename F>
void row_moves(Fits&& fits, F&& f) {
  constexpr int W = 16 / sizeof(T), H = W > 2 ? W / 2 : W;
  if (fits(W, 16)) f(std::integral_constant<int, W>());
  else if (H < W && fits(H, 8)) f(std::integral_constant<int, H>());
  else f(std::integral_constant<int, 1>());
}

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
