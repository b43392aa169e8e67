// One step of AdamW (I. Loshchilov, F. Hutter, "Decoupled weight decay
// regularization", 2019) over many tensors at once, and the norm of many
// gradients.
//
//   g' = g min(1, max_norm / |g|)            |g|: over all tensors
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: each operand is read once and written once (a gradient twice
// where it is clipped).  The tensors' addresses travel with the launch, within its 4
// KB of arguments (84 tensors come near them; 56 with masters and scales and 160 for
// norms leave 600 and 800 bytes), so a step over new gradients copies nothing ahead of
// it and a recorded one replays; a workgroup finds its tensor by ballots over the
// tensors' first units.
//
// States of 8 bits: m and r = sqrt(v) as e4m3 codes, 256 elements to a float32
// scale (the block's largest magnitude / 448): r has half the range of v, and
// e4m3 under a scale covers 2^-9 .. 448, 17.8 binades, of it.  An average that
// moves by less than half a code's step a step (b2 = 0.999: 0.1 % of v) would
// stay where it is under rounding to nearest, so codes are rounded up with the
// probability of the value's distance from the one below: from 16 bits of
// Philox-4x32 on (position / 4, tensor, step), half a word for each of m and r.
// A positive r never becomes code zero (it is divided by).  The draw has r's mean, so
// v = r^2 gains r's variance: under normal gradients and b2 = 0.999 v settles 5.5 %
// above its exact average (steps 2.7 % shorter), one element in a hundred at twice it.
#include "philox.h"
#include "row_types.h"

#include <math.h>

#include <algorithm>

namespace {

constexpr int WG = 256, UNIT = 4096, BLOCK = TACE_ADAM_BLOCK;

// a tensor as a launch has it: for the norm, without masters and scales, with them
struct Gradient {
  static constexpr int MOST = 160;
  const void* g;
  int64_t n;
  Gradient() = default;
  explicit Gradient(const tace_adam_tensor& t) : g(t.g), n(t.n) {}
};
struct Plain {
  static constexpr int MOST = 84;
  void* p;
  const void* g;
  void *m, *s;
  int64_t n;
  Plain() = default;
  explicit Plain(const tace_adam_tensor& t) : p(t.p), g(t.g), m(t.m), s(t.s), n(t.n) {}
  __device__ __forceinline__ void* the_master() const { return nullptr; }
  __device__ __forceinline__ float* the_scales() const { return nullptr; }
};
struct Full : Plain {
  static constexpr int MOST = 56;
  void* master;
  float* scales;
  Full() = default;
  explicit Full(const tace_adam_tensor& t) : Plain(t), master(t.master), scales((float*)t.scales) {}
  __device__ __forceinline__ void* the_master() const { return master; }
  __device__ __forceinline__ float* the_scales() const { return scales; }
};

template <typename E>
struct Tensors {
  E t[E::MOST];
  int first[E::MOST + 1];   // units of the tensors before
  int count;
};

// the tensor of a unit (uniform over the workgroup)
template <typename E>
__device__ __forceinline__ int tensor_of(const Tensors<E>& ts, int unit) {
  int before = 0;
#pragma unroll
  for (int at = 0; at < E::MOST; at += 64) {
    const int k = at + ((int)threadIdx.x & 63);
    before += __popcll(__ballot(k < ts.count && ts.first[k < E::MOST ? k : 0] <= unit));
  }
  return __builtin_amdgcn_readfirstlane(before - 1);
}

// ------------------------------------------------------------------- norm ----
// Sums of squares in double (a float32 square has no room for values past 2^64 or
// below 2^-63, whose norm has), a workgroup's, then the last workgroup to finish
// adds them in order.
__device__ __forceinline__ double over_wg(double d, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = d;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T>
__global__ __launch_bounds__(WG) void k_grad_norm(Tensors<Gradient> ts, double* __restrict__ part, int slot0, int slots,
                                                  bool last, unsigned long long* ticket, bool wide,
                                                  void* __restrict__ norm) {
  typedef row_sum_t<T> S;
  constexpr int W = 16 / sizeof(T);
  __shared__ double lds[4];
  __shared__ bool mine;
  double sum = 0;
  const int units = ts.first[ts.count];
  for (int unit = (int)blockIdx.x; unit < units; unit += (int)gridDim.x) {
    const int k = tensor_of(ts, unit);
    const T* g = (const T*)ts.t[k].g;
    const int64_t i0 = (int64_t)(unit - ts.first[k]) * UNIT, left = ts.t[k].n - i0;
    const int n = (int)(left < UNIT ? left : UNIT);
    g += i0;
    double s = 0;
    if (((uintptr_t)g & 15) == 0 && n == UNIT) {
      row_vec_t<T, W> v[UNIT / WG / W];
#pragma unroll
      for (int i = 0; i < UNIT / WG / W; ++i) v[i] = ((const row_vec_t<T, W>*)g)[threadIdx.x + WG * i];
#pragma unroll
      for (int i = 0; i < UNIT / WG / W; ++i) {
        S a[W];
        row_widen<T, W>(v[i], a);
#pragma unroll
        for (int e = 0; e < W; ++e) s += (double)a[e] * (double)a[e];
      }
    } else {
      for (int i = (int)threadIdx.x; i < n; i += WG) s += (double)g[i] * (double)g[i];
    }
    sum += s;
  }
  const double total = over_wg(sum, lds);
  if (threadIdx.x == 0) {
    // (written past the caches of its XCD, and waited for: no fence, which would write all of them back)
    __hip_atomic_store(part + slot0 + blockIdx.x, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (last) {
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      mine = atomicAdd(ticket, 1ull) == gridDim.x - 1;
    }
  }
  if (!last) return;
  __syncthreads();
  if (!mine) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  double all = 0;
  for (int i = (int)threadIdx.x; i < slots; i += WG)
    all += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  all = sqrt(over_wg(all, lds));
  if (threadIdx.x == 0) {
    if (wide) *(double*)norm = all;
    else *(float*)norm = (float)all;
    *ticket = 0;
  }
}

// ------------------------------------------------------------------- step ----
template <typename S>
struct Step {
  S lr, b1, b2, rest1, rest2, eps, decay, max_norm;   // rest: 1 - b
  S log_b1, log_b2;
  const void* lr_at;   // device learning rate, or null
  int lr_wide;
  const void* norm;    // device norm, or null
  long long* counter;  // steps done, ticket
  unsigned seed_lo, seed_hi, tensor0;
  int ticks;           // whether this launch ends the step
};

template <typename S>
struct Now {
  S clip, keep, rate, root;   // gradients' factor, 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

// p, m and v (or r) after the step.  Each product and sum is rounded by itself, as
// in a program of one operation after the other: codes' draws then fall alike in
// both (a largest element a last place higher or lower, rounded the other way,
// would move its block's next scale by 7 %).  The step waits for memory anyway.
template <typename S>
__device__ __forceinline__ void adam(const Step<S>& st, const Now<S>& c, S g, S& p, S& m, S& v, S& r) {
#pragma clang fp contract(off)
  g *= c.clip;
  m = m * st.b1 + g * st.rest1;
  v = v * st.b2 + g * g * st.rest2;
  r = sqrt(v);
  p = p * c.keep - m / (r * c.root + st.eps) * c.rate;
}

template <typename S>
__device__ __forceinline__ Now<S> coefficients(const Step<S>& st, long long t, S norm) {
  Now<S> c;
  S lr = st.lr;
  if (st.lr_at) lr = st.lr_wide ? (S) * (const double*)st.lr_at : (S) * (const float*)st.lr_at;
  // 1 - b^t without cancellation
  c.rate = lr / -expm1((S)t * st.log_b1);
  c.root = (S)1 / sqrt(-expm1((S)t * st.log_b2));
  c.keep = (S)1 - lr * st.decay;
  c.clip = st.norm && norm > st.max_norm ? st.max_norm / norm : (S)1;
  return c;
}

// x's block of 256 (4 elements a lane) as codes of a shared scale, rounded at
// random by the halves of `words` at `shift`
__device__ __forceinline__ int drawn_codes(const float* x, const unsigned* words, int shift, bool root, float* scale) {
  float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  const bool bad = !(x[0] == x[0] && x[1] == x[1] && x[2] == x[2] && x[3] == x[3]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if (__ballot(bad)) top = __builtin_nanf("");
  if (top < 0x1p-100f) top = 0.0f;   // (448 / top overflows below 2^-118)
  const float up = top == 0.0f ? 0.0f : 1.0f / top * 448.0f;   // (as tensors' quotients with numbers are made)
  *scale = top * (1.0f / 448.0f);
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = x[e] * up, a = fabsf(y);
    // the codes' step at a: 2^(exponent - 3), at least 2^-9
    const int ex = max((int)(__float_as_uint(a) >> 23), 127 - 6);
    const float step = __uint_as_float((unsigned)(ex - 3) << 23), per = __uint_as_float((unsigned)(254 - (ex - 3)) << 23);
    const float u = (float)((words[e] >> shift) & 0xffffu) * 0x1p-16f;
    float c = fminf(floorf(a * per + u) * step, 448.0f);
    if (root && a > 0.0f) c = fmaxf(c, 0x1p-9f);
    q[e] = y == y ? copysignf(c, y) : y;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}

template <int V, typename T>
__device__ __forceinline__ void load4(const T* p, int n, row_sum_t<T>* a) {
  if constexpr (V == 4) {
    row_widen<T, 4>(*(const row_vec_t<T, 4>*)p, a);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = e < n ? (row_sum_t<T>)p[e] : (row_sum_t<T>)0;
  }
}
template <int V, typename T>
__device__ __forceinline__ void store4(T* p, int n, const row_sum_t<T>* a) {
  if constexpr (V == 4) {
    *(row_vec_t<T, 4>*)p = row_round<T, 4>(a);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = (T)a[e];
  }
}

// A unit of up to 4,096 elements; V = 4: whole, its addresses multiples of four
// elements (a lane's four go as one move each).  EIGHT: a wavefront's 256
// elements are a block.
template <typename T, bool EIGHT, int V, typename E>
__device__ __forceinline__ void run_unit(const Step<row_sum_t<T>>& st, const E& t, int tensor,
                                         int64_t i0, int n, long long steps) {
  typedef row_sum_t<T> S;
  constexpr int U = sizeof(T) == 8 ? 2 : 4;   // passes whose loads go out together
  const bool master = t.the_master() != nullptr;
  T* p = (T*)t.p + i0;
  const T* g = (const T*)t.g + i0;
  S* w = master ? (S*)t.the_master() + i0 : nullptr;
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < UNIT / (4 * WG); r += U) {
    S pv[U][4], gv[U][4], mv[U][4], sv[U][4];
    float sm[U], sr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = 4 * ((r + u) * WG + (int)threadIdx.x), left = n - i;
      if (V != 4 && 4 * ((r + u) * WG + (int)threadIdx.x - lane) >= n) continue;   // (a wavefront without elements)
      load4<V>(g + i, left, gv[u]);
      if (std::is_same<T, S>::value || !master) load4<V>(p + i, left, pv[u]);
      else load4<V>(w + i, left, pv[u]);
      if constexpr (EIGHT) {
        int cm = 0, cs = 0;
        if constexpr (V == 4) {
          cm = *(const int*)((const char*)t.m + i0 + i);
          cs = *(const int*)((const char*)t.s + i0 + i);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e < left) {
              cm |= (int)((const unsigned char*)t.m)[i0 + i + e] << (8 * e);
              cs |= (int)((const unsigned char*)t.s)[i0 + i + e] << (8 * e);
            }
          }
        }
        const float2 sc = ((const float2*)t.the_scales())[(i0 + i - 4 * lane) / BLOCK];
        sm[u] = sc.x;
        sr[u] = sc.y;
        mv[u][0] = __builtin_amdgcn_cvt_f32_fp8(cm, 0), mv[u][1] = __builtin_amdgcn_cvt_f32_fp8(cm, 1);
        mv[u][2] = __builtin_amdgcn_cvt_f32_fp8(cm, 2), mv[u][3] = __builtin_amdgcn_cvt_f32_fp8(cm, 3);
        sv[u][0] = __builtin_amdgcn_cvt_f32_fp8(cs, 0), sv[u][1] = __builtin_amdgcn_cvt_f32_fp8(cs, 1);
        sv[u][2] = __builtin_amdgcn_cvt_f32_fp8(cs, 2), sv[u][3] = __builtin_amdgcn_cvt_f32_fp8(cs, 3);
      } else {
        load4<V>((const S*)t.m + i0 + i, left, mv[u]);
        load4<V>((const S*)t.s + i0 + i, left, sv[u]);
      }
    }
    S norm = 0;
    if (st.norm) norm = sizeof(S) == 8 ? (S) * (const double*)st.norm : (S) * (const float*)st.norm;
    const Now<S> now = coefficients(st, steps, norm);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = 4 * ((r + u) * WG + (int)threadIdx.x), left = n - i;
      if (V != 4 && 4 * ((r + u) * WG + (int)threadIdx.x - lane) >= n) continue;
      S rv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (EIGHT) {
          mv[u][e] *= sm[u];
          sv[u][e] *= sr[u];
          sv[u][e] *= sv[u][e];
        }
        adam<S>(st, now, gv[u][e], pv[u][e], mv[u][e], sv[u][e], rv[e]);
      }
      if (std::is_same<T, S>::value) {
        store4<V>((S*)p + i, left, pv[u]);
      } else {
        if (master) store4<V>(w + i, left, pv[u]);
        store4<V>(p + i, left, pv[u]);
      }
      if constexpr (EIGHT) {
        const int64_t at = i0 + i;
        unsigned words[4] = {(unsigned)(at >> 2), (unsigned)tensor, (unsigned)steps,
                             (unsigned)((unsigned long long)steps >> 32)};
        philox(words, st.seed_lo, st.seed_hi);
        float2 sc;
        const int cm = drawn_codes(mv[u], words, 0, false, &sc.x), cs = drawn_codes(rv, words, 16, true, &sc.y);
        if constexpr (V == 4) {
          *(int*)((char*)t.m + at) = cm;
          *(int*)((char*)t.s + at) = cs;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e < left) {
              ((unsigned char*)t.m)[at + e] = (unsigned char)(cm >> (8 * e));
              ((unsigned char*)t.s)[at + e] = (unsigned char)(cs >> (8 * e));
            }
          }
        }
        if (lane == 0) ((float2*)t.the_scales())[at / BLOCK] = sc;
      } else {
        store4<V>((S*)t.m + i0 + i, left, mv[u]);
        store4<V>((S*)t.s + i0 + i, left, sv[u]);
      }
    }
  }
}

// whether a unit's operands can be moved four elements at a time
template <typename T, bool EIGHT, typename E>
__device__ __forceinline__ bool fours(const E& t, int64_t i0) {
  const uintptr_t a4 = (uintptr_t)((T*)t.p + i0) | (uintptr_t)((const T*)t.g + i0);
  uintptr_t s4 = EIGHT ? ((uintptr_t)t.m | (uintptr_t)t.s) * sizeof(row_sum_t<T>) : (uintptr_t)t.m | (uintptr_t)t.s;
  s4 |= (uintptr_t)t.the_master();
  return a4 % (4 * sizeof(T)) == 0 && s4 % (4 * sizeof(row_sum_t<T>)) == 0;
}

template <typename T, bool EIGHT, typename E>
__global__ __launch_bounds__(WG) void k_adamw(Tensors<E> ts, Step<row_sum_t<T>> st) {
  typedef row_sum_t<T> S;
  const int unit = (int)blockIdx.x, k = tensor_of(ts, unit);
  const E& t = ts.t[k];
  const int64_t i0 = (int64_t)(unit - ts.first[k]) * UNIT, left = t.n - i0;
  const int n = (int)(left < UNIT ? left : UNIT);
  long long steps = st.counter[0] + 1;
  bool go = true;
  if (st.norm) {   // (no step on a norm that is no number)
    const S norm = sizeof(S) == 8 ? (S) * (const double*)st.norm : (S) * (const float*)st.norm;
    go = norm < (S)__builtin_inf();
  }
  if (go) {
    if (n == UNIT && fours<T, EIGHT>(t, i0)) run_unit<T, EIGHT, 4>(st, t, (int)st.tensor0 + k, i0, n, steps);
    else run_unit<T, EIGHT, 1>(st, t, (int)st.tensor0 + k, i0, n, steps);
  }
  if (!st.ticks) return;
  // The last workgroup counts the step: every other has read the counter.  (No
  // fence: nothing else passes between workgroups, and writing the caches back
  // for each took 366 instead of 120 us over 18 M elements.)
  asm volatile("" : "+v"(steps) : : "memory");   // read by now
  __syncthreads();
  if (threadIdx.x == 0) {
    if (atomicAdd((unsigned long long*)st.counter + 1, 1ull) == gridDim.x - 1) {
      st.counter[1] = 0;
      if (go) st.counter[0] = steps;
    }
  }
}

// ------------------------------------------------------------------- host ----
int check_tensors(int type, const tace_adam_tensor* t, int64_t count, bool states, int eight) {
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("adamw: unknown row type");
  if (count < 0 || (count && !t)) return tace_fail_msg("adamw: null argument");
  if (eight && type == TACE_ROW_F64) return tace_fail_msg("adamw: float64 has no states of 8 bits");
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n < 0 || t[i].n > ((int64_t)1 << 34)) return tace_fail_msg("adamw: tensors of up to 2^34 elements");
    if (t[i].n == 0) continue;
    if (!t[i].g || (states && (!t[i].p || !t[i].m || !t[i].s || (eight && !t[i].scales))))
      return tace_fail_msg("adamw: null argument");
    if (states && t[i].master && (type == TACE_ROW_F32 || type == TACE_ROW_F64))
      return tace_fail_msg("adamw: weights of 16 bits have masters");
  }
  return 0;
}

// calls f(tensors, index of the first, whether they are the last) for launches of as
// many tensors as fit.  (60 of 1 to 131,072 elements: a step takes 27 us in one
// launch, 32 in two.)
template <typename E, typename F>
bool chunks(const tace_adam_tensor* t, int64_t count, F&& f) {
  int64_t end = count;
  while (end > 0 && t[end - 1].n == 0) --end;
  Tensors<E> ts;
  ts.count = 0;
  ts.first[0] = 0;
  int64_t from = 0;
  for (int64_t i = 0; i < end; ++i) {
    const int64_t units = (t[i].n + UNIT - 1) / UNIT;
    if (ts.count && ((int64_t)ts.first[ts.count] + units > (1 << 23) || ts.count == E::MOST)) {
      if (ts.first[ts.count]) f(ts, from, false);   // (not where all are empty)
      ts.count = 0;
      from = i;
    }
    ts.t[ts.count] = E(t[i]);
    ts.first[ts.count + 1] = ts.first[ts.count] + (int)units;
    ++ts.count;
  }
  if (ts.count) f(ts, from, true);
  return ts.count > 0;
}

// Workgroups of a norm: four units each, 256 to 1,024.  The last one's ticket is one
// address for all, about 10 ns each: 968 units take 12.2 us with 256, 14.7 with
// 512, 20.0 with 968 workgroups; 61,043 units 283, 235 and (1,024) 219 us.
int norm_wgs(const Tensors<Gradient>& ts) {
  const int units = ts.first[ts.count];
  return std::min(units, std::min(std::max(units / 4, 256), 1024));
}
int64_t norm_slots(const tace_adam_tensor* t, int64_t count) {
  int64_t slots = 0;
  chunks<Gradient>(t, count, [&](const Tensors<Gradient>& ts, int64_t, bool) { slots += norm_wgs(ts); });
  return slots;
}

}  // namespace

extern "C" int64_t tace_grad_norm_work(const tace_adam_tensor* tensors, int64_t count) {
  if (check_tensors(TACE_ROW_F32, tensors, count, false, 0)) return -1;
  return norm_slots(tensors, count) * (int64_t)sizeof(double);
}

extern "C" int tace_grad_norm(int type, const tace_adam_tensor* tensors, int64_t count, int64_t* ticket, void* norm,
                              void* work, int64_t work_bytes, void* stream) {
  if (check_tensors(type, tensors, count, false, 0)) return -1;
  const int64_t slots = norm_slots(tensors, count);
  if (slots == 0 || slots > INT32_MAX / 2) return tace_fail_msg("grad_norm: no gradients, or too many");
  if (!ticket || !norm || !work || ((uintptr_t)work & 7) || work_bytes < slots * (int64_t)sizeof(double))
    return tace_fail_msg("grad_norm: null argument, or the workspace is too small or not 8-byte aligned");
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    int64_t slot0 = 0;
    chunks<Gradient>(tensors, count, [&](const Tensors<Gradient>& ts, int64_t, bool last) {
      hipLaunchKernelGGL((k_grad_norm<T>), dim3((unsigned)norm_wgs(ts)), dim3(WG), 0, (hipStream_t)stream, ts,
                         (double*)work, (int)slot0, (int)slots, last, (unsigned long long*)ticket,
                         type == TACE_ROW_F64, norm);
      slot0 += norm_wgs(ts);
    });
  });
  return tace_check_launch("grad_norm");
}

extern "C" int tace_adamw(int type, int eight, const tace_adam_tensor* tensors, int64_t count, int64_t* counter,
                          double lr, const void* lr_at, int lr_wide, double beta1, double beta2, double eps,
                          double decay, const void* norm, double max_norm, uint64_t seed, void* stream) {
  if (check_tensors(type, tensors, count, true, eight)) return -1;
  if (count > INT32_MAX) return tace_fail_msg("adamw: too many tensors");
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0))
    return tace_fail_msg("adamw: betas are in [0, 1), eps is not negative");
  if (!counter) return tace_fail_msg("adamw: null argument");
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += tensors[i].n;
  if (total == 0) return 0;
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    typedef row_sum_t<T> S;
    Step<S> st;
    st.lr = (S)lr, st.b1 = (S)beta1, st.b2 = (S)beta2, st.rest1 = (S)(1 - beta1), st.rest2 = (S)(1 - beta2);
    st.eps = (S)eps, st.decay = (S)decay, st.max_norm = (S)max_norm;
    st.log_b1 = (S)::log(beta1), st.log_b2 = (S)::log(beta2);
    st.lr_at = lr_at, st.lr_wide = lr_wide, st.norm = norm, st.counter = (long long*)counter;
    st.seed_lo = (unsigned)seed, st.seed_hi = (unsigned)(seed >> 32);
    auto launch = [&](auto eight_type, auto entry) {
      typedef decltype(entry) E;
      constexpr bool EIGHT = decltype(eight_type)::value;
      static_assert(sizeof(Tensors<E>) + sizeof(Step<S>) <= 4096, "a launch's arguments");
      chunks<E>(tensors, count, [&](const Tensors<E>& ts, int64_t from, bool last) {
        st.tensor0 = (unsigned)from;
        st.ticks = last;
        hipLaunchKernelGGL((k_adamw<T, EIGHT, E>), dim3((unsigned)ts.first[ts.count]), dim3(WG), 0, (hipStream_t)stream, ts,
                           st);
      });
    };
    if constexpr (!std::is_same<T, double>::value) {
      if (eight) return launch(std::true_type(), Full());
    }
    bool masters = false;
    for (int64_t i = 0; i < count; ++i) masters |= tensors[i].master != nullptr;
    if constexpr (!std::is_same<T, S>::value) {
      if (masters) return launch(std::false_type(), Full());
    }
    launch(std::false_type(), Plain());
  });
  return tace_check_launch("adamw");
}
