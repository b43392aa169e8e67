// Root-mean-square norm of rows with the residual's addition before it, and an
// output of 8 bits with a scale a row.
//
// A row is one degree block of one atom: d = comps[b] components of C channels,
// n = d C contiguous elements (plain rows: one block, d = 1).
//   h = x + r (rounded to the rows' type);  q = 1 / sqrt(sum h^2 / n + eps)
//   y_j = h_j q w[j mod C]
// so one factor per (row, block) commutes with rotations of the components.
// Backward, with u_j = gy_j w[j mod C] and gh the gradient of h from elsewhere:
//   dh_j = q (u_j - h_j q^2 (sum u h) / n) + gh_j
//   dw_c = sum over rows and components of gy_j h_j q
// 8 bits: scale = max |y| / 448, code_j = e4m3(448 h_j w_j / max |h w|), y_j's for any q.
// Bound by HBM.  A group of LPR lanes owns a row and holds it in registers between
// the sum and the output, so each input is read once; groups walk over rows of
// one block, their weights (and in the backward pass the weights' gradient) in
// registers.  Rows past 16,384 elements (float64: 8,192; rows that are not moved by 16
// bytes: 4,096) do not fit and spill, up to 948 (1,268) bytes a lane in the backward
// pass: 4,000 rows of 32,768 in bfloat16 614 us forward and backward, of 16,384 168.  The gradient's sums leave a workgroup once: groups meet in LDS,
// a second launch adds the workgroups in order.
//
// Measured (forward, backward with the weights' gradient): 12,288 rows of degrees 0
// to 3 with 128 channels, float32, with residual: 78 + 93 us, 5.2 and 4.6 TB/s;
// 8,191 rows of 4,096, bfloat16: 24 + 48 us, 5.7 and 4.2 TB/s; 101,306 rows of 256 to
// 8 bits with residual: 32 to 40 us, 5.7 to 4.6 TB/s (a copy: 5.0).  Channels that are no
// multiple of 16 bytes move one element at a time: 20,000 rows in bfloat16, forward and
// backward, of 1,003 112 us and of 1,008 66; 100,000 of 100 to 8 bits 38, of 104 12.5.
#include "row_types.h"

namespace {

constexpr int WG = 256;

struct NormParts {
  int count, channels;
  int comps[TACE_ROW_MAX_BLOCKS];
  int before[TACE_ROW_MAX_BLOCKS];        // components of the blocks before
  int first[TACE_ROW_MAX_BLOCKS + 1];     // workgroups of the blocks before
};

__device__ __forceinline__ int norm_block(const NormParts& pt, int wg) {
  int b = 0;
  while (wg >= pt.first[b + 1]) ++b;
  return b;
}

struct Add {
  template <typename S>
  __device__ __forceinline__ static S of(S a, S b) { return a + b; }
};
struct Top {   // NaN stays
  template <typename S>
  __device__ __forceinline__ static S of(S a, S b) { return b > a || b != b ? b : a; }
};

// over a row's LPR lanes; lds: a slot for each wavefront of the workgroup
template <int LPR, typename Op, typename S>
__device__ __forceinline__ S over_row(S v, S* lds) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v = Op::of(v, __shfl_xor(v, o, 64));
  if constexpr (LPR > 64) {
    __syncthreads();   // (the slots' last readers)
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < LPR / 64; ++i) v = Op::of(v, lds[i]);
  }
  return v;
}

// Waves a SIMD of rows to 8 bits, where the compiler would take a few registers more
// than they leave (one is spilled at most): 60,000 float32 rows of degrees 0 to 3, 128
// channels, with residual 304 us, 336 without.
constexpr int code_waves(int V, int LPR, int NV) {
  return LPR == 64 && NV == 4 ? (V == 4 ? 5 : V == 8 ? 4 : 1) : 1;
}

// V values as e4m3 codes, to nearest even (|v| <= 448 but for rounding; NaN stays)
template <int V>
__device__ __forceinline__ void store_codes(unsigned char* p, const float* v) {
  if constexpr (V == 1) {
    *p = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], 0.0f, 0, false);
  } else {
    int word[V / 2];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      word[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      word[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], word[i], true);
    }
    if constexpr (V == 4) *(int*)p = word[0];
    else *(int2*)p = int2{word[0], word[1]};
  }
}

// this lane's weights: vector i starts at channel at[i]
template <typename T, int V, int LPR, int NV>
__device__ __forceinline__ void lane_weights(const void* weight, bool wide, int b, int C, int li, int nvec,
                                             row_sum_t<T>* w) {
  typedef row_sum_t<T> S;
  const unsigned cv = (unsigned)C / V;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int idx = li + LPR * i;
    if (idx >= nvec) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[i * V + e] = 0;
      continue;
    }
    const int64_t c = (int64_t)b * C + (int)((unsigned)idx % cv) * V;
    if (wide) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[i * V + e] = ((const S*)weight)[c + e];
    } else {
      row_widen<T, V>(*(const row_vec_t<T, V>*)((const T*)weight + c), w + i * V);
    }
  }
}

// Q: y as e4m3 codes with scales [rows, blocks]
template <typename T, int V, int LPR, int NV, bool Q>
__global__ __launch_bounds__(LPR > WG ? LPR : WG, Q ? code_waves(V, LPR, NV) : 1) void k_rms_fwd(
    const T* __restrict__ x, const T* __restrict__ res, const void* __restrict__ weight, bool wide, int64_t rows,
    NormParts pt, row_sum_t<T> eps, T* __restrict__ h, void* __restrict__ y, float* __restrict__ scales,
    row_sum_t<T>* __restrict__ inv) {
  typedef row_sum_t<T> S;
  typedef row_vec_t<T, V> Vec;
  constexpr int G = LPR > WG ? 1 : WG / LPR;
  __shared__ S slots[16];
  const int b = norm_block(pt, (int)blockIdx.x), C = pt.channels;
  const int width = pt.comps[b] * C, nvec = width / V;
  const int64_t base = rows * C * pt.before[b];
  const int group = (int)threadIdx.x / LPR, li = (int)threadIdx.x % LPR;
  const int64_t stride = (int64_t)(pt.first[b + 1] - pt.first[b]) * G;
  S w[NV * V];
  lane_weights<T, V, LPR, NV>(weight, wide, b, C, li, nvec, w);
  // (a row of several wavefronts: uniform over the workgroup)
  for (int64_t r = (int64_t)((int)blockIdx.x - pt.first[b]) * G + group; r < rows; r += stride) {
    const int64_t at = base + r * width;
    S a[NV * V];
    Vec in[NV], add[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx < nvec) {
        in[i] = ((const Vec*)(x + at))[idx];
        if (res) add[i] = ((const Vec*)(res + at))[idx];
      }
    }
    S sum = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx < nvec) {
        row_widen<T, V>(in[i], a + i * V);
        if (res) {
          S o[V];
          row_widen<T, V>(add[i], o);
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] += a[i * V + e];
          const Vec hv = row_round<T, V>(o);
          ((Vec*)(h + at))[idx] = hv;
          row_widen<T, V>(hv, a + i * V);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) a[i * V + e] = 0;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) sum += a[i * V + e] * a[i * V + e];
    }
    sum = over_row<LPR, Add>(sum, slots);
    const S q = (S)1 / sqrt(sum / width + eps);
    if (inv && li == 0) inv[r * pt.count + b] = q;
    // 8 bits: instead of q a power of two near q / 1024, times 448: h w of few bits stays
    // exact, and a value between two codes is seen to be there, however q was rounded
    // (but in rows below 2^-60, whose quotients' remainders float32 does not hold).
    S factor = q, two = 0;
    if constexpr (Q) {
      two = __uint_as_float(__float_as_uint(q) & 0x7f800000u) * 0x1p-10f;
      factor = two * 448;
    }
    S top = 0, most = 0, per = 0;
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
      a[i] = a[i] * factor * w[i];
      if constexpr (Q) {
        // (past the row's end: zero times what may be infinite)
        if (li + LPR * (i / V) >= nvec) a[i] = 0;
        top = Top::of(top, (S)fabs(a[i]));
      }
    }
    if constexpr (Q) {
      top = over_row<LPR, Top>(top, slots);
      const S scale = top / (448 * 448) * (q / two);   // the row's largest |y| / 448
      // (smaller rows are zeros, as those of zeros: near float32's end quotients lose their bits)
      const bool none = top == 0 || scale < (S)(0x1p-100 / 448);
      if (li == 0) scales[r * pt.count + b] = none ? 0.0f : (float)scale;
      // a code is that of a / most, rounded once: by a corrected product with the reciprocal.  (A
      // division for each element: 101,306 rows of 256 in bfloat16 41 instead of 37 us.)
      most = none ? (S)0 : top / 448;
      per = none ? (S)0 : 1 / most;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx >= nvec) continue;
      if constexpr (Q) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float t = (float)a[i * V + e], near = t * (float)per;
          v[e] = fmaf(fmaf(-near, (float)most, t), (float)per, near);
        }
        store_codes<V>((unsigned char*)y + at + (int64_t)idx * V, v);
      } else {
        ((Vec*)((T*)y + at))[idx] = row_round<T, V>(a + i * V);
      }
    }
  }
}

// part: for each workgroup its sums of the weights' gradient, [C] (rows of up to
// WG lanes) or [d C]
template <typename T, int V, int LPR, int NV>
__global__ __launch_bounds__(LPR > WG ? LPR : WG) void k_rms_bwd(
    const T* __restrict__ gy, const T* __restrict__ gh, const T* __restrict__ h, const void* __restrict__ weight,
    bool wide, const row_sum_t<T>* __restrict__ inv, int64_t rows, NormParts pt, T* __restrict__ dh,
    row_sum_t<T>* __restrict__ part) {
  typedef row_sum_t<T> S;
  typedef row_vec_t<T, V> Vec;
  constexpr int G = LPR > WG ? 1 : WG / LPR;
  constexpr bool FOLD = LPR <= WG;
  __shared__ S slots[16];
  __shared__ S meet[FOLD ? WG * NV * V : 1];
  const int b = norm_block(pt, (int)blockIdx.x), C = pt.channels, d = pt.comps[b];
  const int width = d * C, nvec = width / V;
  const int64_t base = rows * C * pt.before[b];
  const int group = (int)threadIdx.x / LPR, li = (int)threadIdx.x % LPR;
  const int64_t stride = (int64_t)(pt.first[b + 1] - pt.first[b]) * G;
  S w[NV * V], dw[NV * V];
  lane_weights<T, V, LPR, NV>(weight, wide, b, C, li, nvec, w);
#pragma unroll
  for (int i = 0; i < NV * V; ++i) dw[i] = 0;
  for (int64_t r = (int64_t)((int)blockIdx.x - pt.first[b]) * G + group; r < rows; r += stride) {
    const int64_t at = base + r * width;
    Vec g[NV], hv[NV], add[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx < nvec) {
        g[i] = ((const Vec*)(gy + at))[idx];
        hv[i] = ((const Vec*)(h + at))[idx];
        if (gh) add[i] = ((const Vec*)(gh + at))[idx];
      }
    }
    const S q = inv[r * pt.count + b];
    S dot = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (li + LPR * i >= nvec) continue;
      S a[V], o[V];
      row_widen<T, V>(g[i], a);
      row_widen<T, V>(hv[i], o);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dot += a[e] * w[i * V + e] * o[e];
        dw[i * V + e] += a[e] * (o[e] * q);
      }
    }
    dot = over_row<LPR, Add>(dot, slots);
    const S k = dot / width * q * q;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx >= nvec) continue;
      S a[V], o[V];
      row_widen<T, V>(g[i], a);
      row_widen<T, V>(hv[i], o);
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = q * (a[e] * w[i * V + e] - o[e] * k);
      if (gh) {
        row_widen<T, V>(add[i], o);
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] += o[e];
      }
      ((Vec*)(dh + at))[idx] = row_round<T, V>(a);
    }
  }
  if (!part) return;
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx < nvec) {
#pragma unroll
        for (int e = 0; e < V; ++e) meet[group * width + idx * V + e] = dw[i * V + e];
      }
    }
    __syncthreads();
    for (int c = (int)threadIdx.x; c < C; c += WG) {
      S sum = 0;
      for (int j = c; j < G * width; j += C) sum += meet[j];
      part[(int64_t)blockIdx.x * C + c] = sum;
    }
  } else {
    S* out = part;   // (the blocks before: their workgroups' rows)
    for (int i = 0; i < b; ++i) out += (int64_t)(pt.first[i + 1] - pt.first[i]) * pt.comps[i] * C;
    out += (int64_t)((int)blockIdx.x - pt.first[b]) * width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = li + LPR * i;
      if (idx < nvec) {
#pragma unroll
        for (int e = 0; e < V; ++e) out[idx * V + e] = dw[i * V + e];
      }
    }
  }
}

// dw [blocks, C] from the workgroups' sums: each block's are one matrix of
// count (x d where a workgroup's are [d C]) rows of C
constexpr int SUM_COLS = 32, SUM_ROWS = 16;
template <typename T>
__global__ __launch_bounds__(SUM_COLS* SUM_ROWS) void k_rms_dw(const row_sum_t<T>* __restrict__ part, NormParts pt,
                                                               bool folded, bool wide, void* __restrict__ dw) {
  typedef row_sum_t<T> S;
  __shared__ S meet[SUM_ROWS][SUM_COLS];
  const int b = (int)blockIdx.y, C = pt.channels;
  const int col = (int)threadIdx.x % SUM_COLS, row = (int)threadIdx.x / SUM_COLS;
  const int c = (int)blockIdx.x * SUM_COLS + col;
  const S* p = part;
  for (int i = 0; i < b; ++i) p += (int64_t)(pt.first[i + 1] - pt.first[i]) * (folded ? 1 : pt.comps[i]) * C;
  const int n = (pt.first[b + 1] - pt.first[b]) * (folded ? 1 : pt.comps[b]);
  S sum = 0;
  if (c < C) {
    int r = row;
    for (; r + 7 * SUM_ROWS < n; r += 8 * SUM_ROWS) {
      S v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)(r + i * SUM_ROWS) * C + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
    for (; r < n; r += SUM_ROWS) sum += p[(int64_t)r * C + c];
  }
  meet[row][col] = sum;
  __syncthreads();
  if (row != 0 || c >= C) return;
#pragma unroll
  for (int i = 1; i < SUM_ROWS; ++i) sum += meet[i][col];
  if (wide) ((S*)dw)[(int64_t)b * C + c] = sum;
  else ((T*)dw)[(int64_t)b * C + c] = (T)sum;
}

// ------------------------------------------------------------------- host ----
// Lanes and vectors a row: the fewest lanes that hold the widest block's vectors
// with few registers.
template <int V, typename F>
void row_shape(int nvec, F&& f) {
  using std::integral_constant;
  typedef integral_constant<int, 1> I1;
  typedef integral_constant<int, 2> I2;
  typedef integral_constant<int, 4> I4;
  if (nvec <= 16) f(integral_constant<int, 16>(), I1());
  else if (nvec <= 32) f(integral_constant<int, 32>(), I1());
  else if (nvec <= 64) f(integral_constant<int, 64>(), I1());
  else if (nvec <= 128) f(integral_constant<int, 64>(), I2());
  else if (nvec <= 256) f(integral_constant<int, 64>(), I4());
  else if (nvec <= 512) f(integral_constant<int, 256>(), I2());
  else if (nvec <= 1024) f(integral_constant<int, 256>(), I4());
  else if (nvec <= 2048) f(integral_constant<int, 1024>(), I2());
  else if (nvec <= 4096) f(integral_constant<int, 1024>(), I4());
  else f(integral_constant<int, 1024>(), integral_constant<int, V < 8 ? 32 / V : 4>());   // (up to 32,768 elements)
}

// (twice as many in the backward pass take as long, and the second launch 3 us more)
constexpr int FWD_WGS = 2048, BWD_WGS = 1024;

int widest(int blocks, const int32_t* comps) {
  int top = 0;
  for (int b = 0; b < blocks; ++b) top = comps[b] > top ? comps[b] : top;
  return top;
}

// Workgroups of each block, by its share of the time: a row waits for memory as long
// as two components more take.  (By its elements alone the blocks of degree 0 were
// last: 103 instead of 88 us in the backward pass of degrees 0 to 3.)
NormParts make_parts(int64_t rows, int channels, int blocks, const int32_t* comps, int groups, int most) {
  NormParts pt;
  pt.count = blocks;
  pt.channels = channels;
  int total = 0;
  for (int b = 0; b < blocks; ++b) total += comps[b] + 2;
  int before = 0, wgs = 0;
  for (int b = 0; b < blocks; ++b) {
    pt.comps[b] = comps[b];
    pt.before[b] = before;
    pt.first[b] = wgs;
    before += comps[b];
    const int64_t need = (rows + groups - 1) / groups, share = (int64_t)most * (comps[b] + 2) / total + 1;
    wgs += (int)(need < share ? need : share);
  }
  pt.first[blocks] = wgs;
  return pt;
}

int check_norm(int64_t rows, int channels, int blocks, const int32_t* comps) {
  if (rows < 0 || channels < 1 || blocks < 1 || blocks > TACE_ROW_MAX_BLOCKS || !comps)
    return tace_fail_msg("rms_norm: bad sizes");
  int64_t total = 0;
  for (int b = 0; b < blocks; ++b) {
    if (comps[b] < 1 || comps[b] > 1024 || (int64_t)comps[b] * channels > 32768)
      return tace_fail_msg("rms_norm: components are not 1 to 1024 of at most 32768 elements");
    total += comps[b];
  }
  if (rows > INT32_MAX - 8192 || rows * total > ((int64_t)1 << 46) / channels)
    return tace_fail_msg("rms_norm: bad sizes");
  return 0;
}

// elements of the workgroups' sums for moves of V elements
template <int V>
int64_t part_elems(int64_t rows, int channels, int blocks, const int32_t* comps) {
  int64_t n = 0;
  row_shape<V>(widest(blocks, comps) * channels / V, [&](auto lpr, auto) {
    constexpr int LPR = decltype(lpr)::value;
    const NormParts pt = make_parts(rows, channels, blocks, comps, LPR > WG ? 1 : WG / LPR, BWD_WGS);
    for (int b = 0; b < blocks; ++b)
      n += (int64_t)(pt.first[b + 1] - pt.first[b]) * channels * (LPR > WG ? comps[b] : 1);
  });
  return n;
}

}  // namespace

extern "C" int tace_rms_norm_fwd(int type, const void* x, const void* residual, const void* weight, int weight_wide,
                                 int64_t rows, int32_t channels, int32_t blocks, const int32_t* comps, double eps,
                                 void* h, void* y, float* scales, void* inv, void* stream) {
  if (check_norm(rows, channels, blocks, comps)) return -1;
  if (scales && type == TACE_ROW_F64) return tace_fail_msg("rms_norm: rows of 8 bits are made of float32 and 16-bit rows");
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("rms_norm: unknown row type");
  if (rows == 0) return 0;
  if (!x || !weight || !y || (!residual) != (!h)) return tace_fail_msg("rms_norm: null argument");
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    typedef row_sum_t<T> S;
    constexpr int W = 16 / sizeof(T);
    auto launch = [&](auto v) {
      constexpr int V = decltype(v)::value;
      row_shape<V>(widest(blocks, comps) * channels / V, [&](auto lpr, auto nv) {
        constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value, N = LPR > WG ? LPR : WG;
        const NormParts pt = make_parts(rows, channels, blocks, comps, N / LPR, FWD_WGS);
        const dim3 grid((unsigned)pt.first[blocks]);
        if constexpr (!std::is_same<T, double>::value) {
          if (scales) {
            hipLaunchKernelGGL((k_rms_fwd<T, V, LPR, NV, true>), grid, dim3(N), 0, (hipStream_t)stream, (const T*)x,
                               (const T*)residual, weight, weight_wide != 0, rows, pt, (S)eps, (T*)h, y, scales, (S*)inv);
            return;
          }
        }
        hipLaunchKernelGGL((k_rms_fwd<T, V, LPR, NV, false>), grid, dim3(N), 0, (hipStream_t)stream, (const T*)x,
                           (const T*)residual, weight, weight_wide != 0, rows, pt, (S)eps, (T*)h, y, scales, (S*)inv);
      });
    };
    if (channels % W == 0 && row_aligned(x) && row_aligned(residual) && row_aligned(weight) && row_aligned(h) &&
        row_aligned(y))
      launch(std::integral_constant<int, W>());
    else
      launch(std::integral_constant<int, 1>());
  });
  return tace_check_launch("rms_norm_fwd");
}

extern "C" int64_t tace_rms_norm_bwd_work(int type, int64_t rows, int32_t channels, int32_t blocks,
                                          const int32_t* comps) {
  if (check_norm(rows, channels, blocks, comps)) return -1;
  int64_t bytes = -1;
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    constexpr int W = 16 / sizeof(T);
    const int64_t one = part_elems<1>(rows, channels, blocks, comps);
    const int64_t vec = channels % W == 0 ? part_elems<W>(rows, channels, blocks, comps) : 0;
    bytes = (one > vec ? one : vec) * (int64_t)sizeof(row_sum_t<T>);
  });
  if (bytes < 0) tace_fail_msg("rms_norm: unknown row type");
  return bytes;
}

extern "C" int tace_rms_norm_bwd(int type, const void* gy, const void* gh, const void* h, const void* weight,
                                 int weight_wide, const void* inv, int64_t rows, int32_t channels, int32_t blocks,
                                 const int32_t* comps, void* dh, void* dw, void* work, int64_t work_bytes,
                                 void* stream) {
  if (check_norm(rows, channels, blocks, comps)) return -1;
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("rms_norm: unknown row type");
  if (rows == 0) return tace_fail_msg("rms_norm: no rows have no gradient");
  if (!gy || !h || !weight || !inv || !dh) return tace_fail_msg("rms_norm: null argument");
  if (dw && (!work || !row_aligned(work) ||
             work_bytes < tace_rms_norm_bwd_work(type, rows, channels, blocks, comps)))
    return tace_fail_msg("rms_norm: the workspace is too small or not 16-byte aligned");
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    typedef row_sum_t<T> S;
    constexpr int W = 16 / sizeof(T);
    auto launch = [&](auto v) {
      constexpr int V = decltype(v)::value;
      row_shape<V>(widest(blocks, comps) * channels / V, [&](auto lpr, auto nv) {
        constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value, N = LPR > WG ? LPR : WG;
        const NormParts pt = make_parts(rows, channels, blocks, comps, N / LPR, BWD_WGS);
        hipLaunchKernelGGL((k_rms_bwd<T, V, LPR, NV>), dim3((unsigned)pt.first[blocks]), dim3(N), 0,
                           (hipStream_t)stream, (const T*)gy, (const T*)gh, (const T*)h, weight, weight_wide != 0,
                           (const S*)inv, rows, pt, (T*)dh, dw ? (S*)work : (S*)nullptr);
        if (dw)
          hipLaunchKernelGGL((k_rms_dw<T>), dim3((unsigned)((channels + SUM_COLS - 1) / SUM_COLS), (unsigned)blocks),
                             dim3(SUM_COLS * SUM_ROWS), 0, (hipStream_t)stream, (const S*)work, pt, LPR <= WG,
                             weight_wide != 0, dw);
      });
    };
    if (channels % W == 0 && row_aligned(gy) && row_aligned(gh) && row_aligned(h) && row_aligned(weight) &&
        row_aligned(dh))
      launch(std::integral_constant<int, W>());
    else
      launch(std::integral_constant<int, 1>());
  });
  return tace_check_launch("rms_norm_bwd");
}
