// Linear layers of experts: matrix products of ragged groups of rows, each with
// its expert's weights, and their gradients.
//
// Rows sorted by expert (rowptr [E + 1], on the device: no size of a group is
// known to the host) in `blocks` blocks of comps[b] rows of K elements each, so
// group (b, e) is rows  R before[b] + comps[b] rowptr[e] ..  of one matrix, and
//   Y = s X W[e][b],   dX = s G W[e][b]^T,   dW[e][b] = s X^T G
// are one kernel over output tiles: A [M, n] B [n, N] with either operand stored
// along the summed index or across it.
//
// Tiles without a table: group g of the sorted groups takes tile slots
// start(g) / TM + g and up, at least ceil(length / TM) of them since
// floor(end / TM) - floor(start / TM) + 1 >= ceil((end - start) / TM); so slot ->
// group is one ballot over the starts, and rows / TM + groups slots cover all.
//
// Tiles pass through LDS, the next step's loads in registers meanwhile.  An
// operand stored along the summed index is read from LDS as 16-byte fragments,
// one stored across it by the transposing read (ds_read_b64_tr_b16).  LDS rows
// are permuted in 16- or 32-byte pieces so that either read meets every bank
// once.  bfloat16 and float16 go to the MFMA as they are, float32 as three
// bfloat16 terms (bf16x3.h, split as it enters LDS), e4m3 codes as the bfloat16
// of the same value; sums are float32.  (The MFMA of 8-bit codes has twice the
// rate, but aligns the products it adds to few bits: off by up to 2^-11.9 of the
// largest product for random codes of all exponents and 2^-17 of the sum of
// magnitudes for normally distributed ones, 16 x 16 x 128 and 16 x 16 x 32 alike.
// Few tokens are bound by reading the weights, which either form does once.)
// float64 has a kernel of its own.
#include "bf16x3.h"
#include "row_types.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef double d4 __attribute__((ext_vector_type(4)));

constexpr int WG = 256;

struct E4m3 {
  unsigned short pair;   // two codes: rows are addressed by pairs
};

// ------------------------------------------------------------------ groups ----
struct Groups {
  const int* rowptr;
  int64_t rows;   // of rowptr, dropped ones among them
  int experts, blocks;
  int comps[TACE_ROW_MAX_BLOCKS], before[TACE_ROW_MAX_BLOCKS];

  // (rows outside the range and orders that are none give other groups, but rows in range)
  __device__ __forceinline__ int64_t end_of(int e) const {   // first row of expert e; of the dropped rows for e = experts
    if (e > experts) return rows;
    const int64_t v = rowptr[e];
    return v < 0 ? 0 : v > rows ? rows : v;
  }
};

struct Place {
  int64_t first;    // row of the stacked blocks
  int64_t count;    // rows from there on
  int64_t group0;   // the group's first row
  int64_t part;     // slots of the group before this one
  int expert, block;
};

// The group of a slot of 2^shift rows, its rows from the slot's on (count <= 0:
// none).  Groups of a block: the experts, and the dropped rows as one more.
__device__ __forceinline__ Place place_of(const Groups& gr, int slot, int shift) {
  const int lane = (int)threadIdx.x & 63, per = gr.experts + 1, n = per * gr.blocks;
  int found = 0;
  for (int g0 = 0; g0 < n; g0 += 64) {
    const int g = g0 + lane;
    bool ok = false;
    if (g < n) {
      const int b = g / per, e = g - b * per;
      const int64_t start = gr.rows * gr.before[b] + gr.comps[b] * gr.end_of(e);
      ok = (start >> shift) + g <= slot;
    }
    const int here = __popcll(__ballot(ok));
    found += here;
    if (here < 64) break;
  }
  const int g = __builtin_amdgcn_readfirstlane(found > 0 ? found - 1 : 0);
  Place p;
  p.block = g / per;
  p.expert = g - p.block * per;
  const int64_t base = gr.rows * gr.before[p.block];
  p.group0 = base + gr.comps[p.block] * gr.end_of(p.expert);
  const int64_t end = base + gr.comps[p.block] * gr.end_of(p.expert + 1);
  p.part = (int64_t)slot - g - (p.group0 >> shift);
  p.first = p.group0 + (p.part << shift);
  p.count = end - p.first;
  return p;
}

// workgroups of an XCD (every eighth) take a contiguous range of tiles
__device__ __forceinline__ int tile_of(int tiles) {
  const int per = (int)(gridDim.x >> 3), i = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  return i < tiles ? i : -1;
}

// ----------------------------------------------------------------- operand ----
// T in memory -> 16-bit planes in LDS.  A step is BK of the summed index.
template <typename T>
struct Plane {
  static constexpr int COUNT = 1, BK = 64;
};
template <>
struct Plane<float> {
  static constexpr int COUNT = 3, BK = 32;
};

template <typename T>
struct Chunk {   // eight elements
  u4 v[sizeof(T) == 4 ? 2 : 1];
};

template <typename T>
__device__ __forceinline__ Chunk<T> zero_chunk() {
  Chunk<T> c;
#pragma unroll
  for (unsigned i = 0; i < sizeof(c.v) / sizeof(u4); ++i) c.v[i] = u4{0u, 0u, 0u, 0u};
  return c;
}

template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p) {   // 16-byte aligned
  Chunk<T> c;
#pragma unroll
  for (unsigned i = 0; i < sizeof(c.v) / sizeof(u4); ++i) c.v[i] = ((const u4*)p)[i];
  return c;
}

// the first n of eight elements anywhere, zeros behind them
template <typename T>
__device__ __forceinline__ Chunk<T> load_some(const T* p, int n) {
  union {
    T e[8];
    Chunk<T> c;
  } r;
  r.c = zero_chunk<T>();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) r.e[i] = p[i];
  return r.c;
}

// One operand's tile: TM outputs by BK of the summed index.  ACROSS: memory runs
// along the outputs (element (i, k) at p + k ld + i), else along the summed index
// (p + i ld + k).
template <typename T, int TM, bool ACROSS>
struct Tile {
  static constexpr int P = Plane<T>::COUNT, BK = Plane<T>::BK, CHUNKS = TM * BK / 8, PER = (CHUNKS + WG - 1) / WG;
  static constexpr int ELEMS = P * TM * BK;   // 16-bit
  static constexpr bool ALL = CHUNKS % WG == 0;

  Chunk<T> r[PER];

  // (line, piece) of a thread's q-th chunk: lines are outputs, or steps of the summed index
  __device__ __forceinline__ static void at(int q, int* line, int* piece) {
    constexpr int PIECES = (ACROSS ? TM : BK) / 8;
    const int u = (int)threadIdx.x + WG * q;
    *line = u / PIECES;
    *piece = u % PIECES;
  }

  // LDS place (16-bit elements) of a piece of eight
  __device__ __forceinline__ static int lds_at(int line, int piece) {
    if constexpr (ACROSS) {
      // 32-byte slots: eight (four, two) lines share the banks a transposing read's half wave takes
      constexpr int SLOTS = TM / 16;
      const int f = SLOTS >= 8 ? (line & 3) | ((line >> 1) & 4) : SLOTS == 4 ? ((line >> 1) & 1) | ((line >> 2) & 2)
                                                                            : (line >> 3) & (SLOTS - 1);
      return line * TM + (((piece >> 1) ^ f) << 4) + ((piece & 1) << 3);
    } else {
      return line * BK + ((piece ^ (BK == 64 ? (line >> 1) & 7 : (line >> 2) & 3)) << 3);
    }
  }

  // FAST: sizes are multiples of eight and rows 16-byte aligned; loads are
  // unconditional at clamped places (store() puts zeros past the summed index).
  // rows: where given, output i is read from row rows[i] (not ACROSS).
  template <bool FAST>
  __device__ __forceinline__ void load(const T* __restrict__ p, int64_t ld, int outs, int64_t k0, int64_t n,
                                       const int* rows) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      int line, piece;
      at(q, &line, &piece);
      if (!ALL && line >= (ACROSS ? BK : TM)) continue;
      if constexpr (ACROSS) {
        const int64_t k = k0 + line;
        if constexpr (FAST) {
          const int i = min(8 * piece, outs - 8);
          r[q] = load_chunk<T>(p + min(k, n - 1) * ld + i);
        } else {
          r[q] = k < n ? load_some<T>(p + k * ld + 8 * piece, outs - 8 * piece) : zero_chunk<T>();
        }
      } else {
        const int i = min(line, outs - 1);
        const T* row = p + (rows ? (int64_t)rows[i] : (int64_t)i) * ld;
        const int64_t k = k0 + 8 * piece;
        if constexpr (FAST) r[q] = load_chunk<T>(row + min(k, n - 8));
        else r[q] = k < n ? load_some<T>(row + k, (int)min(n - k, (int64_t)8)) : zero_chunk<T>();
      }
    }
  }

  __device__ __forceinline__ void store(unsigned short* lds, int64_t k0, int64_t n) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      int line, piece;
      at(q, &line, &piece);
      if (!ALL && line >= (ACROSS ? BK : TM)) continue;
      const bool in = k0 + (ACROSS ? line : 8 * piece) < n;
      unsigned short* d = lds + lds_at(line, piece);
      Chunk<T> c = r[q];
      if (!in) c = zero_chunk<T>();
      if constexpr (P == 3) {
        bx3_bf8 t[3];
        bx3_split8((const float*)&c, t);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(u4*)(d + i * TM * BK) = __builtin_bit_cast(u4, t[i]);
      } else {
        *(u4*)d = c.v[0];
      }
    }
  }

  // eight of the summed index, 8 fg + 32 s .., of output 16 j + fr (plane i)
  __device__ __forceinline__ static s8 fragment(const unsigned short* lds, int j, int s, int i, int fr, int fg) {
    const unsigned short* l = lds + i * TM * BK;
    if constexpr (ACROSS) {
      // (16 lanes give 4 lines of 32 bytes and get a column each)
      union {
        s4 h[2];
        s8 v;
      } o;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int line = 32 * s + 8 * fg + 4 * h + (fr >> 2);
        o.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4*)(l + lds_at(line, 2 * j + ((fr >> 1) & 1)) + ((fr & 1) << 2)));
      }
      return o.v;
    } else {
      return *(const s8*)(l + lds_at(16 * j + fr, 4 * s + fg));
    }
  }
};

template <typename T>
__device__ __forceinline__ f4 mfma(s8 a, s8 b, f4 c) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// eight e4m3 codes (half h of 16) as bfloat16, which holds them exactly
__device__ __forceinline__ s8 widen_codes(s8 c, int h) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const u4 w = __builtin_bit_cast(u4, c);
  u4 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o[2 * i] = __builtin_bit_cast(unsigned, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[2 * h + i], 1.0f, false));
    o[2 * i + 1] = __builtin_bit_cast(unsigned, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[2 * h + i], 1.0f, true));
  }
  return __builtin_bit_cast(s8, o);
}

// acc[i][j][r]: output row 16 i + fr, column 16 j + 4 fg + r of a wavefront's tile
template <typename T, typename TA, typename TB, int FM, int FN>
__device__ __forceinline__ void step(const unsigned short* la, const unsigned short* lb, int i0, int j0, int fr, int fg,
                                     f4 (&acc)[FM][FN]) {
  constexpr int P = Plane<T>::COUNT;
  if constexpr (std::is_same<T, E4m3>::value) {
    // a lane's 16 codes are its eight of two MFMA steps: the same order of the
    // summed index in both operands
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      s8 a[FM], b[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = TA::fragment(la, i0 + i, s, 0, fr, fg);
#pragma unroll
      for (int j = 0; j < FN; ++j) b[j] = TB::fragment(lb, j0 + j, s, 0, fr, fg);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s8 x[FM], y[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) x[i] = widen_codes(a[i], h);
#pragma unroll
        for (int j = 0; j < FN; ++j) y[j] = widen_codes(b[j], h);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(y[j], x[i], acc[i][j]);
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < Plane<T>::BK / 32; ++s) {
      s8 a[FM][P], b[FN][P];
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) a[i][p] = TA::fragment(la, i0 + i, s, p, fr, fg);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int p = 0; p < P; ++p) b[j][p] = TB::fragment(lb, j0 + j, s, p, fr, fg);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          if constexpr (P == 3) {
#pragma unroll
            for (int t = 0; t < 6; ++t) acc[i][j] = mfma<T>(b[j][BX3_TB[t]], a[i][BX3_TA[t]], acc[i][j]);
          } else {
            acc[i][j] = mfma<T>(b[j][0], a[i][0], acc[i][j]);
          }
        }
    }
  }
}

// ------------------------------------------------------------------ kernel ----
// What a tile is: its operands from its first row / column on, and where it goes.
template <typename T>
struct Work {
  const T *a, *b;
  int64_t lda, ldb, sum;   // sum: length of the summed index
  int m, n;                // valid rows and columns (to the operands' ends)
  const int* rows;         // A's rows, or null
};

// Float32 sums of three terms that are not finite are made again from the inputs:
// an infinity's second term is a NaN where float32's own product is infinite.
template <typename T, bool AT, bool BT>
__device__ float sum_again(const Work<T>& w, int i, int j) {
  float s = 0.0f;
  for (int64_t k = 0; k < w.sum; ++k)
    s = fmaf((float)w.a[AT ? k * w.lda + i : i * w.lda + k], (float)w.b[BT ? k * w.ldb + j : j * w.ldb + k], s);
  return s;
}

template <typename T, bool AT, bool BT, int WM, int WN, int FM, int FN, bool FAST, typename Store>
__device__ __forceinline__ void product(const Work<T>& w, unsigned short* lds, Store&& put) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN, BK = Plane<T>::BK;
  typedef Tile<T, TM, AT> TA;
  typedef Tile<T, TN, BT> TB;
  static_assert(WM * WN * 64 == WG, "four wavefronts");
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, fr = lane & 15, fg = lane >> 4;
  const int i0 = wave / WN * FM, j0 = wave % WN * FN;
  unsigned short *la = lds, *lb = lds + TA::ELEMS;
  f4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  TA a;
  TB b;
  if (w.sum > 0) {
    a.template load<FAST>(w.a, w.lda, w.m, 0, w.sum, w.rows);
    b.template load<FAST>(w.b, w.ldb, w.n, 0, w.sum, nullptr);
  }
  for (int64_t k0 = 0; k0 < w.sum; k0 += BK) {
    __syncthreads();   // (the last step's readers)
    a.store(la, k0, w.sum);
    b.store(lb, k0, w.sum);
    __syncthreads();
    if (k0 + BK < w.sum) {
      a.template load<FAST>(w.a, w.lda, w.m, k0 + BK, w.sum, w.rows);
      b.template load<FAST>(w.b, w.ldb, w.n, k0 + BK, w.sum, nullptr);
    }
    step<T, TA, TB, FM, FN>(la, lb, i0, j0, fr, fg, acc);
  }
  float z = 0.0f;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      put(16 * (i0 + i) + fr, 16 * (j0 + j) + 4 * fg, acc[i][j]);
      if constexpr (Plane<T>::COUNT == 3) {
#pragma unroll
        for (int r = 0; r < 4; ++r) z = fmaf(acc[i][j][r], 0.0f, z);
      }
    }
  if constexpr (Plane<T>::COUNT == 3) {
    if (z == z) return;
    unsigned long long bad[(FM * FN + 15) / 16] = {};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(fabsf(acc[i][j][r]) < __builtin_inff()))
            bad[(i * FN + j) / 16] |= 1ull << (4 * ((i * FN + j) % 16) + r);
#pragma unroll
    for (int q = 0; q < (FM * FN + 15) / 16; ++q) {
      while (bad[q]) {
        const int bit = __ffsll((long long)bad[q]) - 1, f = 16 * q + (bit >> 2);
        bad[q] &= bad[q] - 1;
        const int row = 16 * (i0 + f / FN) + fr, col = 16 * (j0 + f % FN) + 4 * fg + (bit & 3);
        if (row < w.m && col < w.n) put.one(row, col, sum_again<T, AT, BT>(w, row, col));
      }
    }
  }
}

// stores of a tile's four consecutive columns
template <typename O>
struct Put {
  O* out;   // the tile's first element
  int64_t ldo;
  int m, n;
  float scale;
  bool fours;   // rows of a multiple of four, aligned
  const float *row_scale, *col_scale;   // of the tile's rows (by `rows` where given) and columns, or null
  const int* rows;
  __device__ __forceinline__ void one(int i, int j, float v) const {
    out[i * ldo + j] = (O)(v * scale);
  }
  __device__ __forceinline__ void operator()(int i, int j, f4 v) const {
    if (i >= m || j >= n) return;
    float s = scale;
    if (row_scale) s *= row_scale[rows ? rows[i] : i];
    O* p = out + i * ldo + j;
    if (fours) {
      typedef O o4 __attribute__((ext_vector_type(4)));
      o4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (O)(v[r] * (col_scale ? s * col_scale[j + r] : s));
      *(o4*)p = o;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j + r < n) p[r] = (O)(v[r] * (col_scale ? s * col_scale[j + r] : s));
    }
  }
};

template <typename O>
__device__ __forceinline__ void zero_rows(O* out, int64_t ldo, int m, int n) {
  for (int u = (int)threadIdx.x; u < m * n; u += WG) out[(u / n) * ldo + u % n] = (O)0.0f;
}

// Y = s X W (BT) or dX = s G W^T: a group's rows by all columns
template <typename T, bool BT, int WM, int WN, int FM, int FN, bool FAST>
__global__ __launch_bounds__(WG) void k_expert_rows(const T* __restrict__ x, const T* __restrict__ weight, Groups gr,
                                                    int64_t wsize, int sum, int n, float scale, T* __restrict__ out,
                                                    int tiles, int cols) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  __shared__ __attribute__((aligned(16))) unsigned short lds[Tile<T, TM, false>::ELEMS + Tile<T, TN, BT>::ELEMS];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const Place p = place_of(gr, t / cols, __builtin_ctz(TM));
  if (p.count <= 0) return;
  const int c0 = t % cols * TN, m = (int)min(p.count, (int64_t)TM), nn = n - c0;
  T* o = out + p.first * n + c0;
  if (p.expert >= gr.experts) {
    zero_rows(o, n, m, min(nn, TN));
    return;
  }
  const T* wt = weight + ((int64_t)p.expert * gr.blocks + p.block) * wsize;
  const Work<T> w{x + p.first * sum, wt + (BT ? (int64_t)c0 : (int64_t)c0 * sum), sum, BT ? n : sum, sum, m, nn, nullptr};
  product<T, false, BT, WM, WN, FM, FN, FAST>(w, lds, Put<T>{o, n, m, nn, scale, FAST, nullptr, nullptr, nullptr});
}

// dW: up to 2^shift rows of a group, by tiles of [K, N].  A group of one such
// part goes to dw itself, others as float32 sums to part [slots, K N].
template <typename T, int WM, int WN, int FM, int FN, bool FAST>
__global__ __launch_bounds__(WG) void k_expert_weights(const T* __restrict__ x, const T* __restrict__ g, Groups gr,
                                                       int shift, int K, int N, float scale, T* __restrict__ dw,
                                                       float* __restrict__ part, int tiles, int per, int cols) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  __shared__ __attribute__((aligned(16))) unsigned short lds[Tile<T, TM, true>::ELEMS + Tile<T, TN, true>::ELEMS];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const int slot = t / per, tile = t - slot * per, r0 = tile / cols * TM, c0 = tile % cols * TN;
  const Place p = place_of(gr, slot, shift);
  if (p.expert >= gr.experts || (p.part > 0 && p.count <= 0)) return;
  const int64_t n = min(max(p.count, (int64_t)0), (int64_t)1 << shift);
  const Work<T> w{x + p.first * K + r0, g + p.first * N + c0, K, N, n, K - r0, N - c0, nullptr};
  const int64_t at = (int64_t)r0 * N + c0, size = (int64_t)K * N;
  if (p.part == 0 && p.count <= n) {
    T* o = dw + ((int64_t)p.expert * gr.blocks + p.block) * size + at;
    product<T, true, true, WM, WN, FM, FN, FAST>(w, lds, Put<T>{o, N, K - r0, N - c0, scale, FAST, nullptr, nullptr, nullptr});
  } else {
    product<T, true, true, WM, WN, FM, FN, FAST>(
        w, lds, Put<float>{part + slot * size + at, N, K - r0, N - c0, 1.0f, FAST, nullptr, nullptr, nullptr});
  }
}

// dW of the groups of several parts: their sums in order
template <typename T>
__global__ __launch_bounds__(WG) void k_expert_join(const float* __restrict__ part, Groups gr, int shift, int64_t size,
                                                    float scale, T* __restrict__ dw) {
  const int b = (int)blockIdx.y / gr.experts, e = (int)blockIdx.y - b * gr.experts;
  const int64_t base = gr.rows * gr.before[b], first = base + gr.comps[b] * gr.end_of(e);
  const int64_t n = base + gr.comps[b] * gr.end_of(e + 1) - first;
  const int parts = (int)((n + ((int64_t)1 << shift) - 1) >> shift);
  if (parts <= 1) return;
  const int64_t slot = (first >> shift) + b * (gr.experts + 1) + e;
  const float* p = part + slot * size;
  T* o = dw + ((int64_t)e * gr.blocks + b) * size;
  if ((size & 3) == 0 && ((uintptr_t)dw & 15) == 0) {
    const int64_t i = 4 * ((int64_t)blockIdx.x * WG + threadIdx.x);
    if (i >= size) return;
    f4 sum = *(const f4*)(p + i);
    for (int q = 1; q < parts; ++q) sum += *(const f4*)(p + q * size + i);
    typedef T o4 __attribute__((ext_vector_type(4)));
    o4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (T)(sum[r] * scale);
    *(o4*)(o + i) = v;
  } else {
    for (int64_t i = 4 * ((int64_t)blockIdx.x * WG) + threadIdx.x; i < min(size, 4 * ((int64_t)blockIdx.x + 1) * WG); i += WG) {
      float sum = p[i];
      for (int q = 1; q < parts; ++q) sum += p[q * size + i];
      o[i] = (T)(sum * scale);
    }
  }
}

// Y = s_row s_col (codes of X) (codes of W [E, N, K])^T, rows gathered where order is given
template <typename O, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WG) void k_expert_codes(const E4m3* __restrict__ x, const float* __restrict__ xs,
                                                     const int* __restrict__ order, unsigned choices, int tokens,
                                                     const E4m3* __restrict__ weight, const float* __restrict__ ws,
                                                     Groups gr, int pairs, int n, O* __restrict__ out, int tiles, int cols) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  __shared__ __attribute__((aligned(16))) unsigned short lds[Tile<E4m3, TM, false>::ELEMS + Tile<E4m3, TN, false>::ELEMS];
  __shared__ int rows[TM];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const Place p = place_of(gr, t / cols, __builtin_ctz(TM));
  if (p.count <= 0) return;
  const int c0 = t % cols * TN, m = (int)min(p.count, (int64_t)TM), nn = n - c0;
  O* o = out + p.first * n + c0;
  if (p.expert >= gr.experts) {
    zero_rows(o, n, m, min(nn, TN));
    return;
  }
  if (order) {   // (a slot outside the tokens is taken for the last)
    for (int i = (int)threadIdx.x; i < TM; i += WG) {
      const unsigned slot = (unsigned)order[p.first + min(i, m - 1)];
      rows[i] = (int)min(min(slot, (unsigned)gr.rows - 1) / choices, (unsigned)tokens - 1);
    }
    __syncthreads();
  }
  const E4m3* wt = weight + (int64_t)p.expert * n * pairs;
  const Work<E4m3> w{order ? x : x + p.first * pairs, wt + (int64_t)c0 * pairs, pairs, pairs, pairs, m, nn,
                     order ? rows : nullptr};
  product<E4m3, false, false, WM, WN, FM, FN, true>(
      w, lds, Put<O>{o, n, m, nn, 1.0f, (n & 3) == 0 && ((uintptr_t)out & 15) == 0, order ? xs : xs + p.first,
                     ws + (int64_t)p.expert * n + c0, order ? rows : nullptr});
}

// ----------------------------------------------------------------- float64 ----
// 64 x 64 tiles, 16 of the summed index a step, v_mfma_f64_16x16x4_f64 (a lane
// has one element of either operand; with the operands in turn it holds row
// lane % 16 and columns lane / 16 + 4 r of the product).
constexpr int DT = 64, DK = 16, DS = 80;   // LDS rows of 640 bytes: two lines of 16 doubles meet every bank once

template <bool ACROSS>
struct TileD {
  double r[4];
  __device__ __forceinline__ static void at(int q, int* i, int* k) {
    const int u = (int)threadIdx.x + WG * q;
    *i = ACROSS ? u % DT : u / DK;
    *k = ACROSS ? u / DT : u % DK;
  }
  __device__ __forceinline__ void load(const double* __restrict__ p, int64_t ld, int outs, int64_t k0, int64_t n) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int i, k;
      at(q, &i, &k);
      i = min(i, outs - 1);
      const int64_t kk = min(k0 + k, n - 1);
      r[q] = p[ACROSS ? kk * ld + i : i * ld + kk];
    }
  }
  __device__ __forceinline__ void store(double* lds, int64_t k0, int64_t n) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int i, k;
      at(q, &i, &k);
      lds[k * DS + i] = k0 + k < n ? r[q] : 0.0;
    }
  }
};

template <bool AT, bool BT, typename Store>
__device__ __forceinline__ void product_f64(const Work<double>& w, double* lds, Store&& put) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, fr = lane & 15, fg = lane >> 4;
  const int i0 = (wave >> 1) * 32, j0 = (wave & 1) * 32;
  double *la = lds, *lb = lds + DK * DS;
  d4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = d4{0, 0, 0, 0};
  TileD<AT> a;
  TileD<BT> b;
  if (w.sum > 0) {
    a.load(w.a, w.lda, w.m, 0, w.sum);
    b.load(w.b, w.ldb, w.n, 0, w.sum);
  }
  for (int64_t k0 = 0; k0 < w.sum; k0 += DK) {
    __syncthreads();
    a.store(la, k0, w.sum);
    b.store(lb, k0, w.sum);
    __syncthreads();
    if (k0 + DK < w.sum) {
      a.load(w.a, w.lda, w.m, k0 + DK, w.sum);
      b.load(w.b, w.ldb, w.n, k0 + DK, w.sum);
    }
#pragma unroll
    for (int s = 0; s < DK / 4; ++s) {
      double x[2], y[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = la[(4 * s + fg) * DS + i0 + 16 * i + fr];
        y[i] = lb[(4 * s + fg) * DS + j0 + 16 * i + fr];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(y[j], x[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) put(i0 + 16 * i + fr, j0 + 16 * j + fg + 4 * r, acc[i][j][r]);
}

template <bool BT>
__global__ __launch_bounds__(WG) void k_expert_rows_f64(const double* __restrict__ x, const double* __restrict__ weight,
                                                        Groups gr, int64_t wsize, int sum, int n, double scale,
                                                        double* __restrict__ out, int tiles, int cols) {
  __shared__ double lds[2 * DK * DS];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const Place p = place_of(gr, t / cols, __builtin_ctz(DT));
  if (p.count <= 0) return;
  const int c0 = t % cols * DT, m = (int)min(p.count, (int64_t)DT), nn = n - c0;
  double* o = out + p.first * n + c0;
  if (p.expert >= gr.experts) {
    zero_rows(o, n, m, min(nn, DT));
    return;
  }
  const double* wt = weight + ((int64_t)p.expert * gr.blocks + p.block) * wsize;
  const Work<double> w{x + p.first * sum, wt + (BT ? (int64_t)c0 : (int64_t)c0 * sum), sum, BT ? n : sum, sum, m, nn, nullptr};
  product_f64<false, BT>(w, lds, [&](int i, int j, double v) {
    if (i < m && j < nn) o[(int64_t)i * n + j] = v * scale;
  });
}

__global__ __launch_bounds__(WG) void k_expert_weights_f64(const double* __restrict__ x, const double* __restrict__ g,
                                                           Groups gr, int shift, int K, int N, double scale,
                                                           double* __restrict__ dw, double* __restrict__ part, int tiles,
                                                           int per, int cols) {
  __shared__ double lds[2 * DK * DS];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const int slot = t / per, tile = t - slot * per, r0 = tile / cols * DT, c0 = tile % cols * DT;
  const Place p = place_of(gr, slot, shift);
  if (p.expert >= gr.experts || (p.part > 0 && p.count <= 0)) return;
  const int64_t n = min(max(p.count, (int64_t)0), (int64_t)1 << shift);
  const Work<double> w{x + p.first * K + r0, g + p.first * N + c0, K, N, n, K - r0, N - c0, nullptr};
  const int64_t at = (int64_t)r0 * N + c0, size = (int64_t)K * N;
  const bool whole = p.part == 0 && p.count <= n;
  double* o = whole ? dw + ((int64_t)p.expert * gr.blocks + p.block) * size + at : part + slot * size + at;
  const double s = whole ? scale : 1.0;
  product_f64<true, true>(w, lds, [&](int i, int j, double v) {
    if (i < K - r0 && j < N - c0) o[(int64_t)i * N + j] = v * s;
  });
}

__global__ __launch_bounds__(WG) void k_expert_join_f64(const double* __restrict__ part, Groups gr, int shift,
                                                        int64_t size, double scale, double* __restrict__ dw) {
  const int b = (int)blockIdx.y / gr.experts, e = (int)blockIdx.y - b * gr.experts;
  const int64_t base = gr.rows * gr.before[b], first = base + gr.comps[b] * gr.end_of(e);
  const int64_t n = base + gr.comps[b] * gr.end_of(e + 1) - first;
  const int parts = (int)((n + ((int64_t)1 << shift) - 1) >> shift);
  if (parts <= 1) return;
  const double* p = part + ((first >> shift) + b * (gr.experts + 1) + e) * size;
  double* o = dw + ((int64_t)e * gr.blocks + b) * size;
  for (int64_t i = 4 * ((int64_t)blockIdx.x * WG) + threadIdx.x; i < min(size, 4 * ((int64_t)blockIdx.x + 1) * WG); i += WG) {
    double sum = p[i];
    for (int q = 1; q < parts; ++q) sum += p[q * size + i];
    o[i] = sum * scale;
  }
}

// -------------------------------------------------------------------- host ----
constexpr int64_t MOST_WGS = (int64_t)1 << 23;   // (below 2^31 threads)

int check_groups(int64_t rows, int experts, int blocks, const int32_t* comps, int32_t K, int32_t N, const int32_t* rowptr,
                 Groups* gr) {
  if (rows < 0 || rows > INT32_MAX - 8192 || experts < 0 || blocks < 1 || blocks > TACE_ROW_MAX_BLOCKS || !comps || K < 1 ||
      N < 1 || K > 65536 || N > 65536)
    return tace_fail_msg("expert_linear: bad sizes");
  int total = 0;
  for (int b = 0; b < blocks; ++b) {
    if (comps[b] < 1 || comps[b] > 1024) return tace_fail_msg("expert_linear: components are not 1 to 1024");
    gr->comps[b] = comps[b];
    gr->before[b] = total;
    total += comps[b];
  }
  if (experts > (1 << 20) || rows * total > (int64_t)INT32_MAX * 64)
    return tace_fail_msg("expert_linear: bad sizes");
  if (!rowptr) return tace_fail_msg("expert_linear: null argument");
  gr->rowptr = rowptr;
  gr->rows = rows;
  gr->experts = experts;
  gr->blocks = blocks;
  return 0;
}

int total_comps(const Groups& gr) { return gr.before[gr.blocks - 1] + gr.comps[gr.blocks - 1]; }
int64_t slots_of(const Groups& gr, int shift) {
  return ((gr.rows * total_comps(gr)) >> shift) + (int64_t)gr.blocks * (gr.experts + 1);
}
unsigned grid_of(int64_t tiles) { return (unsigned)((tiles + 7) / 8 * 8); }

// Tiles of 128 x 128 where they fill the card, 64 x 64 below, 16 x 128 for
// experts of a few rows each (a product then reads its weights once and little
// else; higher tiles would be mostly empty).
enum { T128, T64, T16 };
int rows_tile(const Groups& gr, int n) {
  const int64_t rows = gr.rows * total_comps(gr), groups = (int64_t)gr.blocks * (gr.experts > 0 ? gr.experts : 1);
  if (rows <= 24 * groups) return T16;
  return slots_of(gr, 7) * ((n + 127) / 128) >= 512 ? T128 : T64;
}

template <typename F>
void with_tile(int tile, F&& f) {
  using std::integral_constant;
  typedef integral_constant<int, 1> I1;
  typedef integral_constant<int, 2> I2;
  typedef integral_constant<int, 4> I4;
  if (tile == T128) f(I2(), I2(), I4(), I4());
  else if (tile == T64) f(I2(), I2(), I2(), I2());
  else f(I1(), I4(), I1(), I2());
}

// A weight gradient's rows go in parts of 2^shift: about 1,024 workgroups, at
// least 256 rows each.
int weight_shift(const Groups& gr, int64_t per) {
  const int64_t rows = gr.rows * total_comps(gr);
  int shift = 8;
  while (((int64_t)1 << shift) < rows && (rows >> shift) * per > 1024) ++shift;
  return shift;
}
bool weight_small(int K, int N) { return K <= 64 || N <= 64; }
int64_t weight_tiles(int type, int K, int N) {
  const int64_t t = type == TACE_ROW_F64 || weight_small(K, N) ? 64 : 128;
  return ((K + t - 1) / t) * ((N + t - 1) / t);
}
bool in_parts(const Groups& gr, int shift) {
  int most = 1;
  for (int b = 0; b < gr.blocks; ++b) most = gr.comps[b] > most ? gr.comps[b] : most;
  return gr.rows * most > (int64_t)1 << shift;
}

}  // namespace

extern "C" int tace_expert_linear(int type, int transposed, const void* x, const void* weight, const int32_t* rowptr,
                                  int64_t rows, int32_t experts, int32_t blocks, const int32_t* comps, int32_t K, int32_t N,
                                  double scale, void* out, void* stream) {
  Groups gr;
  if (check_groups(rows, experts, blocks, comps, K, N, rowptr, &gr)) return -1;
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("expert_linear: unknown row type");
  if (rows == 0) return 0;
  if (!x || (!weight && experts) || !out) return tace_fail_msg("expert_linear: null argument");
  const int sum = transposed ? N : K, n = transposed ? K : N;
  const int64_t wsize = (int64_t)K * N;
  if (type == TACE_ROW_F64) {
    const int64_t cols = (n + DT - 1) / DT, tiles = slots_of(gr, 6) * cols;
    if (tiles > MOST_WGS) return tace_fail_msg("expert_linear: bad sizes");
    if (transposed)
      hipLaunchKernelGGL((k_expert_rows_f64<false>), dim3(grid_of(tiles)), dim3(WG), 0, (hipStream_t)stream, (const double*)x,
                         (const double*)weight, gr, wsize, sum, n, scale, (double*)out, (int)tiles, (int)cols);
    else
      hipLaunchKernelGGL((k_expert_rows_f64<true>), dim3(grid_of(tiles)), dim3(WG), 0, (hipStream_t)stream, (const double*)x,
                         (const double*)weight, gr, wsize, sum, n, scale, (double*)out, (int)tiles, (int)cols);
    return tace_check_launch("expert_linear");
  }
  const bool fast = sum % 8 == 0 && n % 8 == 0 && row_aligned(x) && row_aligned(weight) && row_aligned(out);
  bool fits = true;
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    if constexpr (!std::is_same<T, double>::value) {
      with_tile(rows_tile(gr, n), [&](auto wm, auto wn, auto fm, auto fn) {
        constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, FM = decltype(fm)::value, FN = decltype(fn)::value;
        constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
        const int64_t cols = (n + TN - 1) / TN, tiles = slots_of(gr, __builtin_ctz(TM)) * cols;
        if (!(fits = tiles <= MOST_WGS)) return;
        auto launch = [&](auto bt, auto quick) {
          hipLaunchKernelGGL((k_expert_rows<T, decltype(bt)::value, WM, WN, FM, FN, decltype(quick)::value>),
                             dim3(grid_of(tiles)), dim3(WG), 0, (hipStream_t)stream, (const T*)x, (const T*)weight, gr,
                             wsize, sum, n, (float)scale, (T*)out, (int)tiles, (int)cols);
        };
        if (transposed) fast ? launch(std::false_type(), std::true_type()) : launch(std::false_type(), std::false_type());
        else fast ? launch(std::true_type(), std::true_type()) : launch(std::true_type(), std::false_type());
      });
    }
  });
  if (!fits) return tace_fail_msg("expert_linear: bad sizes");
  return tace_check_launch("expert_linear");
}

extern "C" int64_t tace_expert_linear_grad_work(int type, int64_t rows, int32_t experts, int32_t blocks,
                                                const int32_t* comps, int32_t K, int32_t N) {
  Groups gr;
  static const int32_t none = 0;
  if (check_groups(rows, experts, blocks, comps, K, N, &none, &gr)) return -1;
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("expert_linear: unknown row type"), -1;
  const int shift = weight_shift(gr, weight_tiles(type, K, N));
  if (!in_parts(gr, shift)) return 0;
  return slots_of(gr, shift) * K * N * (type == TACE_ROW_F64 ? 8 : 4);
}

extern "C" int tace_expert_linear_grad(int type, const void* x, const void* g, const int32_t* rowptr, int64_t rows,
                                       int32_t experts, int32_t blocks, const int32_t* comps, int32_t K, int32_t N,
                                       double scale, void* dw, void* work, int64_t work_bytes, void* stream) {
  Groups gr;
  if (check_groups(rows, experts, blocks, comps, K, N, rowptr, &gr)) return -1;
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("expert_linear: unknown row type");
  if (experts == 0) return 0;
  if ((rows && (!x || !g)) || !dw) return tace_fail_msg("expert_linear: null argument");
  const int64_t per = weight_tiles(type, K, N), size = (int64_t)K * N;
  const int shift = weight_shift(gr, per);
  const bool parts = in_parts(gr, shift);
  const int64_t tiles = slots_of(gr, shift) * per;
  if (tiles > MOST_WGS || (int64_t)blocks * experts > 65535) return tace_fail_msg("expert_linear: bad sizes");
  if (parts && (!work || !row_aligned(work) ||
                work_bytes < tace_expert_linear_grad_work(type, rows, experts, blocks, comps, K, N)))
    return tace_fail_msg("expert_linear: the workspace is too small or not 16-byte aligned");
  const dim3 grid(grid_of(tiles)), join((unsigned)((size + 4 * WG - 1) / (4 * WG)), (unsigned)(blocks * experts));
  const hipStream_t st = (hipStream_t)stream;
  if (type == TACE_ROW_F64) {
    hipLaunchKernelGGL(k_expert_weights_f64, grid, dim3(WG), 0, st, (const double*)x, (const double*)g, gr, shift, K, N,
                       scale, (double*)dw, (double*)work, (int)tiles, (int)per, (N + DT - 1) / DT);
    if (parts)
      hipLaunchKernelGGL(k_expert_join_f64, join, dim3(WG), 0, st, (const double*)work, gr, shift, size, scale, (double*)dw);
    return tace_check_launch("expert_linear_grad");
  }
  const bool fast = K % 8 == 0 && N % 8 == 0 && row_aligned(x) && row_aligned(g) && row_aligned(dw);
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    if constexpr (!std::is_same<T, double>::value) {
      with_tile(weight_small(K, N) ? T64 : T128, [&](auto wm, auto wn, auto fm, auto fn) {
        constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, FM = decltype(fm)::value, FN = decltype(fn)::value;
        if constexpr (WM == 2) {
          auto launch = [&](auto quick) {
            hipLaunchKernelGGL((k_expert_weights<T, WM, WN, FM, FN, decltype(quick)::value>), grid, dim3(WG), 0, st,
                               (const T*)x, (const T*)g, gr, shift, K, N, (float)scale, (T*)dw, (float*)work, (int)tiles,
                               (int)per, (N + 16 * WN * FN - 1) / (16 * WN * FN));
          };
          fast ? launch(std::true_type()) : launch(std::false_type());
        }
      });
      if (parts)
        hipLaunchKernelGGL((k_expert_join<T>), join, dim3(WG), 0, st, (const float*)work, gr, shift, size, (float)scale,
                           (T*)dw);
    }
  });
  return tace_check_launch("expert_linear_grad");
}

extern "C" int tace_expert_linear_e4m3(int out_type, const void* x, const float* x_scale, const int32_t* order,
                                       int32_t choices, const void* weight, const float* w_scale, const int32_t* rowptr,
                                       int64_t rows, int32_t experts, int32_t K, int32_t N, void* out, void* stream) {
  Groups gr;
  const int32_t one = 1;
  if (check_groups(rows, experts, 1, &one, K, N, rowptr, &gr)) return -1;
  if (out_type != TACE_ROW_F32 && out_type != TACE_ROW_BF16 && out_type != TACE_ROW_F16)
    return tace_fail_msg("expert_linear_e4m3: the output is float32, bfloat16 or float16");
  if (K % 16 != 0) return tace_fail_msg("expert_linear_e4m3: K is not a multiple of 16");
  if (choices < 1 || (order && rows % choices != 0)) return tace_fail_msg("expert_linear_e4m3: bad sizes");
  if (rows == 0) return 0;
  if (!x || !x_scale || (experts && (!weight || !w_scale)) || !out)
    return tace_fail_msg("expert_linear_e4m3: null argument");
  if (!row_aligned(x) || !row_aligned(weight)) return tace_fail_msg("expert_linear_e4m3: codes are not 16-byte aligned");
  bool fits = true;
  row_dispatch(out_type, [&](auto zero) {
    typedef decltype(zero) O;
    if constexpr (!std::is_same<O, double>::value) {
      with_tile(rows_tile(gr, N), [&](auto wm, auto wn, auto fm, auto fn) {
        constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, FM = decltype(fm)::value, FN = decltype(fn)::value;
        constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
        const int64_t cols = (N + TN - 1) / TN, tiles = slots_of(gr, __builtin_ctz(TM)) * cols;
        if (!(fits = tiles <= MOST_WGS)) return;
        hipLaunchKernelGGL((k_expert_codes<O, WM, WN, FM, FN>), dim3(grid_of(tiles)), dim3(WG), 0, (hipStream_t)stream,
                           (const E4m3*)x, x_scale, order, (unsigned)choices, (int)(rows / choices),
                           (const E4m3*)weight, w_scale, gr, K / 2, N, (O*)out, (int)tiles, (int)cols);
      });
    }
  });
  if (!fits) return tace_fail_msg("expert_linear_e4m3: bad sizes");
  return tace_check_launch("expert_linear_e4m3");
}
