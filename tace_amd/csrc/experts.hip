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
// Tiles without a table: every wavefront sums the groups' tiles up to each over its
// lanes and looks its own up there.  The products of rows are launched for a bound
// (rows / height + groups) and share out the tiles that exist; the weights'
// gradients cut the rows into stretches (see Units).
//
// 16-bit elements with sizes of multiples of eight and aligned rows are streamed:
// loads write LDS themselves, a step of 64 ahead, over all tiles of a workgroup
// without a pause (stream_products).  What else there is goes to LDS through
// registers (product): float32 as three bfloat16 terms (bf16x3.h, split on the
// way), e4m3 codes as they are, odd sizes element by element; float64 has its own
// MFMA (product_f64).  An operand stored along the summed index is read from LDS
// as 16-byte fragments, one stored across it by the transposing read
// (ds_read_b64_tr_b16); LDS rows are permuted in 16- or 32-byte pieces so that
// either read meets every bank once.  Sums are float32 (double for float64).
//
// e4m3 codes are multiplied as the bfloat16 of the same value.  The MFMA of 8-bit
// codes has up to three times the rate (library products of 8192 cubed: 3,214 and 1,066
// TFLOP/s), but aligns the products it adds to few bits: off by up to 2^-11.9 of the
// largest product for random codes of all exponents and 2^-17 of the sum of magnitudes
// for normally distributed ones, 16 x 16 x 128 and 16 x 16 x 32 alike.  An output of
// float32 would show either, one of 16 bits the first; prompts pay for it: 8,000
// tokens, 2 of 16 experts each, 1024 x 4096, 243 us (552 TFLOP/s, registers in between).
// Few tokens are bound by reading the weights, which either form does once: 24 tokens
// there 15.5 us, 16.4 as calls in a row with the weights in the caches, 17.5 (3.9
// TB/s) where ten layers' weights take turns.
//
// Measured, us (forward, rows' gradient, weights' gradient): bfloat16, 32,768 rows
// of 8 experts of 1024 x 2048: 187, 178, 176 + 19 (137 GFLOP each; 735, 772 and 705
// TFLOP/s, from caches that hold other data; 950 forward from warm ones); 202,612
// rows of 16 experts of 256 x 512, bound by memory and the latency of four steps a
// tile: 109, 90, 75 + 14 (311 MB each, 2.9 to 3.5 TB/s).  float32, 196,608 rows of
// 128 x 128 (its three terms' MFMA takes as long as the memory): 66, 67, 54 + 15.
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

  // (rows outside the range and orders that are none give other groups, but rows in range; from row 0 to the
  // last in any case, so every row is some group's)
  __device__ __forceinline__ int64_t end_of(int e) const {   // first row of expert e; of the dropped rows for e = experts
    if (e > experts) return rows;
    if (e == 0) return 0;
    const int64_t v = rowptr[e];
    return v < 0 ? 0 : v > rows ? rows : v;
  }
};

__host__ __device__ inline int total_comps(const Groups& gr) { return gr.before[gr.blocks - 1] + gr.comps[gr.blocks - 1]; }

// Whether a result of so many bytes is stored past the caches (nt; streamed products
// alone): they hold 256 MB, so the next kernel finds little of as much in them, while it
// takes the place of what is read again.  (Measured at 104 and 207 MB; a quarter of the
// caches is a guess for what is between.)  202,612 rows of 256 x 512 in bfloat16 (207 MB forward, 104
// back): a forward and backward pass 271 us, 287 without.
__device__ __forceinline__ bool large_result(int64_t bytes) { return bytes >= ((int64_t)64 << 20); }

struct Place {
  int64_t first;    // row of the stacked blocks
  int64_t count;    // rows of the group from there on
  int expert, block;
};

// What a tile is, by elements from its operands' and outputs' first ones; a lane
// holds one, a wavefront takes them one after the other.
struct Job {
  int64_t a, b, out;
  int sum;          // the summed index
  int m, n;         // rows and columns, up to the tile's
  int kind, whole;

  __device__ __forceinline__ static int of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  __device__ __forceinline__ static int64_t of(int64_t v, int lane) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)v, lane);
    return (int64_t)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | lo);
  }
  __device__ __forceinline__ Job lane(int l) const {
    return Job{of(a, l), of(b, l), of(out, l), of(sum, l), of(m, l), of(n, l), of(kind, l), of(whole, l)};
  }
};
enum { NO_TILE, ZERO_TILE, PRODUCT };

// The sum over the lanes up to each (within rows of 16, then from row to row).
template <int CTRL, int ROWS>
__device__ __forceinline__ int plus_dpp(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int up_to_lane(int v) {
  v = plus_dpp<0x111, 0xf>(v);
  v = plus_dpp<0x112, 0xf>(v);
  v = plus_dpp<0x114, 0xf>(v);
  v = plus_dpp<0x118, 0xf>(v);
  v = plus_dpp<0x142, 0xa>(v);
  return plus_dpp<0x143, 0xc>(v);
}

// Numbers the slots of 2^shift rows of all groups without gaps and finds a slot's
// group, a slot a lane: 64 groups at a time are in the lanes, with the sum of their
// slots up to each.  Groups of a block: the experts and the dropped rows.
struct Places {
  const Groups& gr;
  int shift, n, base;   // base: the first group in the lanes
  int64_t from, to;     // this lane's group's rows
  int upto;             // slots of the lanes' groups up to this one

  __device__ __forceinline__ Places(const Groups& gr, int shift)
      : gr(gr), shift(shift), n((gr.experts + 1) * gr.blocks) {
    take(0);
  }
  __device__ __forceinline__ void take(int at) {
    const int lane = (int)threadIdx.x & 63, per = gr.experts + 1, g = at + lane;
    base = at;
    from = to = 0;
    int slots = 0;
    if (g < n) {
      const int b = g / per, e = g - b * per;
      const int64_t block0 = gr.rows * gr.before[b];
      from = block0 + gr.comps[b] * gr.end_of(e);
      to = block0 + gr.comps[b] * gr.end_of(e + 1);
      slots = to > from ? (int)((to - from + ((int64_t)1 << shift) - 1) >> shift) : 0;
    }
    upto = up_to_lane(slots);
  }
  __device__ __forceinline__ int last() const { return __builtin_amdgcn_readlane(upto, 63); }
  // all slots
  __device__ __forceinline__ int total() {
    if (n <= 64) return last();
    int sum = 0;
    for (int at = 0; at < n; at += 64) {
      take(at);
      sum += last();
    }
    return sum;
  }
  __device__ __forceinline__ Place place(int g, int64_t part, int64_t f, int64_t t) const {
    const int per = gr.experts + 1, b = g / per;
    return Place{f + (part << shift), t - f - (part << shift), g - b * per, b};
  }
  // a slot that is the same in all lanes
  __device__ __forceinline__ Place find_one(int slot) {
    int before = 0;
    for (int at = 0; at < n; at += 64) {
      if (n > 64) take(at);
      if (slot - before < last()) {
        const int l = __popcll(__ballot(before + upto <= slot));   // groups that end before
        return place(at + l, slot - before - (l ? Job::of(upto, max(l - 1, 0)) : 0), Job::of(from, l), Job::of(to, l));
      }
      before += last();
    }
    return Place{0, 0, gr.experts, 0};
  }
  // each lane's own (every lane of the wavefront calls it); slots behind the last give a place without rows
  __device__ __forceinline__ Place find(int slot) {
    Place p{0, 0, gr.experts, 0};
    int before = 0;
    for (int at = 0; at < n; at += 64) {
      if (n > 64) take(at);
      int lane = 0;   // the first of the 64 groups whose slots reach past this one
#pragma unroll
      for (int o = 32; o > 0; o >>= 1)
        if (__shfl(upto, lane + o - 1, 64) <= slot - before) lane += o;
      const int64_t f = __shfl((long long)from, lane, 64), t = __shfl((long long)to, lane, 64);
      const int prior = __shfl(upto, max(lane - 1, 0), 64);
      if (slot >= before && slot - before < last()) p = place(at + lane, slot - before - (lane ? prior : 0), f, t);
      before += last();
    }
    return p;
  }
};

// Tiles of an XCD (every eighth workgroup) are contiguous, its workgroups take them
// in turn: what runs together shares rows and columns in the XCD's L2.
struct Share {
  int first, end, step;
};
__device__ __forceinline__ Share share_of(int tiles) {
  const int x = (int)(blockIdx.x & 7);
  return {(int)((int64_t)tiles * x / 8) + (int)(blockIdx.x >> 3), (int)((int64_t)tiles * (x + 1) / 8), (int)(gridDim.x >> 3)};
}

// The (row, column) of tile t of rows x cols in blocks of eight rows, down the
// columns of a block: 64 tiles beside each other then have 8 rows and 8 columns
// of operands, where 64 along the rows had one to four rows and all columns.
__device__ __forceinline__ void blocked(int t, int rows, int cols, int* row, int* col) {
  const int block = t / (8 * cols), r = t - block * 8 * cols, high = min(rows - 8 * block, 8);
  *row = 8 * block + r % high;
  *col = r / high;
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

// the first n of eight elements anywhere, zeros behind them (eight go as 16-byte
// loads, which need no alignment but that of the elements)
template <typename T>
__device__ __forceinline__ Chunk<T> load_some(const T* p, int n) {
  union {
    T e[8];
    Chunk<T> c;
  } r;
  if (n >= 8) {
    __builtin_memcpy(&r.c, p, sizeof(r.c));
    return r.c;
  }
  r.c = zero_chunk<T>();
#pragma unroll
  for (int i = 0; i < 7; ++i)
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
      // 32-byte slots: eight (four) lines share the banks a transposing read's half wave takes
      static_assert(TM % 64 == 0, "tiles of 64 or 128");
      const int f = TM >= 128 ? (line & 3) | ((line >> 1) & 4) : ((line >> 1) & 1) | ((line >> 2) & 2);
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

// The same for 32 x 32 products of 16 of the summed index (a lane: eight of output
// lane % 32, from 8 (lane / 32) on); 16-bit elements, steps of 64.  (Their sums
// of 16 registers are updated in place, by the instruction's form; with those
// of four the compiler moved them about, 32 moves for 64 products.)
template <typename T, int TM, bool ACROSS>
struct WideTile {
  static constexpr int BK = 64, ELEMS = TM * BK;
  static_assert(sizeof(T) == 2 && TM % 64 == 0, "16-bit tiles");

  __device__ __forceinline__ static int lds_at(int line, int piece) {
    if constexpr (ACROSS) {
      // (16 lanes read 32 bytes of four lines; lines 8 apart, and the 32 bytes
      // beside, are read by the other lanes)
      const int f = (TM >= 128 ? (line & 3) << 1 : line & 2) | ((line >> 3) & 1);
      return line * TM + (((piece >> 1) ^ f) << 4) + ((piece & 1) << 3);
    } else {
      return line * BK + ((piece ^ ((line >> 1) & 7)) << 3);
    }
  }
  // A lane's first elements, of which all its fragments are at constant distances:
  // one for each of F blocks (ACROSS), or for each 16 of the summed index.  (The
  // compiler is kept from seeing how they come about: of longer sums it loses which
  // array they are in, and waits for the loads into the other one.)
  template <int F>
  struct At {
    int v[ACROSS ? F : BK / 16];
    __device__ __forceinline__ At(int block0, int lane) {
#pragma unroll
      for (int k = 0; k < (ACROSS ? F : BK / 16); ++k) {
        if constexpr (ACROSS)
          v[k] = lds_at(8 * (lane >> 5) + ((lane >> 2) & 3), 4 * (block0 + k) + ((lane >> 3) & 2) + ((lane >> 1) & 1)) +
                 ((lane & 1) << 2);
        else
          v[k] = lds_at(32 * block0 + (lane & 31), 2 * k + (lane >> 5));
        asm volatile("" : "+v"(v[k]));
      }
    }
  };
  // of block j's 16 s .. of the summed index
  template <int F>
  __device__ __forceinline__ static s8 fragment(const unsigned short* l, const At<F>& at, int j, int s) {
    if constexpr (ACROSS) {
      union {
        s4 h[2];
        s8 v;
      } o;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4*)(l + (16 * s + 4 * h) * TM + at.v[j]));
      return o.v;
    } else {
      return *(const s8*)(l + 32 * j * BK + at.v[s]);
    }
  }
};

typedef float f16v __attribute__((ext_vector_type(16)));
template <typename T>
__device__ __forceinline__ f16v mfma32(s8 a, s8 b, f16v c) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

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
// an infinity's second term is a NaN where float32's own product is infinite.  A sum
// that is NaN stays so, and ends.  16,384 rows of 2 experts of 512 x 512, forward and
// backward: 198 us; under a gradient of NaN 239, of one row of NaN 206 (one load at a
// time and to the sums' ends: 16,700; eight at a time cost usual products 1 %).
template <typename T, bool AT, bool BT>
__device__ float sum_again(const Work<T>& w, int i, int j) {
  const int64_t da = AT ? w.lda : 1, db = BT ? w.ldb : 1;
  const T *a = w.a + (AT ? (int64_t)i : i * w.lda), *b = w.b + (BT ? (int64_t)j : j * w.ldb);
  float s = 0.0f;
  int64_t k = 0;
  for (; k + 4 <= w.sum && s == s; k += 4) {   // (their loads go out together)
    float x[4], y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = (float)a[(k + u) * da], y[u] = (float)b[(k + u) * db];
#pragma unroll
    for (int u = 0; u < 4; ++u) s = fmaf(x[u], y[u], s);
  }
  for (; k < w.sum && s == s; ++k) s = fmaf((float)a[k * da], (float)b[k * db], s);
  return s;
}

template <typename T, bool AT, bool BT, int WM, int WN, int FM, int FN, bool FAST, typename Store>
__device__ __forceinline__ void product(const Work<T>& w, Store&& put) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN, BK = Plane<T>::BK;
  typedef Tile<T, TM, AT> TA;
  typedef Tile<T, TN, BT> TB;
  __shared__ __attribute__((aligned(16))) unsigned short lds[TA::ELEMS + TB::ELEMS];
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

// ------------------------------------------------- loads straight into LDS ----
// One operand's steps by loads that write LDS themselves (16 bytes a lane, a
// wavefront's 1,024 in a row): the permutation of LDS rows is made by the lanes'
// addresses, which repeat after a few loads but for whole lines.  Offsets past
// the descriptor's range read zeros: lines behind the tile's rows or the summed
// index's end cost no branch.
template <typename T, int TM, bool ACROSS, int WAVES>
struct Stream {
  typedef WideTile<T, TM, ACROSS> L;
  static constexpr int BK = L::BK, LINE = (ACROSS ? TM : BK) * 2, LOADS = TM * BK * 2 / 1024;
  static constexpr int COUNT = LOADS / WAVES;                 // a wavefront's
  static constexpr int LINES = 1024 / LINE;                   // a load's
  static constexpr unsigned NONE = 0x80000000u;
  // lines that differ by a multiple of 16 are permuted alike
  static constexpr int KINDS = COUNT < 16 / LINES ? COUNT : 16 / LINES;
  static_assert(sizeof(T) == 2 && LOADS % WAVES == 0 && LINES >= 1 && LINES <= 16, "whole loads, as many for each");

  const T* p;
  unsigned ld, range;    // bytes of a line, and up to the end of the last one with values
  int first;             // this wavefront's first load
  unsigned at[KINDS];    // this lane's offsets, in bytes,
  int k[KINDS];          // and places on the summed index (not ACROSS)

  __device__ __forceinline__ Stream() : first(__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * COUNT) {}
  __device__ __forceinline__ void set(const T* from0, int64_t elems, int outs) {
    p = from0;
    ld = (unsigned)elems * 2;
    range = (unsigned)outs * ld;
#pragma unroll
    for (int j = 0; j < KINDS; ++j) {
      int line, from;
      place(j, (int)threadIdx.x & 63, &line, &from);
      k[j] = from;
      at[j] = !ACROSS || from < outs ? (unsigned)line * ld + (unsigned)from * 2 : NONE;
    }
  }

  // the line and the first of the eight elements that this lane's j-th load brings
  __device__ __forceinline__ void place(int j, int lane, int* line, int* from) const {
    const int pos = (first + j) * 1024 + lane * 16;
    *line = pos / LINE;
    *from = L::lds_at(*line, pos % LINE / 16) - *line * (LINE / 2);   // (the permutation is its own inverse)
  }

  // the step at p, of which n of the summed index are left, into lds; then the next
  __device__ __forceinline__ void issue(unsigned short* lds, int n) {
    const unsigned most = ACROSS ? (n <= 0 ? 0u : min((unsigned)n, (unsigned)BK) * ld) : range;
    // (the same in every lane, which the compiler loses sight of)
    const uintptr_t u = (uintptr_t)p;
    const uintptr_t q = (uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 |
                        (unsigned)__builtin_amdgcn_readfirstlane((int)u);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)q, (short)0, __builtin_amdgcn_readfirstlane((int)most),
                                                        0x00027000);
    const unsigned line_bytes = (unsigned)__builtin_amdgcn_readfirstlane((int)ld);
    auto load = [&](int j, unsigned o) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(lds + (first + j) * 512), 16, (int)o, 0, 0, 0);
    };
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const unsigned o = at[j % KINDS] + (unsigned)(j / KINDS * KINDS * LINES) * line_bytes;
      load(j, ACROSS || k[j % KINDS] < n ? o : NONE);   // (n may be negative: a step of zeros)
    }
    p += ACROSS ? (int64_t)(ld / 2) * BK : BK;
    if (!ACROSS) range -= min(range, (unsigned)(BK * 2));
  }
};

// waits until at most LOADS of this wavefront's loads are in flight and (READS)
// none of its LDS reads, then for the other wavefronts.  (The builtin's counts
// are the compiler's too: it adds no waits of its own.)
template <int LOADS, bool READS>
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | (READS ? 0x0070 : 0x0f70));
  asm volatile("s_barrier" ::: "memory");
}

// the fragments of 32 of the summed index, of a wavefront's FM x FN blocks of 32
template <typename TA, typename TB, int FM, int FN>
struct Fragments {
  typedef typename TA::template At<FM> AtA;
  typedef typename TB::template At<FN> AtB;
  s8 a[2][FM], b[2][FN];
  __device__ __forceinline__ void read(const unsigned short* l, int half, const AtA& at_a, const AtB& at_b) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < FM; ++i) a[s][i] = TA::fragment(l, at_a, i, 2 * half + s);
#pragma unroll
      for (int j = 0; j < FN; ++j) b[s][j] = TB::fragment(l + TA::ELEMS, at_b, j, 2 * half + s);
    }
    __builtin_amdgcn_sched_barrier(0);   // (these go out before what follows)
  }
  template <typename T>
  __device__ __forceinline__ void multiply(f16v (&acc)[FM][FN]) const {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32<T>(b[s][j], a[s][i], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
};

// Products of 16-bit elements, sizes multiples of eight and rows aligned: a
// wavefront's list of tiles (the lanes in `mask`) as one stream of steps, so a
// tile's first loads fly while the one before is multiplied and stored.
//
// Two buffers of 64 of the summed index.  Either half's fragments are read while
// the other half is multiplied; the barrier is between the halves of a step, when
// its second half is in registers: the buffer then takes the step after the
// next, whose loads fly for a whole step.  Tiles take an even number of steps
// (the last may be zeros that no load brings), so a step's buffer is known to
// the compiler, as it must be for it to wait for no load in flight.
template <typename T, bool AT, bool BT, int WM, int WN, int FM, int FN, typename Store>
__device__ __forceinline__ void stream_products(const T* __restrict__ a_base, const T* __restrict__ b_base, int64_t lda,
                                                int64_t ldb, const Job& jobs, unsigned long long mask, Store& store) {
  constexpr int TM = 32 * WM * FM, TN = 32 * WN * FN, BK = 64;
  typedef WideTile<T, TM, AT> TA;
  typedef WideTile<T, TN, BT> TB;
  typedef Stream<T, TM, AT, WM * WN> SA;
  typedef Stream<T, TN, BT, WM * WN> SB;
  constexpr int NEXT = SA::COUNT + SB::COUNT;   // a step's loads of a wavefront
  // (arrays of their own: the compiler then knows which loads a read waits for)
  __shared__ __attribute__((aligned(16))) unsigned short even[TA::ELEMS + TB::ELEMS], odd[TA::ELEMS + TB::ELEMS];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int i0 = wave / WN * FM, j0 = wave % WN * FN;

  unsigned long long ahead = mask;   // tiles whose steps are not loaded yet
  int left = 0;                      // of the summed index of the one that is, from the next step on
  SA a;
  SB b;
  auto turn = [&]() {
    const int l = __ffsll((long long)ahead) - 1;
    ahead &= ahead - 1;
    a.set(a_base + Job::of(jobs.a, l), lda, Job::of(jobs.m, l));
    b.set(b_base + Job::of(jobs.b, l), ldb, Job::of(jobs.n, l));
    left = Job::of(jobs.sum, l);
  };
  auto load = [&](unsigned short* to) {
    a.issue(to, left);
    b.issue(to + TA::ELEMS, left);
    left -= BK;
  };
  turn();
  load(even);
  load(odd);
  arrive<NEXT, false>();
  const typename TA::template At<FM> at_a(i0, lane);
  const typename TB::template At<FN> at_b(j0, lane);
  Fragments<TA, TB, FM, FN> f, g;
  f.read(even, 0, at_a, at_b);
  g.read(even, 1, at_a, at_b);
  bool more = true;
  f16v acc[FM][FN];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f16v{};
  };
  // Loops begin with nothing to read until all loads are there (at a loop's head
  // the compiler no longer knows which are for the other buffer, and waits).
  auto pair = [&](auto stores) {
    f.template multiply<T>(acc);
    arrive<0, true>();
    if (left <= 0) {
      more = ahead != 0;
      if (more) turn();
    }
    if (more) load(even);
    if constexpr (decltype(stores)::value) store.later();
    f.read(odd, 0, at_a, at_b);
    g.template multiply<T>(acc);
    g.read(odd, 1, at_a, at_b);
    f.template multiply<T>(acc);
    arrive<decltype(stores)::value ? Store::STORES : 0, true>();   // (the stores after the loads stay in flight)
    if (more) load(odd);
    f.read(even, 0, at_a, at_b);   // (the next tile's, if there is one)
    g.template multiply<T>(acc);
    g.read(even, 1, at_a, at_b);
  };
  for (; mask; mask &= mask - 1) {
    const int l = __ffsll((long long)mask) - 1;
    clear();
    pair(std::true_type());
    for (int n = Job::of(jobs.sum, l) - 2 * BK; n > 0; n -= 2 * BK) pair(std::false_type());
    store.tile(jobs.lane(l), acc, lane, i0, j0);
  }
  store.later();
}

// stores of a tile's four consecutive columns
template <typename O>
struct Put {
  O* out;   // the tile's first element
  int64_t ldo;
  int m, n;
  row_sum_t<O> scale;
  const float *row_scale, *col_scale;   // of the tile's rows (by `rows` where given) and columns, or null
  const int* rows;
  __device__ __forceinline__ void one(int i, int j, float v) const {
    out[i * ldo + j] = (O)(v * scale);
  }
  __device__ __forceinline__ void operator()(int i, int j, double v) const {
    if (i < m && j < n) out[i * ldo + j] = (O)(v * scale);
  }
  __device__ __forceinline__ void operator()(int i, int j, f4 v) const {
    if (i >= m || j >= n) return;
    float s = (float)scale;
    if (row_scale) s *= row_scale[rows ? rows[i] : i];
    O* p = out + i * ldo + j;
    if (j + 4 <= n) {   // (one move, whatever the alignment)
      typedef O o4 __attribute__((ext_vector_type(4)));
      o4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (O)(v[r] * (col_scale ? s * col_scale[j + r] : s));
      __builtin_memcpy(p, &o, sizeof(o));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j + r < n) p[r] = (O)(v[r] * (col_scale ? s * col_scale[j + r] : s));
    }
  }
};

// the output, or float32 sums
template <typename T>
struct PutPart {
  Put<T> out;
  Put<row_sum_t<T>> part;
  bool whole;
  __device__ __forceinline__ void one(int i, int j, float v) const {
    if (whole) out.one(i, j, v);
    else part.one(i, j, v);
  }
  template <typename V>
  __device__ __forceinline__ void operator()(int i, int j, V v) const {
    if (whole) out(i, j, v);
    else part(i, j, v);
  }
};

// A tile's results rounded and kept, and stored behind the next tile's first loads:
// the step after waits for the loads alone (vmcnt counts both, in order), where
// stores at a tile's end were waited for by themselves.  A wavefront's blocks pass
// through 2 or 4 KB of its own in LDS before, so that a store writes whole rows of
// its blocks (128 bytes) and not 16 bytes of each of 32 rows.  (A lane holds row
// lane % 32 and columns 8 q + 4 (lane / 32) .. + 3 of a block of 32.)
template <typename T, int WAVES, int FM, int FN, typename Make>
struct Results {
  // pieces (PutPart) have too many registers in use for that, and long sums between them
  static constexpr bool LATE = std::is_same<std::decay_t<std::invoke_result_t<Make, const Job&>>, Put<T>>::value;
  static constexpr int SLOTS = 8 * FN, READS = SLOTS / 4;   // 8-byte slots of a row; 16-byte reads a lane for 32 rows
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  Make make;
  bool past;   // (large_result)
  static constexpr int STORES = LATE ? FM * READS : 0;
  static constexpr unsigned NONE = 0x80000000u;
  u4 lined[FM][READS];
  T* base;                  // the tile's first element,
  unsigned range, ld, at;   // and bytes of its rows, of a row, and before this lane's first

  __device__ __forceinline__ Results(Make make, bool past) : make(make), past(past), base(nullptr), range(0), ld(0), at(NONE) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int n = 0; n < READS; ++n) lined[i][n] = u4{0u, 0u, 0u, 0u};
  }
  __device__ __forceinline__ void tile(const Job& j, const f16v (&acc)[FM][FN], int lane, int i0, int j0) {
    const auto to = make(j);
    if constexpr (LATE) {
      rows_of(to, acc, lane, i0, j0);
    } else if (to.whole) {
      rows_of(to.out, acc, lane, i0, j0);
      flush();
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int k = 0; k < FN; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            to.part(32 * (i0 + i) + (lane & 31), 32 * (j0 + k) + 8 * q + 4 * (lane >> 5),
                    f4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]});
    }
  }
  __device__ __forceinline__ void rows_of(const Put<T>& put, const f16v (&acc)[FM][FN], int lane, int i0, int j0) {
    __shared__ __attribute__((aligned(16))) u2 stage[WAVES][32 * SLOTS];
    u2* w = stage[(int)threadIdx.x >> 6];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      // slots of a row in another order by row: two lanes to a bank in writing, one in reading
      const int row = lane & 31;
#pragma unroll
      for (int k = 0; k < FN; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          t4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (T)(acc[i][k][4 * q + r] * put.scale);
          w[row * SLOTS + ((8 * k + 2 * q + (lane >> 5)) ^ (row & (SLOTS - 1)))] = __builtin_bit_cast(u2, v);
        }
#pragma unroll
      for (int n = 0; n < READS; ++n) {
        const int u = lane + 64 * n, r = u / (SLOTS / 2), c = (u % (SLOTS / 2)) ^ ((r & (SLOTS - 1)) >> 1);
        int place = r * SLOTS + 2 * c;
        asm volatile("" : "+v"(place));   // (as At's)
        const u4 v = *(const u4*)(w + place);
        lined[i][n] = r & 1 ? u4{v[2], v[3], v[0], v[1]} : v;
      }
    }
    const int col = 32 * j0 + lane % (SLOTS / 2) * 8;   // (eight columns are all there or none)
    base = put.out;
    ld = (unsigned)put.ldo * 2;
    range = (unsigned)put.m * ld;
    at = col < put.n ? (unsigned)(32 * i0 + lane / (SLOTS / 2)) * ld + (unsigned)col * 2 : NONE;
  }
  // (STORES instructions whatever there is to store: the next step counts them)
  __device__ __forceinline__ void later() {
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LATE) flush();
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void flush() {
    const uintptr_t u = (uintptr_t)base;
    const uintptr_t q = (uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 |
                        (unsigned)__builtin_amdgcn_readfirstlane((int)u);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)q, (short)0, __builtin_amdgcn_readfirstlane((int)range),
                                                        0x00027000);
    const unsigned line = (unsigned)__builtin_amdgcn_readfirstlane((int)ld);
    auto all = [&](auto aux) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int n = 0; n < READS; ++n)
          __builtin_amdgcn_raw_buffer_store_b128(lined[i][n], rsrc, (int)(at + (unsigned)(32 * i + n * (128 / SLOTS)) * line),
                                                 0, decltype(aux)::value);
    };
    if (past) all(std::integral_constant<int, 2>());   // (nt)
    else all(std::integral_constant<int, 0>());
    range = 0;
  }
};

template <typename O>
__device__ __forceinline__ void zero_rows(O* out, int64_t ldo, int m, int n) {
  constexpr int V = 16 / sizeof(O);
  const int pieces = (n + V - 1) / V;
  for (int u = (int)threadIdx.x; u < m * pieces; u += (int)blockDim.x) {
    const int i = u / pieces, j = (u - i * pieces) * V;
    O* p = out + i * ldo + j;
    if (j + V <= n) {
      const u4 z = {0u, 0u, 0u, 0u};
      __builtin_memcpy(p, &z, sizeof(z));
    } else {
      for (int e = 0; j + e < n; ++e) p[e] = (O)0.0f;
    }
  }
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
__device__ __forceinline__ void product_f64(const Work<double>& w, Store&& put) {
  __shared__ double lds[2 * DK * DS];
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

template <typename T, bool FAST>
constexpr bool STREAMS = FAST && sizeof(T) == 2;

// waves a SIMD for a wavefront's tile of that many fragments
constexpr int waves_for(int fragments) { return fragments > 32 ? 1 : fragments > 4 ? 2 : 4; }

// Walks over a workgroup's tiles: make(t) gives each lane's, zero(job) fills one,
// put(job) stores a tile's results.
template <typename T, bool AT, bool BT, int WM, int WN, int FM, int FN, bool FAST, typename Make, typename Zero, typename Store>
__device__ __forceinline__ void walk(const T* __restrict__ a, const T* __restrict__ b, int64_t lda, int64_t ldb, Share sh, bool past,
                                     Make&& make, Zero&& zero, Store&& put) {
  for (int t0 = sh.first; t0 < sh.end; t0 += 64 * sh.step) {
    asm volatile("" : : : "memory");   // (what make() reads is read again)
    const int t = t0 + ((int)threadIdx.x & 63) * sh.step;
    Job jobs = make(min(t, sh.end - 1));
    if (t >= sh.end) jobs.kind = NO_TILE;
    for (unsigned long long z = __ballot(jobs.kind == ZERO_TILE); z; z &= z - 1) zero(jobs.lane(__ffsll((long long)z) - 1));
    unsigned long long mask = __ballot(jobs.kind == PRODUCT);
    if (mask == 0) continue;
    if constexpr (STREAMS<T, FAST>) {
      Results<T, WM * WN, FM / 2, FN / 2, std::decay_t<Store>> store(put, past);
      stream_products<T, AT, BT, WM, WN, FM / 2, FN / 2>(a, b, lda, ldb, jobs, mask, store);
      if (t0 + 64 * sh.step < sh.end) __syncthreads();
    } else {
      for (; mask; mask &= mask - 1) {
        const Job j = jobs.lane(__ffsll((long long)mask) - 1);
        const Work<T> w{a + j.a, b + j.b, lda, ldb, j.sum, j.m, j.n, nullptr};
        if constexpr (std::is_same<T, double>::value) product_f64<AT, BT>(w, put(j));
        else product<T, AT, BT, WM, WN, FM, FN, FAST>(w, put(j));
      }
    }
  }
}

// Y = s X W (BT) or dX = s G W^T: tiles of TM rows by TN columns
template <typename T, bool BT, int WM, int WN, int FM, int FN, bool FAST>
__global__ __launch_bounds__(64 * WM * WN, waves_for(FM * FN)) void k_expert_rows(
    const T* __restrict__ x, const T* __restrict__ weight, Groups gr, int64_t wsize, int sum, int n, row_sum_t<T> scale,
    T* __restrict__ out, int cols) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  const int slots = Places(gr, __builtin_ctz(TM)).total();
  walk<T, false, BT, WM, WN, FM, FN, FAST>(
      x, weight, sum, BT ? n : sum, share_of(slots * cols), large_result(gr.rows * total_comps(gr) * n * (int)sizeof(T)),
      [&](int t) {   // (asked for again for every 64 tiles: nothing of it stays in registers)
        int slot, col;
        blocked(t, slots, cols, &slot, &col);
        const Place p = Places(gr, __builtin_ctz(TM)).find(slot);
        const int c0 = col * TN;
        return Job{p.first * sum,
                   ((int64_t)p.expert * gr.blocks + p.block) * wsize + (BT ? (int64_t)c0 : (int64_t)c0 * sum),
                   p.first * n + c0, sum, (int)min(p.count, (int64_t)TM), min(n - c0, TN),
                   p.count <= 0 ? NO_TILE : p.expert < gr.experts ? PRODUCT : ZERO_TILE, 1};
      },
      [&](const Job& j) { zero_rows(out + j.out, n, j.m, j.n); },
      [&](const Job& j) { return Put<T>{out + j.out, n, j.m, j.n, scale, nullptr, nullptr, nullptr}; });
}

// dW: the groups' rows as one line of units of 128 (a group without rows is one
// unit, of zeros), cut into `cuts` equal stretches.  A stretch's groups' tiles of
// [K, N] are shared by `team` workgroups, which then read the same rows at the same
// time and have equal work, however the rows are spread over the groups.  (Equal
// lengths of a line of all tiles' units cost up to a third more: workgroups side
// by side were at different rows, and the L2 held none of them twice.)  A group
// within one stretch goes to dw itself; pieces of others go as float32 sums to
// part [2 cuts, tiles], first groups of a stretch before last ones, and are added
// up in order.
struct Units {
  const Groups& gr;
  int n;               // groups
  int64_t from, to;    // this lane's group's rows
  int upto;            // units of the lanes' groups up to this one

  __device__ __forceinline__ explicit Units(const Groups& gr) : gr(gr), n(gr.experts * gr.blocks) { take(0); }
  __device__ __forceinline__ static int64_t units(int64_t rows) { return rows > 0 ? (rows + 127) >> 7 : 1; }
  __device__ __forceinline__ void take(int at) {
    const int lane = (int)threadIdx.x & 63, g = at + lane;
    from = to = upto = 0;
    if (g < n) {
      const int b = g / gr.experts, e = g - b * gr.experts;
      from = gr.rows * gr.before[b] + gr.comps[b] * gr.end_of(e);
      to = gr.rows * gr.before[b] + gr.comps[b] * gr.end_of(e + 1);
      upto = (int)units(to - from);
    }
    upto = up_to_lane(upto);
  }
  __device__ __forceinline__ int last() const { return Job::of(upto, 63); }
  __device__ __forceinline__ int64_t total() {
    if (n <= 64) return last();
    int64_t sum = 0;
    for (int at = 0; at < n; at += 64) {
      take(at);
      sum += last();
    }
    return sum;
  }
  // the group of a unit below the total, the same in all lanes
  __device__ __forceinline__ int group_of(int64_t unit) {
    int64_t before = 0;
    for (int at = 0; at < n; at += 64) {
      if (n > 64) take(at);
      if (unit < before + last()) return at + __popcll(__ballot(before + upto <= unit));
      before += last();
    }
    return n - 1;
  }
  // each lane's own group (every lane of the wavefront calls it)
  struct Span {
    int64_t first, count;   // units
    int64_t row, rows;
  };
  __device__ __forceinline__ Span span(int g) {
    Span s{0, 1, 0, 0};
    int64_t before = 0;
    for (int at = 0; at < n; at += 64) {
      if (n > 64) take(at);
      const int l = min(max(g - at, 0), 63);
      const int64_t f = __shfl((long long)from, l, 64), t = __shfl((long long)to, l, 64);
      const int prior = __shfl(upto, max(l - 1, 0), 64);
      if (g >= at && g - at < 64) s = Span{before + (l ? prior : 0), units(t - f), f, t > f ? t - f : 0};
      before += last();
    }
    return s;
  }
};

// (a unit at least in each)
__device__ __forceinline__ int stretches(int64_t units, int cuts) { return (int)min(units, (int64_t)cuts); }
// the first unit of stretch i of n
__device__ __forceinline__ int64_t cut_of(int64_t units, int i, int n) { return units / n * i + units % n * i / n; }

template <typename T, int WM, int WN, int FM, int FN, bool FAST>
__global__ __launch_bounds__(64 * WM * WN, waves_for(FM * FN)) void k_expert_weights(
    const T* __restrict__ x, const T* __restrict__ g, Groups gr, int K, int N, row_sum_t<T> scale, T* __restrict__ dw,
    row_sum_t<T>* __restrict__ part, int per, int cols, int cuts, int team) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  const int64_t size = (int64_t)K * N;
  // (an XCD's workgroups beside each other)
  const int line = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  const int cut = line / team, mate = line - cut * team, rounds = (per - mate + team - 1) / team;
  if (rounds <= 0) return;
  int64_t u0, u1;
  int g0, groups;
  {
    Units units(gr);
    const int64_t total = units.total();
    const int n = stretches(total, cuts);
    if (cut >= n) return;
    u0 = cut_of(total, cut, n);
    u1 = cut_of(total, cut + 1, n);
    g0 = units.group_of(u0);
    groups = units.group_of(u1 - 1) - g0 + 1;
  }
  walk<T, true, true, WM, WN, FM, FN, FAST>(
      x, g, K, N, Share{0, groups * rounds, 1}, large_result(gr.experts * gr.blocks * size * (int)sizeof(T)),
      [&](int t) {
        const int of = t / rounds, tile = mate + (t - of * rounds) * team, grp = g0 + of;
        const Units::Span s = Units(gr).span(grp);
        int row, col;
        blocked(tile, per / cols, cols, &row, &col);
        const int r0 = row * TM, c0 = col * TN, b = grp / gr.experts, e = grp - b * gr.experts;
        const int64_t a = max(u0 - s.first, (int64_t)0), z = min(u1 - s.first, s.count);   // of the group's units
        const int64_t first = s.row + (a << 7), rows = min(z << 7, s.rows) - (a << 7);
        const bool whole = a == 0 && z == s.count;
        return Job{first * K + r0, first * N + c0,
                   whole ? ((int64_t)e * gr.blocks + b) * size + (int64_t)r0 * N + c0
                         : ((int64_t)(2 * cut + (of ? 1 : 0)) * per + tile) * TM * TN,
                   (int)rows, min(K - r0, TM), min(N - c0, TN), rows > 0 ? PRODUCT : ZERO_TILE, whole};
      },
      [&](const Job& j) { zero_rows(dw + j.out, N, j.m, j.n); },
      [&](const Job& j) {
        return PutPart<T>{{dw + j.out, N, j.m, j.n, scale, nullptr, nullptr, nullptr},
                          {part + j.out, TN, TM, TN, 1, nullptr, nullptr, nullptr}, j.whole != 0};
      });
}

// dW of the groups of several stretches: their pieces' sums in order
template <typename T, int TM, int TN>
__global__ __launch_bounds__(WG) void k_expert_join(const row_sum_t<T>* __restrict__ part, Groups gr, int K, int N,
                                                    row_sum_t<T> scale, T* __restrict__ dw, int per, int cols, int cuts, int parts) {
  typedef row_sum_t<T> s4v __attribute__((ext_vector_type(4)));
  const int64_t tile = blockIdx.x / parts;
  const int grp = (int)(tile / per), place = (int)(tile - (int64_t)grp * per);
  Units units(gr);
  const int64_t total = units.total();
  const Units::Span s = units.span(grp);
  cuts = stretches(total, cuts);
  // the stretch of a unit
  auto cut_with = [&](int64_t unit) {
    int i = (int)((float)unit / (float)total * cuts);
    i = min(max(i, 0), cuts - 1);
    while (i > 0 && cut_of(total, i, cuts) > unit) --i;
    while (i + 1 < cuts && cut_of(total, i + 1, cuts) <= unit) ++i;
    return i;
  };
  const int i0 = cut_with(s.first), i1 = cut_with(s.first + s.count - 1);
  if (i0 == i1) return;
  int row, col;
  blocked(place, per / cols, cols, &row, &col);
  const int r0 = row * TM, c0 = col * TN, b = grp / gr.experts, e = grp - b * gr.experts;
  T* o = dw + ((int64_t)e * gr.blocks + b) * K * N + (int64_t)r0 * N + c0;
  const int64_t step = (int64_t)2 * per * TM * TN;
  // (the first stretch's piece is of its last group, if it has more)
  const int64_t lead = cut_of(total, i0, cuts) < s.first ? step / 2 : 0;
  const int share = TM * TN / parts;
  for (int q = 4 * (int)threadIdx.x; q < share; q += 4 * WG) {
    const int at = (int)(blockIdx.x % parts) * share + q, i = at / TN, j = at % TN;
    if (r0 + i >= K || c0 + j >= N) continue;
    const row_sum_t<T>* p = part + (int64_t)place * TM * TN + at + i0 * step;
    s4v sum = *(const s4v*)(p + lead);
    int k = 1;
    const int count = i1 - i0 + 1;
    for (; k + 8 <= count; k += 8) {   // (their loads go out together)
      s4v v[8];
#pragma unroll
      for (int m = 0; m < 8; ++m) v[m] = *(const s4v*)(p + (k + m) * step);
#pragma unroll
      for (int m = 0; m < 8; ++m) sum += v[m];
    }
    for (; k < count; ++k) sum += *(const s4v*)(p + k * step);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (c0 + j + r < N) o[(int64_t)i * N + j + r] = (T)(sum[r] * scale);
  }
}

// Y = s_row s_col (codes of X) (codes of W [E, N, K])^T, rows gathered where order is given
template <typename O, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WG) void k_expert_codes(const E4m3* __restrict__ x, const float* __restrict__ xs,
                                                     const int* __restrict__ order, unsigned choices, int tokens,
                                                     const E4m3* __restrict__ weight, const float* __restrict__ ws,
                                                     Groups gr, int pairs, int n, O* __restrict__ out, int tiles, int cols) {
  constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
  __shared__ int rows[TM];
  const int t = tile_of(tiles);
  if (t < 0) return;
  const Place p = Places(gr, __builtin_ctz(TM)).find_one(t / cols);
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
      w, Put<O>{o, n, m, nn, 1.0f, order ? xs : xs + p.first,
                     ws + (int64_t)p.expert * n + c0, order ? rows : nullptr});
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

int64_t slots_of(const Groups& gr, int shift) {
  return ((gr.rows * total_comps(gr)) >> shift) + (int64_t)gr.blocks * (gr.experts + 1);
}
// the tiles that there are kernels for
template <typename T, bool FAST>
constexpr bool has_tile(int tm, int tn) {
  if (std::is_same<T, double>::value) return !FAST && tm == 64;
  return tm >= (STREAMS<T, FAST> ? 64 : 16);
}

template <typename F>
void choose(bool a, bool b, F&& f) {
  auto one = [&](auto x) { b ? f(x, std::true_type()) : f(x, std::false_type()); };
  a ? one(std::true_type()) : one(std::false_type());
}

unsigned grid_of(int64_t tiles) { return (unsigned)((tiles + 7) / 8 * 8); }
// workgroups that walk over tiles: as many as run at once
unsigned walkers(int64_t tiles, int most) { return grid_of(tiles < most ? tiles : most); }

// Tiles of 128 x 128 where there are 512 full ones, as many as run at once, 64 x 64
// below: 32,768 rows of 256 x 512 in bfloat16 take 18.5 us with the one and 21.3
// with the other, 8,192 rows 9.9 and 9.6, 2,048 rows of 128 x 128 in float32 12.8
// and 7.4, 768 rows of 1024 x 4096 for 16 experts 98.9 and 74.6.  16 x 128 for
// experts of up to 24 rows each in what does not stream (a product reads its
// weights once and little else): 48 rows there 53 us and, with 64 x 64, 67; 384
// rows 63 and 68, 768 rows 106 and 75.
enum { T128, T64, T16 };
bool fills(int64_t rows, int64_t cols) { return (rows >> 7) * ((cols + 127) / 128) >= 512; }
int rows_tile(const Groups& gr, int n, bool streams) {
  const int64_t rows = gr.rows * total_comps(gr), groups = (int64_t)gr.blocks * (gr.experts > 0 ? gr.experts : 1);
  if (!streams && rows <= 24 * groups) return T16;
  return fills(rows, n) ? T128 : T64;
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

// The weight gradient's tiles, by the same rule: 2,048 rows of 128 x 128 in float32
// take 22 us with 128 x 128 and 16 with 64 x 64, 196,608 rows 72 and 74; 202,612
// rows of 256 x 512 in bfloat16 96 and 149.  Many experts' matrices take the large
// ones too: most of the time goes to storing them.
int64_t tiles_of(int tile, int K, int N) {
  const int64_t t = tile == T64 ? 64 : 128;
  return ((K + t - 1) / t) * ((N + t - 1) / t);
}
int weight_tile(int type, const Groups& gr, int K, int N) {
  const bool wide = type != TACE_ROW_F64 && K > 64 && N > 64;
  const bool many = (int64_t)gr.blocks * gr.experts * tiles_of(T64, K, N) > 65536;
  return wide && (many || fills(gr.rows * total_comps(gr), 128 * tiles_of(T128, K, N))) ? T128 : T64;
}
// whether a group may have more than a unit
bool may_be_cut(const Groups& gr) {
  for (int b = 0; b < gr.blocks; ++b)
    if (gr.rows * gr.comps[b] > 128) return true;
  return false;
}
// As many workgroups as run at once, in teams whose members have one to four of the
// tiles each, whichever leaves the fewest idle.
struct Teams {
  int cuts, team;
};
Teams teams_of(int tile, const Groups& gr, int64_t per) {
  const int64_t most = tile == T64 ? 1024 : 512;
  const int64_t units = ((gr.rows * total_comps(gr)) >> 7) + (int64_t)gr.blocks * gr.experts;   // (there are no more)
  Teams best{1, (int)(per < most ? per : most)};
  double used = -1;
  for (int64_t r = 1; r <= 4; ++r) {
    const int64_t team = (per + r - 1) / r;
    if (team > most) continue;
    const int64_t cuts = std::min(most / team, units);
    const double u = (double)(cuts * per) / (double)(r * most) - 0.02 * (double)r;
    if (u > used) used = u, best = {(int)cuts, (int)team};
  }
  return best;
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
  const bool fast = type != TACE_ROW_F64 && sum % 8 == 0 && n % 8 == 0 && row_aligned(x) && row_aligned(weight) && row_aligned(out);
  bool fits = true;
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    typedef row_sum_t<T> S;
    with_tile(std::is_same<T, double>::value ? T64 : rows_tile(gr, n, fast && sizeof(T) == 2), [&](auto wm, auto wn, auto fm, auto fn) {
      constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, FM = decltype(fm)::value, FN = decltype(fn)::value;
      constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
      const int64_t cols = (n + TN - 1) / TN, tiles = slots_of(gr, __builtin_ctz(TM)) * cols;
      if (!(fits = tiles <= MOST_WGS)) return;
      choose(transposed == 0, fast, [&](auto bt, auto quick) {
        constexpr bool BT = decltype(bt)::value, FAST = decltype(quick)::value;
        if constexpr (has_tile<T, FAST>(TM, TN))
          hipLaunchKernelGGL((k_expert_rows<T, BT, WM, WN, FM, FN, FAST>),
                             dim3(STREAMS<T, FAST> ? walkers(tiles, TM == 128 ? 512 : 1024) : grid_of(tiles)),
                             dim3(64 * WM * WN), 0, (hipStream_t)stream, (const T*)x, (const T*)weight, gr, wsize, sum, n,
                             (S)scale, (T*)out, (int)cols);
      });
    });
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
  if (experts == 0 || rows == 0) return 0;
  const int tile = weight_tile(type, gr, K, N);
  const int64_t per = tiles_of(tile, K, N), side = tile == T64 ? 64 : 128;
  const Teams teams = teams_of(tile, gr, per);
  return teams.cuts > 1 && may_be_cut(gr) ? 2 * per * teams.cuts * side * side * (type == TACE_ROW_F64 ? 8 : 4) : 0;
}

extern "C" int tace_expert_linear_grad(int type, const void* x, const void* g, const int32_t* rowptr, int64_t rows,
                                       int32_t experts, int32_t blocks, const int32_t* comps, int32_t K, int32_t N,
                                       double scale, void* dw, void* work, int64_t work_bytes, void* stream) {
  Groups gr;
  if (check_groups(rows, experts, blocks, comps, K, N, rowptr, &gr)) return -1;
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("expert_linear: unknown row type");
  if (experts == 0) return 0;
  if ((rows && (!x || !g)) || !dw) return tace_fail_msg("expert_linear: null argument");
  const int tile = weight_tile(type, gr, K, N);
  const int64_t per = tiles_of(tile, K, N);
  if ((int64_t)blocks * experts * per > MOST_WGS / 2) return tace_fail_msg("expert_linear: bad sizes");
  const Teams teams = teams_of(tile, gr, per);
  const bool joins = teams.cuts > 1 && may_be_cut(gr);
  if (joins && (!work || !row_aligned(work) ||
                work_bytes < tace_expert_linear_grad_work(type, rows, experts, blocks, comps, K, N)))
    return tace_fail_msg("expert_linear: the workspace is too small or not 16-byte aligned");
  const unsigned n = grid_of((int64_t)teams.cuts * teams.team);
  // workgroups of a tile's sums: one move a thread, fewer where there are many tiles (32 tiles of 128 x 128: 15.2 us with
  // 16, 19.6 with 8, 32.7 with 4; 1,024 tiles: 19.6 with 4, 30.7 with 8)
  int parts = tile == T64 ? 4 : 16;
  while (parts > 2 && parts * (int64_t)blocks * experts * per > 4096) parts /= 2;
  const hipStream_t st = (hipStream_t)stream;
  const bool fast = type != TACE_ROW_F64 && K % 8 == 0 && N % 8 == 0 && row_aligned(x) && row_aligned(g) && row_aligned(dw);
  row_dispatch(type, [&](auto zero) {
    typedef decltype(zero) T;
    typedef row_sum_t<T> S;
    with_tile(tile, [&](auto wm, auto wn, auto fm, auto fn) {
      constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, FM = decltype(fm)::value, FN = decltype(fn)::value;
      constexpr int TM = 16 * WM * FM, TN = 16 * WN * FN;
      if constexpr (TM == TN && (TM == 64 || (TM == 128 && !std::is_same<T, double>::value))) {
        const int cols = (N + TN - 1) / TN;
        choose(fast, true, [&](auto quick, auto) {
          hipLaunchKernelGGL((k_expert_weights<T, WM, WN, FM, FN, decltype(quick)::value>), dim3(n), dim3(64 * WM * WN), 0,
                             st, (const T*)x, (const T*)g, gr, K, N, (S)scale, (T*)dw, (S*)work, (int)per, cols, teams.cuts, teams.team);
        });
        if (joins)
          hipLaunchKernelGGL((k_expert_join<T, TM, TN>), dim3((unsigned)(parts * blocks * experts * per)), dim3(WG), 0, st,
                             (const S*)work, gr, K, N, (S)scale, (T*)dw, (int)per, cols, teams.cuts, parts);
      }
    });
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
      with_tile(rows_tile(gr, N, false), [&](auto wm, auto wn, auto fm, auto fn) {
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
