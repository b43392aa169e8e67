// Dropout whose mask comes from a counter and is made again by every pass that
// needs it, so no pass reads or writes one.
#include "row_types.h"

namespace {

constexpr int WG = 256;

// Philox-4x32 with 10 rounds (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E.
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC11): four words of
// counter c under key k.
__device__ __forceinline__ void philox(unsigned* c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c[0] * 0xD2511F53u, b = (unsigned long long)c[2] * 0xCD9E8D57u;
    c[0] = (unsigned)(b >> 32) ^ c[1] ^ k0;
    c[1] = (unsigned)b;
    c[2] = (unsigned)(a >> 32) ^ c[3] ^ k1;
    c[3] = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

struct Draws {
  const int64_t* state;   // device (seed, offset), or null
  int64_t seed, offset;
  unsigned site, threshold;

  // which of draws 8 block .. 8 block + 7 keep their elements, as bits
  __device__ __forceinline__ unsigned keep8(unsigned block, int64_t s, int64_t o) const {
    unsigned c[4] = {block, site, (unsigned)o, (unsigned)((unsigned long long)o >> 32)};
    philox(c, (unsigned)s, (unsigned)((unsigned long long)s >> 32));
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m |= ((c[i] & 0xffffu) >= threshold ? 1u : 0u) << (2 * i);
      m |= ((c[i] >> 16) >= threshold ? 1u : 0u) << (2 * i + 1);
    }
    return m;
  }
};

struct Parts {
  int count, comps[TACE_ROW_MAX_BLOCKS];
  int before[TACE_ROW_MAX_BLOCKS];   // components of the blocks before
};

// A wavefront makes 512 draws, 8 a lane, and then moves the 512 elements (of
// each component) in the order of memory: of its q-th V each, a lane takes the
// ones that lane q 8 V + lane V / 8 drew for.  Needs channels % V == 0, or one
// block of one component (flat: the last V elements may be fewer).  Bound by
// HBM: the ten rounds are 20 wide multiplications and 34 exclusive ors for 8
// elements, and twice that, for draws of 32 bits, took the same time (81 us for
// 117 M bfloat16): 16 bits are enough for a probability.  us (TB/s): 25 M
// float32 in degrees 0 .. 3 38 (5.3), with a residual 57 (5.3); 117 M bfloat16 in
// degrees 0 .. 2 81 (5.7).  With lanes that kept their own 8 elements (two moves
// of every other 16 bytes, one component after the other) 51, 74 and 89; with
// stores that stay in the caches 40, 59 and 83.
template <typename T, int V>
__global__ __launch_bounds__(WG) void k_dropout_vec(const T* __restrict__ x, const T* __restrict__ res, Draws dr,
                                                    int64_t total, int64_t rows, int channels, Parts pt, bool flat,
                                                    row_sum_t<T> scale, T* __restrict__ out) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  constexpr int Q = 8 / V, U = 4;
  const int lane = (int)threadIdx.x & 63;
  const int64_t w0 = ((int64_t)blockIdx.x * WG + threadIdx.x - lane) * 8;   // the wavefront's first draw
  if (w0 >= total) return;
  const int64_t seed = dr.state ? dr.state[0] : dr.seed, offset = dr.state ? dr.state[1] : dr.offset;
  const unsigned keep = dr.keep8((unsigned)(w0 / 8) + lane, seed, offset);
  auto drop = [&](const Vec& v, const Vec& r, unsigned bits) {
    S a[V], b[V];
    row_widen<T, V>(v, a);
    if (res) row_widen<T, V>(r, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = (bits >> i) & 1 ? a[i] * scale : (S)0;
      if (res) a[i] += b[i];
    }
    return row_round<T, V>(a);
  };
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int e = (q * 64 + lane) * V;   // of the wavefront's draws
    const unsigned bits = __shfl(keep, e / 8, 64) >> (e % 8);
    const int64_t i = w0 + e;
    if (i >= total) continue;
    if (flat) {
      if (i + V <= total) {
        Vec r;
        if (res) r = *(const Vec*)(res + i);
        __builtin_nontemporal_store(drop(*(const Vec*)(x + i), r, bits), (Vec*)(out + i));
      } else {
        for (int k = 0; i + k < total; ++k) {
          S a = (bits >> k) & 1 ? (S)x[i + k] * scale : (S)0;
          if (res) a += (S)res[i + k];
          out[i + k] = (T)a;
        }
      }
    } else {
      const unsigned rb = (unsigned)(i / V) / (unsigned)(channels / V);   // (row, block)
      const int c = (int)(i - (int64_t)rb * channels), b = (int)(rb % (unsigned)pt.count), d = pt.comps[b];
      const int64_t base = (rows * pt.before[b] + (int64_t)(rb / (unsigned)pt.count) * d) * channels + c;
      for (int m = 0; m < d; m += U) {
        Vec v[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t at = base + (int64_t)min(m + u, d - 1) * channels;
          v[u] = *(const Vec*)(x + at);
          if (res) r[u] = *(const Vec*)(res + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (m + u < d)
            __builtin_nontemporal_store(drop(v[u], r[u], bits), (Vec*)(out + base + (int64_t)(m + u) * channels));
      }
    }
  }
}

// any channels and alignment, 8 draws a thread.  Bound by its loads and stores of
// single elements: a thread's 8 draws are neighbours, so a wavefront's addresses
// lie 8 elements apart.  12,288 rows of 99 channels of float32 in degrees 0 .. 3
// 222 us, of 100 (the kernel above) 33.
template <typename T>
__global__ __launch_bounds__(WG) void k_dropout_any(const T* __restrict__ x, const T* __restrict__ res, Draws dr,
                                                    int64_t total, int64_t rows, int channels, Parts pt,
                                                    row_sum_t<T> scale, T* __restrict__ out) {
  typedef row_sum_t<T> S;
  const int64_t block = (int64_t)blockIdx.x * WG + threadIdx.x;
  if (block * 8 >= total) return;
  const int64_t seed = dr.state ? dr.state[0] : dr.seed, offset = dr.state ? dr.state[1] : dr.offset;
  const unsigned keep = dr.keep8((unsigned)block, seed, offset);
  for (int q = 0; q < 8 && block * 8 + q < total; ++q) {
    const int64_t i = block * 8 + q, rb = i / channels;
    const int c = (int)(i - rb * channels), b = (int)(rb % pt.count), d = pt.comps[b];
    const int64_t base = (rows * pt.before[b] + rb / pt.count * d) * channels + c;
    for (int m = 0; m < d; ++m) {
      const int64_t at = base + (int64_t)m * channels;
      S a = (keep >> q) & 1 ? (S)x[at] * scale : (S)0;
      if (res) a += (S)res[at];
      out[at] = (T)a;
    }
  }
}

}  // namespace

extern "C" int tace_dropout(int type, const void* x, const void* residual, const int64_t* state, int64_t seed,
                            int64_t offset, uint32_t site, int32_t threshold, int64_t rows, int32_t channels,
                            int32_t blocks, const int32_t* comps, void* out, void* stream) {
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("tace_dropout: unknown row type");
  if (threshold < 0 || threshold > 65536) return tace_fail_msg("tace_dropout: threshold outside 0 .. 65536");
  if (rows < 0 || channels < 1 || blocks < 1 || blocks > TACE_ROW_MAX_BLOCKS || !comps)
    return tace_fail_msg("tace_dropout: bad sizes");
  Parts pt = {};
  pt.count = blocks;
  int before = 0;
  for (int b = 0; b < blocks; ++b) {
    if (comps[b] < 1 || comps[b] > 1024) return tace_fail_msg("tace_dropout: bad number of components");
    pt.comps[b] = comps[b];
    pt.before[b] = before;
    before += comps[b];
  }
  if (rows == 0) return 0;
  // a block of draws is a 32-bit counter word, and a launch holds less than 2^32 threads
  const int64_t per_row = (int64_t)channels * blocks;
  if (rows > ((int64_t)1 << 34) / per_row) return tace_fail_msg("tace_dropout: over 2^34 draws");
  if (!x || !out) return tace_fail_msg("tace_dropout: null pointer");
  const int64_t total = rows * per_row, grid = (total + 8 * WG - 1) / (8 * WG);
  const bool flat = blocks == 1 && comps[0] == 1;
  const double scale = threshold == 65536 ? 0.0 : 65536.0 / (65536 - threshold);
  row_dispatch(type, [&](auto z) {
    typedef decltype(z) T;
    const Draws dr{state, seed, offset, site, (unsigned)threshold};
    row_moves<T>(
        [&](int v, int bytes) {
          const uintptr_t at = (uintptr_t)x | (uintptr_t)out | (uintptr_t)residual;
          return (flat || channels % v == 0) && at % bytes == 0 && total / v <= UINT32_MAX;
        },
        [&](auto vc) {
          constexpr int V = decltype(vc)::value;
          if constexpr (V > 1)
            hipLaunchKernelGGL((k_dropout_vec<T, V>), dim3((unsigned)grid), dim3(WG), 0, (hipStream_t)stream,
                               (const T*)x, (const T*)residual, dr, total, rows, channels, pt, flat,
                               (row_sum_t<T>)scale, (T*)out);
          else
            hipLaunchKernelGGL((k_dropout_any<T>), dim3((unsigned)grid), dim3(WG), 0, (hipStream_t)stream, (const T*)x,
                               (const T*)residual, dr, total, rows, channels, pt, (row_sum_t<T>)scale, (T*)out);
        });
  });
  return tace_check_launch("tace_dropout");
}
