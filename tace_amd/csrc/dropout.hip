// Dropout whose mask comes from a counter and is made again by every pass that
// needs it, so no pass reads or writes one.
#include "row_types.h"

#include <type_traits>

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

// 8 draws a thread.  V: elements a move (1: any channels and alignment);
// V > 1 needs channels % 8 == 0, or one block of one component (flat).
template <typename T, int V>
__global__ __launch_bounds__(WG) void k_dropout(const T* __restrict__ x, const T* __restrict__ res, Draws dr,
                                                int64_t total, int64_t rows, int channels, Parts pt,
                                                row_sum_t<T> scale, T* __restrict__ out) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  const int64_t block = (int64_t)blockIdx.x * WG + threadIdx.x, i0 = block * 8;
  if (i0 >= total) return;
  const int64_t seed = dr.state ? dr.state[0] : dr.seed, offset = dr.state ? dr.state[1] : dr.offset;
  const unsigned keep = dr.keep8((unsigned)block, seed, offset);
  auto move = [&](int64_t at, unsigned bits) {   // V elements from `at`
    S a[V], r[V];
    row_widen<T, V>(*(const Vec*)(x + at), a);
    if (res) row_widen<T, V>(*(const Vec*)(res + at), r);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = (bits >> i) & 1 ? a[i] * scale : (S)0;
      if (res) a[i] += r[i];
    }
    *(Vec*)(out + at) = row_round<T, V>(a);
  };
  if constexpr (V > 1) {
    if (pt.count == 1 && pt.comps[0] == 1) {   // flat: the last thread may have fewer than 8
      if (i0 + 8 <= total) {
#pragma unroll
        for (int q = 0; q < 8; q += V) move(i0 + q, keep >> q);
      } else {
        for (int q = 0; i0 + q < total; ++q) {
          S a = (keep >> q) & 1 ? (S)x[i0 + q] * scale : (S)0;
          if (res) a += (S)res[i0 + q];
          out[i0 + q] = (T)a;
        }
      }
    } else {
      const int64_t rb = i0 / channels;
      const int c = (int)(i0 - rb * channels), b = (int)(rb % pt.count), d = pt.comps[b];
      const int64_t base = (rows * pt.before[b] + rb / pt.count * d) * channels + c;
      for (int m = 0; m < d; ++m)
#pragma unroll
        for (int q = 0; q < 8; q += V) move(base + (int64_t)m * channels + q, keep >> q);
    }
  } else {
    for (int q = 0; q < 8 && i0 + q < total; ++q) {
      const int64_t i = i0 + q, rb = i / channels;
      const int c = (int)(i - rb * channels), b = (int)(rb % pt.count), d = pt.comps[b];
      const int64_t base = (rows * pt.before[b] + rb / pt.count * d) * channels + c;
      for (int m = 0; m < d; ++m) move(base + (int64_t)m * channels, keep >> q);
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
  const bool vec = (flat || channels % 8 == 0) && row_aligned(x) && row_aligned(out) &&
                   (!residual || row_aligned(residual));
  const double scale = threshold == 65536 ? 0.0 : 65536.0 / (65536 - threshold);
  row_dispatch(type, [&](auto z) {
    typedef decltype(z) T;
    auto run = [&](auto vc) {
      hipLaunchKernelGGL((k_dropout<T, decltype(vc)::value>), dim3((unsigned)grid), dim3(WG), 0, (hipStream_t)stream,
                         (const T*)x, (const T*)residual, Draws{state, seed, offset, site, (unsigned)threshold}, total,
                         rows, channels, pt, (row_sum_t<T>)scale, (T*)out);
    };
    if (vec) run(std::integral_constant<int, 16 / sizeof(T)>());
    else run(std::integral_constant<int, 1>());
  });
  return tace_check_launch("tace_dropout");
}
