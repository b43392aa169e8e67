#pragma once
#include <hip/hip_runtime.h>

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
