// Counter-based draws for dropout: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011). A draw is a function of the seed, the offset, the site and the element's place alone, so the
// backward pass draws again what the forward pass drew and no mask is stored.
#pragma once

#include "bzpf_rows.h"

namespace bzpf {

struct Key {
  uint32_t k0, k1, o0, o1;
};
__device__ __forceinline__ Key drop_key(const Drop& d) {
  const uint64_t seed = (uint64_t)d.rng[0], off = (uint64_t)d.rng[1];
  return Key{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The four words of block n: counter = (n bits 0-31, n bits 32-47 | site << 16, offset), key = seed.
__device__ __forceinline__ u4 draw_block(uint64_t n, uint32_t site, Key k) {
  uint32_t c0 = (uint32_t)n, c1 = (uint32_t)(n >> 32) | site << 16, c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k.k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k.k1;
    c3 = (uint32_t)p0;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return u4{c0, c1, c2, c3};
}

// The draw that a whole row r (of I * J rows a slice) shares: one for each row i or column j of the slice.
__device__ __forceinline__ uint32_t draw_shared(const Drop& d, Key k, int64_t r) {
  int64_t g;
  if (((uint64_t)r | (uint64_t)d.I * (uint64_t)d.J) >> 32 == 0) {  // the 32-bit division is the shorter one
    const uint32_t q = (uint32_t)r, J = (uint32_t)d.J;
    g = d.mode == DROP_ROW ? q / J : (q / ((uint32_t)d.I * J)) * J + q % J;
  } else {
    g = d.mode == DROP_ROW ? r / d.J : (r / (d.I * d.J)) * d.J + r % d.J;
  }
  const u4 w = draw_block((uint64_t)g >> 2, d.site, k);
  const uint32_t a = g & 1 ? w[1] : w[0], b = g & 1 ? w[3] : w[2];
  return g & 2 ? b : a;
}

// Applies the element draws to the eight columns v of a row, the first of them column `s` (0 to 3) of block n. Blocks
// hold four columns counted from the row's start, so that s is 0 but for a chunk moved back from the row's end, which
// then meets three blocks.
__device__ __forceinline__ f8 drop_elements(const Drop& d, Key k, uint64_t n, int s, f8 v) {
  const u4 a = draw_block(n, d.site, k), b = draw_block(n + 1, d.site, k);
  uint32_t w[11] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], 0, 0, 0};
  if (s) {
    const u4 c = draw_block(n + 2, d.site, k);
    w[8] = c[0], w[9] = c[1], w[10] = c[2];
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = s == 1 ? w[e + 1] : s == 2 ? w[e + 2] : w[e + 3];
  }
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = w[e] <= d.last ? 0.f : v[e] * d.scale;
  return v;
}

}  // namespace bzpf
