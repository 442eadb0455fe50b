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

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one v_bitop3_b32 (truth table of a ^ b ^ c)
}

// The four words of block n: counter = (n bits 0-31, n bits 32-47 | site << 16, offset), key = seed.
__device__ __forceinline__ u4 draw_block(uint64_t n, uint32_t site, Key k) {
  uint32_t c0 = (uint32_t)n, c1 = (uint32_t)(n >> 32) | site << 16, c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(p1 >> 32), c1, k.k0);
    c1 = (uint32_t)p1;
    c2 = xor3((uint32_t)(p0 >> 32), c3, k.k1);
    c3 = (uint32_t)p0;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return u4{c0, c1, c2, c3};
}

// Whether the draw that a whole row r (of I * J rows a slice; fewer than 2^32 in all) shares drops it: one draw for each
// row i or column j of the slice.
__device__ __forceinline__ bool drops_row(const Drop& d, Key k, int64_t r) {
  const uint32_t row = (uint32_t)r, J = (uint32_t)d.J, q = row / J;
  const uint32_t g = d.mode == DROP_ROW ? q : q / (uint32_t)d.I * J + (row - q * J);
  const u4 w = draw_block(g >> 2, d.site, k);
  const uint32_t a = g & 1 ? w[1] : w[0], b = g & 1 ? w[3] : w[2];
  return (g & 2 ? b : a) <= d.last;
}

// The element draws of VE columns of a row as bits (bit e set: column e is kept), the first of them column `s` (0 to 3) of
// block n. Blocks hold four columns counted from the row's start, so that s is 0 but for a chunk moved back from the row's
// end, which then meets one block more.
template <int VE>
__device__ __forceinline__ uint32_t kept(const Drop& d, Key k, uint64_t n, int s) {
  const auto block = [&](int j) {
    const u4 w = draw_block(n + j, d.site, k);
    return (w[0] > d.last ? 1u : 0u) | (w[1] > d.last ? 2u : 0u) | (w[2] > d.last ? 4u : 0u) | (w[3] > d.last ? 8u : 0u);
  };
  uint32_t bits = block(0);
  if (VE == 8) bits |= block(1) << 4;
  if (s) bits = (bits | block(VE / 4) << VE) >> s;
  return bits;
}
// v[e] / (1 - p) where bit `first` + e is set, else 0 (whatever v holds).
template <int VE>
__device__ __forceinline__ fv<VE> keep(const Drop& d, uint32_t bits, int first, fv<VE> v) {
#pragma unroll
  for (int e = 0; e < VE; e++) v[e] = bits >> (first + e) & 1 ? v[e] * d.scale : 0.f;
  return v;
}

}  // namespace bzpf
