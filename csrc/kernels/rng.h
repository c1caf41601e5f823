// Counter-based random bits for dropout: Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw,
// "Parallel Random Numbers: As Easy as 1, 2, 3", SC11).
//
// A mask is a pure function of (seed, step, element index): element i takes the (i & 7)-th 16-bit
// piece of the 128 bits drawn at counter (i >> 3, step) under the key `seed`, so the backward pass,
// a replay and every kernel that fuses dropout draw the same mask again and none is ever stored.
// One draw serves 8 elements, i.e. one 16-byte bf16 vector.  Ten rounds are 20 32x32->64 multiplies:
// ~400 SIMD cycles a wave for 64 x 8 elements, about half of the time that HBM takes for their 32
// bytes (bf16 in and out), so the draw hides behind the memory traffic.
#pragma once
#include "common.h"

struct DropArgs {
  uint32_t thr;          // dropped when the 16-bit piece is below thr (0: keep all, 65536: drop all)
  float scale;           // 1 / keep probability
  uint64_t seed, step;
  const long* step_dev;  // device-resident step (captured graphs), overrides `step`
  uint64_t first;        // mask index of the tensor's first element
};
static inline DropArgs drop_args(int thr, float scale, long seed, long step, const void* step_dev, long first = 0) {
  return DropArgs{(uint32_t)thr, scale, (uint64_t)seed, (uint64_t)step, (const long*)step_dev, (uint64_t)first};
}
PTG_DEV uint64_t drop_step(const DropArgs& d) { return d.step_dev ? (uint64_t)*d.step_dev : d.step; }

PTG_DEV U4 philox(uint64_t ctr, uint64_t step, uint64_t seed) {
  uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  U4 o;
  o.x = c0; o.y = c1; o.z = c2; o.w = c3;
  return o;
}

// keep bits of 8 pieces: bit j = (piece j >= thr)
PTG_DEV uint32_t keep8(const U4& w, uint32_t thr) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t b = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b |= (uint32_t)((v[j] & 0xFFFFu) >= thr) << (2 * j);
    b |= (uint32_t)((v[j] >> 16) >= thr) << (2 * j + 1);
  }
  return b;
}
// The same as 8 conditions: each compares a half word in place and lands in a lane mask.
PTG_DEV void keep8(const U4& w, uint32_t thr, bool* k) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    k[2 * j] = (v[j] & 0xFFFFu) >= thr;
    k[2 * j + 1] = (v[j] >> 16) >= thr;
  }
}
// keep bits of the 8 elements from index i on; only an index that is no multiple of 8 needs the
// second draw
PTG_DEV uint32_t keep8_at(uint64_t i, uint64_t step, const DropArgs& d) {
  const uint32_t off = (uint32_t)i & 7u;
  uint32_t b = keep8(philox(i >> 3, step, d.seed), d.thr);
  if (off) b = ((b | (keep8(philox((i >> 3) + 1, step, d.seed), d.thr) << 8)) >> off) & 0xFFu;
  return b;
}
