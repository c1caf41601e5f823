// Dropout with a mask that is drawn where it is used and never stored (rng.h).
//
//   y[i] = keep(i) ? x[i] * scale : 0        forward; the same map on dy is the backward pass
//
// A dropped element is 0 whatever x holds (NaN and infinities included).  The mask may be shared over
// one run of axes: with the tensor seen as [outer][mid][inner], element (o, m, i) takes mask entry
// o * inner + i (Keras noise_shape: [N, 1, 1, C] drops whole channels, [N, 1, 1, 1] whole samples).
//
// Bound by HBM: x in, y out, nothing else (256 x 128 x 160 x 8 bf16: 32 us, 5.2 TB/s).  Each thread owns groups of
// 8 consecutive elements, so a bf16 group is one 16-byte load, one draw and one 16-byte store.
#include "rng.h"

namespace {

template <typename T> struct Vec8;
template <> struct Vec8<bf16_t> {
  U4 v;
  PTG_DEV void load(const bf16_t* p) { v = *(const U4*)p; }
  PTG_DEV void apply(uint32_t keep, float s) {
    float f[8];
    unpack8(v, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (keep >> j) & 1u ? f[j] * s : 0.f;
    v = pack8(f);
  }
  PTG_DEV void store(bf16_t* p) const { *(U4*)p = v; }
};
template <> struct Vec8<float> {
  float4 a, b;
  PTG_DEV void load(const float* p) { a = *(const float4*)p; b = *(const float4*)(p + 4); }
  PTG_DEV void apply(uint32_t keep, float s) {
    float* f = &a.x;
    float* g = &b.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = (keep >> j) & 1u ? f[j] * s : 0.f;
      g[j] = (keep >> (j + 4)) & 1u ? g[j] * s : 0.f;
    }
  }
  PTG_DEV void store(float* p) const { *(float4*)p = a; *(float4*)(p + 4) = b; }
};
PTG_DEV float ldf(const bf16_t* p) { return bf2f(*p); }
PTG_DEV float ldf(const float* p) { return *p; }
PTG_DEV void stf(bf16_t* p, float v) { *p = f2bf(v); }
PTG_DEV void stf(float* p, float v) { *p = v; }

}  // namespace

// One mask bit per element.  `vec`: both pointers are 16-byte aligned; otherwise, and for the last
// n % 8 elements, the group goes element by element.
template <typename T>
__global__ __launch_bounds__(256) void dropout_k(const T* x, T* y, long n, int vec, DropArgs d) {
  const uint64_t step = drop_step(d);
  const long n8 = (n + 7) >> 3, stride = (long)gridDim.x * 256;
  for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < n8; g += stride) {
    const long i = g * 8;
    if (vec && i + 8 <= n) {
      Vec8<T> v;
      v.load(x + i);
      v.apply(keep8(philox((uint64_t)g, step, d.seed), d.thr), d.scale);
      v.store(y + i);
    } else {
      const uint32_t keep = keep8(philox((uint64_t)g, step, d.seed), d.thr);
      const int m = (int)min(8L, n - i);
      for (int j = 0; j < m; ++j) stf(y + i + j, (keep >> j) & 1u ? ldf(x + i + j) * d.scale : 0.f);
    }
  }
}

// Mask shared over `mid`.  With inner % 8 == 0 a group's 8 mask entries are one aligned draw; otherwise
// the entries are walked one by one, with loads and stores of one value, and a draw is made where the 8-entry block
// changes.  256 x 64 x 80 x 16 bf16 by channel: 15.7 us a pass, 5.3 TB/s, the vector pipes 90 % busy (two 64-bit
// divisions a group); 256 x 160 x 160 x 3 by channel: 44 us bf16 (1.8 TB/s), 104 us fp32.
template <typename T>
__global__ __launch_bounds__(256) void dropout_shared_k(const T* x, T* y, long n, long mid, long inner, int vec,
                                                        DropArgs d) {
  const uint64_t step = drop_step(d);
  const long n8 = (n + 7) >> 3, stride = (long)gridDim.x * 256, plane = mid * inner;
  for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < n8; g += stride) {
    const long i = g * 8;
    long o = i / plane;
    long c = (i - o * plane) % inner;
    if (vec && inner % 8 == 0) {  // then n % 8 == 0 as well: every group is whole
      Vec8<T> v;
      v.load(x + i);
      v.apply(keep8(philox((uint64_t)(o * inner + c) >> 3, step, d.seed), d.thr), d.scale);
      v.store(y + i);
      continue;
    }
    const int m = (int)min(8L, n - i);
    long left = plane - (i - o * plane);  // elements of this o from i on
    uint64_t blk = ~0ull;
    uint32_t keep = 0;
    for (int j = 0; j < m; ++j) {
      const uint64_t e = (uint64_t)(o * inner + c);
      if (e >> 3 != blk) {
        blk = e >> 3;
        keep = keep8(philox(blk, step, d.seed), d.thr);
      }
      stf(y + i + j, (keep >> (e & 7)) & 1u ? ldf(x + i + j) * d.scale : 0.f);
      if (++c == inner) c = 0;
      if (--left == 0) { ++o; c = 0; left = plane; }
    }
  }
}

// step += 1 (one thread): the next training pass draws another mask, captured graphs included
__global__ void drop_advance_k(long* step) { *step += 1; }

extern "C" {

// Arguments, 64 bits each (one block costs the host less than as many arguments)
struct DropCall {
  const void* x;
  void* y;
  const void* step_dev;
  int64_t n, f32, thr, seed, step, mid, inner;
  double scale;
};
int ptg_dropout(const void* call, hipStream_t stream) {
  const DropCall& c = *(const DropCall*)call;
  const void* x = c.x;
  void* y = c.y;
  const long n = c.n, mid = c.mid, inner = c.inner;
  const bool f32 = c.f32;
  if (n <= 0) return 0;
  const DropArgs d = drop_args((int)c.thr, (float)c.scale, c.seed, c.step, c.step_dev);
  const int vec = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
  const long n8 = (n + 7) / 8;
  const int grid = (int)((n8 + 255) / 256 < 4096 ? (n8 + 255) / 256 : 4096);
  if (mid <= 1) {
    if (f32) dropout_k<float><<<grid, 256, 0, stream>>>((const float*)x, (float*)y, n, vec, d);
    else dropout_k<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)x, (bf16_t*)y, n, vec, d);
  } else {
    if (f32) dropout_shared_k<float><<<grid, 256, 0, stream>>>((const float*)x, (float*)y, n, mid, inner, vec, d);
    else dropout_shared_k<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)x, (bf16_t*)y, n, mid, inner, vec, d);
  }
  PTG_RETURN_LAUNCH();
}

int ptg_drop_advance(void* step, hipStream_t stream) {
  drop_advance_k<<<1, 1, 0, stream>>>((long*)step);
  PTG_RETURN_LAUNCH();
}

}  // extern "C"
