// Dense products with 4-bit weights: y[m][n] = act(sum_g s[n][g] * sum_{k in g} (q[n][k] - z[n][g]) * x[m][k] + b[n])
//
// q in 0..15, a bf16 scale and a zero point (8 where none is given) for every group of 32, 64 or 128
// inputs of an output; x and y bf16 (y also fp32), sums fp32.
//
// Layout.  Weights are stored in tiles of 16 outputs x 128 inputs, 1 KB each, [N/16][K/128][64 lanes][16
// bytes], so a wave streams contiguous memory and each lane's dword i is its operand of the i-th
// 16x16x32 MFMA: lane l holds output l & 15, inputs i*32 + (l >> 4)*8 + 0..7.  In a dword, input 2s sits
// in nibble s and input 2s + 1 in nibble s + 4, all rotated left by 3 bits.  A nibble u at bits 3..6 of a
// half word under the bits of 16.0 is the bf16 number 16 + u exactly (one mantissa step there is 1/8),
// so two weights take one shift and one and-or and no conversion.
//
// The products run on 16 + u; acc starts from MFMAs with -(16 + z) in place of the weights, which leaves
// sum (u - z) x.  Both products are exact in fp32, and the offset costs at most (16 + 15) / |u - z| of an
// fp32 rounding.  Scales multiply the fp32 sum of a group, never a weight.
#include "common.h"

namespace {

constexpr int QT_K = 128;  // inputs of a weight tile

PTG_DEV f32x4_t mfma32(const U4& a, const U4& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}
// 8 weights of a dword as bf16 16 + u
PTG_DEV U4 dec8(uint32_t w) {
  constexpr uint32_t M = 0x00780078u, E = 0x41804180u;
  U4 o;
  o.x = (w & M) | E;
  o.y = ((w >> 4) & M) | E;
  o.z = ((w >> 8) & M) | E;
  o.w = (__builtin_amdgcn_alignbit(w, w, 12) & M) | E;
  return o;
}

}  // namespace

// One workgroup: 16 outputs, 16 * MT rows, one of the K ranges of the split.  Its 4 waves take the
// tiles of the range in turn and are joined in LDS.  part == nullptr: the range is all of K and the
// workgroup finishes y itself; otherwise it leaves fp32 sums in part[split][M][N].
template <int MT, int GS, bool F32>
__global__ __launch_bounds__(256) void int4_mm_k(const bf16_t* __restrict__ x, const uint8_t* __restrict__ w,
                                                 const bf16_t* __restrict__ scale, const uint8_t* __restrict__ zero,
                                                 const float* __restrict__ bias, void* __restrict__ y,
                                                 float* __restrict__ part, int M, int N, int K, int kt, int act) {
  __shared__ float red[4][MT * 4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, q = lane >> 4;
  const int nt = blockIdx.x, m0 = blockIdx.y * 16 * MT, splits = gridDim.z, sp = blockIdx.z;
  const int t0 = (int)((long)kt * sp / splits), t1 = (int)((long)kt * (sp + 1) / splits);
  constexpr int NG = 4 / GS;  // groups of a tile
  f32x4_t acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int t = t0 + wave; t < t1; t += 4) {
    const long tile = (long)nt * kt + t;
    const U4 wv = *(const U4*)(w + tile * 1024 + lane * 16);
    const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const long si = (tile * NG + g) * 16 + n16;
      const float s = bf2f(scale[si]);
      const float zf = -16.f - (zero ? (float)zero[si] : 8.f);
      const uint32_t zz = (__float_as_uint(zf) >> 16) * 0x10001u;
      U4 zc;
      zc.x = zz; zc.y = zz; zc.z = zz; zc.w = zz;
      f32x4_t d[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) d[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < GS; ++j) {
        const int k = t * QT_K + (g * GS + j) * 32 + q * 8;
        const U4 b = dec8(ww[g * GS + j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int m = m0 + i * 16 + n16;
          U4 a = zero4();
          if (m < M && k < K) __builtin_memcpy(&a, x + (long)m * K + k, 16);
          d[i] = mfma32(a, zc, d[i]);
          d[i] = mfma32(a, b, d[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] += d[i] * s;
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][i * 4 + r][lane] = acc[i][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 4 * 64; e += 256) {
    const int v = e >> 6, l = e & 63, n = nt * 16 + (l & 15), m = m0 + (v >> 2) * 16 + (l >> 4) * 4 + (v & 3);
    if (m >= M || n >= N) continue;
    float s = red[0][v][l] + red[1][v][l] + red[2][v][l] + red[3][v][l];
    const long o = (long)m * N + n;
    if (part) {
      part[(long)sp * M * N + o] = s;
      continue;
    }
    if (bias) s += bias[n];
    if (act) s = fmaxf(s, 0.f);
    if (F32) ((float*)y)[o] = s;
    else ((bf16_t*)y)[o] = f2bf(s);
  }
}

// y = act(sum of the splits + bias)
template <bool F32>
__global__ __launch_bounds__(256) void int4_join_k(const float* __restrict__ part, const float* __restrict__ bias,
                                                   void* __restrict__ y, long total, int N, int splits, int act) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int k = 0; k < splits; ++k) s += part[(long)k * total + i];
  if (bias) s += bias[i % N];
  if (act) s = fmaxf(s, 0.f);
  if (F32) ((float*)y)[i] = s;
  else ((bf16_t*)y)[i] = f2bf(s);
}

namespace {
struct Plan4 { int mt, mb, splits; };
Plan4 plan4(int M, int N, int K) {
  Plan4 p;
  p.mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  p.mb = (M + 16 * p.mt - 1) / (16 * p.mt);
  const long wgs = (long)((N + 15) / 16) * p.mb, kt = (K + QT_K - 1) / QT_K;
  long s = (1024 + wgs - 1) / wgs;  // about 4 workgroups a CU
  if (s > kt / 8) s = kt / 8;       // but at least two tiles a wave
  p.splits = s < 1 ? 1 : (int)s;
  return p;
}
template <int MT, int GS>
void go4(const Plan4& p, const bf16_t* x, const uint8_t* w, const bf16_t* s, const uint8_t* z, const float* b, void* y,
         float* part, int M, int N, int K, int act, int f32, hipStream_t st) {
  const int kt = (K + QT_K - 1) / QT_K;
  const dim3 grid((N + 15) / 16, p.mb, p.splits);
  if (f32) int4_mm_k<MT, GS, true><<<grid, 256, 0, st>>>(x, w, s, z, b, y, part, M, N, K, kt, act);
  else int4_mm_k<MT, GS, false><<<grid, 256, 0, st>>>(x, w, s, z, b, y, part, M, N, K, kt, act);
}
template <int MT>
void go4g(int gs, const Plan4& p, const bf16_t* x, const uint8_t* w, const bf16_t* s, const uint8_t* z,
          const float* b, void* y, float* part, int M, int N, int K, int act, int f32, hipStream_t st) {
  if (gs == 1) go4<MT, 1>(p, x, w, s, z, b, y, part, M, N, K, act, f32, st);
  else if (gs == 2) go4<MT, 2>(p, x, w, s, z, b, y, part, M, N, K, act, f32, st);
  else go4<MT, 4>(p, x, w, s, z, b, y, part, M, N, K, act, f32, st);
}
}  // namespace

extern "C" {

// *floats: workspace of a product of M rows (0 where none is needed)
int ptg_int4_ws(int M, int N, int K, void* floats) {
  const Plan4 p = M > 0 ? plan4(M, N, K) : Plan4{1, 1, 1};
  *(long*)floats = p.splits > 1 ? (long)p.splits * M * N : 0;
  return 0;
}

// w, scale, zero: tile layout; group 32, 64 or 128; zero null: 8 everywhere; act 0 linear, 1 ReLU
int ptg_int4_dense(const void* x, const void* w, const void* scale, const void* zero, const void* bias, void* y,
                   void* ws, int M, int N, int K, int group, int act, int f32, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if ((group != 32 && group != 64 && group != 128) || K < group || K % group) return (int)hipErrorInvalidValue;
  const Plan4 p = plan4(M, N, K);
  float* part = p.splits > 1 ? (float*)ws : nullptr;
  const bf16_t* xs = (const bf16_t*)x;
  const bf16_t* sc = (const bf16_t*)scale;
  const int gs = group / 32;
  if (p.mt == 1)
    go4g<1>(gs, p, xs, (const uint8_t*)w, sc, (const uint8_t*)zero, (const float*)bias, y, part, M, N, K, act, f32, stream);
  else if (p.mt == 2)
    go4g<2>(gs, p, xs, (const uint8_t*)w, sc, (const uint8_t*)zero, (const float*)bias, y, part, M, N, K, act, f32, stream);
  else
    go4g<4>(gs, p, xs, (const uint8_t*)w, sc, (const uint8_t*)zero, (const float*)bias, y, part, M, N, K, act, f32, stream);
  if (part) {
    const long total = (long)M * N;
    const int blocks = (int)((total + 255) / 256);
    if (f32) int4_join_k<true><<<blocks, 256, 0, stream>>>(part, (const float*)bias, y, total, N, p.splits, act);
    else int4_join_k<false><<<blocks, 256, 0, stream>>>(part, (const float*)bias, y, total, N, p.splits, act);
  }
  PTG_RETURN_LAUNCH();
}

}  // extern "C"
