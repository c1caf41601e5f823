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

// A wave computes 16 * MT rows x 16 * NT outputs over its share of K; the NW waves of a workgroup take the
// tiles of the workgroup's K range in turn and are joined in LDS in a fixed order.  One wave is one MFMA
// chain a product tile: sum (16 + u) x on top of -(16 + z) * sum x, the latter from one MFMA with ones for
// every 32 inputs that all NT tiles share.  The next tile's weights, scales and inputs are loaded before
// the current tile is worked on.  part == nullptr: the range is all of K and the workgroup finishes y
// itself; otherwise it leaves fp32 sums in part[split][M][N].
template <int GS>
struct Group {  // of a tile: 4 / GS groups
  static constexpr int NG = 4 / GS;
  bf16_t s[NG];
  uint8_t z[NG];
};
template <int MT, int NT, int NW, int GS, bool HASZ>
__global__ __launch_bounds__(NW * 64) void int4_mm_k(const bf16_t* __restrict__ x, const uint8_t* __restrict__ w,
                                                     const bf16_t* __restrict__ scale,
                                                     const uint8_t* __restrict__ zero, const float* __restrict__ bias,
                                                     void* __restrict__ y, float* __restrict__ part, int M, int N,
                                                     int K, int kt, int act, int f32) {
  constexpr int NG = 4 / GS, R = MT * NT * 4;
  constexpr bool FLAT = R * NW <= 128;  // every wave's sums in LDS at once, else pairwise
  __shared__ float red[(FLAT ? NW : NW / 2) * R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, q = lane >> 4;
  const int sp = blockIdx.x, splits = gridDim.x, nb = blockIdx.y * NT, m0 = blockIdx.z * 16 * MT;
  const int ntiles = (N + 15) / 16;
  const int t0 = (int)((long)kt * sp / splits), t1 = (int)((long)kt * (sp + 1) / splits);
  const bf16_t* xr[MT];
  bool mon[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + i * 16 + n16;
    mon[i] = m < M;
    xr[i] = x + (long)(mon[i] ? m : 0) * K + q * 8;
  }
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[i][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  U4 wn[NT], xn[MT][4];
  Group<GS> gn[NT];
  auto fetch = [&](int t) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int nt = nb + n < ntiles ? nb + n : ntiles - 1;  // a tile that is not there: any, not stored
      const long tile = (long)nt * kt + t;
      wn[n] = *(const U4*)(w + tile * 1024 + lane * 16);
      __builtin_memcpy(gn[n].s, scale + (tile * 16 + n16) * NG, 2 * NG);
      if (HASZ) __builtin_memcpy(gn[n].z, zero + (tile * 16 + n16) * NG, NG);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xn[i][j] = zero4();
        if (mon[i] && t * QT_K + j * 32 + q * 8 < K) __builtin_memcpy(&xn[i][j], xr[i] + t * QT_K + j * 32, 16);
      }
  };
  U4 ones;
  ones.x = 0x3F803F80u; ones.y = ones.x; ones.z = ones.x; ones.w = ones.x;
  int t = t0 + wave;
  if (t < t1) fetch(t);
  while (t < t1) {
    U4 wc[NT], xc[MT][4];
    Group<GS> gc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) { wc[n] = wn[n]; gc[n] = gn[n]; }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) xc[i][j] = xn[i][j];
    t += NW;
    if (t < t1) fetch(t);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t xs[MT];  // sum of the group's inputs, the same in every column
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xs[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) xs[i] = mfma32(xc[i][g * GS + j], ones, xs[i]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t ww[4] = {wc[n].x, wc[n].y, wc[n].z, wc[n].w};
        const float s = bf2f(gc[n].s[g]);
        const float zf = HASZ ? -16.f - (float)gc[n].z[g] : -24.f;
        U4 b[GS];
#pragma unroll
        for (int j = 0; j < GS; ++j) b[j] = dec8(ww[g * GS + j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          f32x4_t d = xs[i] * zf;
#pragma unroll
          for (int j = 0; j < GS; ++j) d = mfma32(xc[i][g * GS + j], b[j], d);
          acc[i][n] += d * s;
        }
      }
    }
  }
  auto put = [&](int slot) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[slot * R + (i * NT + n) * 4 + r][lane] = acc[i][n][r];
  };
  auto out = [&](int v, int l, float s) {  // register v of lane l
    const int i = v / (NT * 4), n = (v / 4) % NT, r = v & 3;
    const int col = (nb + n) * 16 + (l & 15), m = m0 + i * 16 + (l >> 4) * 4 + r;
    if (m >= M || col >= N) return;
    const long o = (long)m * N + col;
    if (part) {
      part[(long)sp * M * N + o] = s;
      return;
    }
    if (bias) s += bias[col];
    if (act) s = fmaxf(s, 0.f);
    if (f32) ((float*)y)[o] = s;
    else ((bf16_t*)y)[o] = f2bf(s);
  };
  if (FLAT) {
    put(wave);
    __syncthreads();
    for (int e = threadIdx.x; e < R * 64; e += NW * 64) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) s += red[k * R + (e >> 6)][e & 63];
      out(e >> 6, e & 63, s);
    }
  } else {
#pragma unroll
    for (int h = NW / 2; h > 0; h >>= 1) {
      if (wave >= h && wave < 2 * h) put(wave - h);
      __syncthreads();
      if (wave < h) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][n][r] += red[wave * R + (i * NT + n) * 4 + r][lane];
      }
      __syncthreads();
    }
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) out((i * NT + n) * 4 + r, lane, acc[i][n][r]);
    }
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
// Workgroups wanted: one a CU.  Two a CU measured 104.7 against 94.1 us on 256 x 2048 x 20480 and 18.4
// against 14.2 us on 16 x 8192 x 8192 (more partial sums to write and join); 1 x 2048 x 20480 is the same.
constexpr int Q_WGS = 256;
struct Plan4 { int mt, nt, mb, nb, splits; };
Plan4 plan4(int M, int N, int K) {
  Plan4 p;
  p.mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  p.nt = M <= 8 ? 1 : M <= 32 ? 2 : 4;
  p.mb = (M + 16 * p.mt - 1) / (16 * p.mt);
  p.nb = (N + 16 * p.nt - 1) / (16 * p.nt);
  const long wgs = (long)p.nb * p.mb, kt = (K + QT_K - 1) / QT_K;
  const int nw = p.mt == 1 ? 16 : 8;
  long s = (Q_WGS + wgs - 1) / wgs;
  if (s > kt / (2 * nw)) s = kt / (2 * nw);  // at least two tiles a wave
  p.splits = s < 1 ? 1 : (int)s;
  return p;
}
struct Args4 {
  const bf16_t* x;
  const uint8_t* w;
  const bf16_t* s;
  const uint8_t* z;
  const float* b;
  void* y;
  float* part;
  int M, N, K, act, f32;
  hipStream_t st;
};
template <int MT, int NT, int NW, int GS>
void go4z(const Plan4& p, const Args4& a) {
  const int kt = (a.K + QT_K - 1) / QT_K;
  const dim3 grid(p.splits, p.nb, p.mb);
  if (a.z)
    int4_mm_k<MT, NT, NW, GS, true><<<grid, NW * 64, 0, a.st>>>(a.x, a.w, a.s, a.z, a.b, a.y, a.part, a.M, a.N, a.K, kt, a.act, a.f32);
  else
    int4_mm_k<MT, NT, NW, GS, false><<<grid, NW * 64, 0, a.st>>>(a.x, a.w, a.s, a.z, a.b, a.y, a.part, a.M, a.N, a.K, kt, a.act, a.f32);
}
template <int MT, int NT, int NW>
void go4(int gs, const Plan4& p, const Args4& a) {
  if (gs == 1) go4z<MT, NT, NW, 1>(p, a);
  else if (gs == 2) go4z<MT, NT, NW, 2>(p, a);
  else go4z<MT, NT, NW, 4>(p, a);
}
}  // namespace

extern "C" {

// *floats: workspace of a product of M rows (0 where none is needed)
int ptg_int4_ws(int M, int N, int K, void* floats) {
  const Plan4 p = M > 0 ? plan4(M, N, K) : Plan4{1, 1, 1, 1, 1};
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
  const Args4 a{(const bf16_t*)x, (const uint8_t*)w, (const bf16_t*)scale, (const uint8_t*)zero, (const float*)bias, y,
                part, M, N, K, act, f32, stream};
  const int gs = group / 32;
  if (p.mt == 1 && p.nt == 1) go4<1, 1, 16>(gs, p, a);
  else if (p.mt == 1) go4<1, 2, 16>(gs, p, a);
  else if (p.mt == 2) go4<2, 2, 8>(gs, p, a);
  else go4<4, 4, 8>(gs, p, a);
  if (part) {
    const long total = (long)M * N;
    const int blocks = (int)((total + 255) / 256);
    if (f32) int4_join_k<true><<<blocks, 256, 0, stream>>>(part, (const float*)bias, y, total, N, p.splits, act);
    else int4_join_k<false><<<blocks, 256, 0, stream>>>(part, (const float*)bias, y, total, N, p.splits, act);
  }
  PTG_RETURN_LAUNCH();
}

}  // extern "C"
