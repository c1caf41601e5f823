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
// The products run on 16 + u; -(16 + z) times the sum of a group's inputs (MFMAs with ones) leaves
// sum (u - z) x.  Products are exact in fp32, and the offset costs at most (16 + 15) / |u - z| of an fp32
// rounding.  Scales multiply the fp32 sum of a group, never a weight.
#include <limits.h>

#include "common.h"

namespace {

constexpr int QT_K = 128;  // inputs of a weight tile

PTG_DEV f32x4_t mfma32(const U4& a, const U4& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}
// 8 weights of a dword as bf16 16 + u
PTG_DEV U4 dec8(uint32_t w, uint32_t E = 0x41804180u) {
  constexpr uint32_t M = 0x00780078u;
  U4 o;
  o.x = (w & M) | E;
  o.y = ((w >> 4) & M) | E;
  o.z = ((w >> 8) & M) | E;
  o.w = (__builtin_amdgcn_alignbit(w, w, 12) & M) | E;
  return o;
}

// An output again, term by term from the definition.  The offset sums above turn an infinity among the
// inputs (and a product that leaves fp32 at 31 times its size) into NaN; an output that came out infinite
// or NaN is settled here, so y is what the formula gives for any x.  Finite outputs never come here.
template <int GS>
PTG_DEV float int4_term_by_term(const bf16_t* x, const uint8_t* w, const bf16_t* scale, const uint8_t* zero, int n,
                                int K, int kt) {
  float s = 0.f;
  for (int k = 0; k < K; k += 8) {
    const long tile = (long)(n >> 4) * kt + k / QT_K;
    const int i = (k & 127) >> 5, quarter = (k & 31) >> 3;
    uint32_t d = *(const uint32_t*)(w + tile * 1024 + (quarter * 16 + (n & 15)) * 16 + i * 4);
    d = __builtin_amdgcn_alignbit(d, d, 3);
    const long si = (tile * 16 + (n & 15)) * (4 / GS) + i / GS;
    const float sc = bf2f(scale[si]), z = zero ? (float)zero[si] : 8.f;
    for (int e = 0; e < 8; ++e)
      s = fmaf(((float)((d >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - z) * sc, bf2f(x[k + e]), s);
    if (s != s) break;
  }
  return s;
}
struct Args4 {
  const bf16_t* x;
  const uint8_t* w;
  const bf16_t* s;
  const uint8_t* z;
  const float* b;
  void* y;
  float* part;  // null: the kernel finishes y itself
  int M, N, K, kt, act, f32;
};
// y[m][n] from the sum s over all of K
template <int GS>
PTG_DEV void int4_finish(const Args4& a, int m, int n, float s) {
  if (!(fabsf(s) < __builtin_inff())) s = int4_term_by_term<GS>(a.x + (long)m * a.K, a.w, a.s, a.z, n, a.K, a.kt);
  if (a.b) s += a.b[n];
  if (a.act && s < 0.f) s = 0.f;  // NaN stays
  const long o = (long)m * a.N + n;
  if (a.f32) ((float*)a.y)[o] = s;
  else ((bf16_t*)a.y)[o] = f2bf(s);
}

}  // namespace

// Up to 32 rows, and small products: bound by reading the weights once (16 x 8192 x 8192: 12.8 us a pass among
// others, 2.9 TB/s, 14.6 in the median where launches are traced; about 2 us pass before the first data are there,
// and the waves wait for 77 % of their time).  A wave computes 16 * MT rows x 16 * NT outputs over its
// share of K; the NW waves of a workgroup take the tiles of the workgroup's K range in turn and are joined
// in LDS in a fixed order.  A product tile is one MFMA chain: sum (16 + u) x on top of -(16 + z) * sum x,
// the latter from one MFMA with ones for every 32 inputs that all NT tiles share.  Waves that need few
// registers hide the memory's latency, not loads ahead of their use: with 2 or 3 tiles in flight a wave
// (88 or 122 registers instead of 62) 1 x 2048 x 20480 took 11.1 or 11.3 us instead of 9.5.
// Where K is split over workgroups they leave fp32 sums in part[split][M][N], else they finish y.
template <int GS>
struct Group {  // of a tile: 4 / GS groups
  static constexpr int NG = 4 / GS;
  bf16_t s[NG];
  uint8_t z[NG];
};
template <int MT, int NT, int NW, int GS, bool HASZ>
__global__ __launch_bounds__(NW * 64) void int4_mm_k(Args4 a, int splits) {
  constexpr int NG = 4 / GS, R = MT * NT * 4;
  constexpr bool FLAT = R * NW <= 128;  // every wave's sums in LDS at once, else pairwise
  __shared__ float red[(FLAT ? NW : NW / 2) * R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, q = lane >> 4;
  const int nbi = splits == 1 ? blockIdx.x : blockIdx.x / splits, sp = blockIdx.x - nbi * splits;
  const int nb = nbi * NT, m0 = blockIdx.y * 16 * MT;
  const int M = a.M, N = a.N, K = a.K, kt = a.kt, ntiles = (N + 15) / 16;
  const int t0 = (int)((long)kt * sp / splits), t1 = (int)((long)kt * (sp + 1) / splits);
  // rows, tiles of outputs and inputs that do not exist read 0
  const Rsrc rx = make_rsrc(a.x + (long)m0 * K, (uint32_t)min(M - m0, 16 * MT) * (uint32_t)K * 2u);
  const Rsrc rw = make_rsrc(a.w + (long)nb * kt * 1024, (uint32_t)min(ntiles - nb, NT) * (uint32_t)kt * 1024u);
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[i][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  struct Tile {
    U4 w[NT], x[MT][4];
    Group<GS> g[NT];
  };
  auto fetch = [&](Tile& f, int t) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f.w[n] = bload16(rw, ((uint32_t)n * (uint32_t)kt + (uint32_t)t) * 1024u + lane * 16u);
      const long at = (((long)min(nb + n, ntiles - 1) * kt + t) * 16 + n16) * NG;
      __builtin_memcpy(f.g[n].s, a.s + at, 2 * NG);
      if (HASZ) __builtin_memcpy(f.g[n].z, a.z + at, NG);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = t * QT_K + j * 32 + q * 8;
        f.x[i][j] = bload16(rx, k < K ? ((uint32_t)(i * 16 + n16) * (uint32_t)K + (uint32_t)k) * 2u : PTG_OOB);
      }
  };
  U4 ones;
  ones.x = 0x3F803F80u; ones.y = ones.x; ones.z = ones.x; ones.w = ones.x;
  auto multiply = [&](const Tile& f) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t xs[MT];  // sum of the group's inputs, the same in every column
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xs[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) xs[i] = mfma32(f.x[i][g * GS + j], ones, xs[i]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t ww[4] = {f.w[n].x, f.w[n].y, f.w[n].z, f.w[n].w};
        const float s = bf2f(f.g[n].s[g]);
        const float zf = HASZ ? -16.f - (float)f.g[n].z[g] : -24.f;
        U4 b[GS];
#pragma unroll
        for (int j = 0; j < GS; ++j) b[j] = dec8(ww[g * GS + j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          f32x4_t d = xs[i] * zf;
#pragma unroll
          for (int j = 0; j < GS; ++j) d = mfma32(f.x[i][g * GS + j], b[j], d);
          acc[i][n] += d * s;
        }
      }
    }
  };
  for (int t = t0 + wave; t < t1; t += NW) {
    Tile f;
    fetch(f, t);
    multiply(f);
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
    if (a.part) a.part[((long)sp * M + m) * N + col] = s;
    else int4_finish<GS>(a, m, col, s);
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

// Larger products of more than 32 rows are bound by the matrix cores and by what feeds them, not by HBM: 256 x
// 2048 x 20480 takes 32 us and 5 for the join, 670 TFLOP/s, with the matrix cores 42 % and the vector pipes 52 %
// busy.  A pair of stages costs 5000 cycles, of which the two
// waves' MFMAs are 2560 and their decoding, scaling and sums 2300: they overlap little.  A workgroup
// takes 64 rows x 256 outputs; 4 waves hold 64 x 64 of them each, twice over: waves 4..7 work on every
// other stage of 128 inputs, so two waves share a SIMD and one multiplies while the other waits, and the
// two halves are added at the end.  A stage (64 rows of inputs, 16 KB, and 16 weight tiles, 16 KB) goes
// straight to LDS, into a ring of QR.  Inputs lie there as rows of 16 chunks of 16 bytes, chunk c of row
// r at place c ^ (r & 15): the 16 rows that a wave reads at once are in 16 places, free of bank conflicts.
constexpr int QT_M = 64, QT_N = 256, QR = 5, Q_XB = QT_M * 256, Q_STAGE = Q_XB + QT_N / 16 * 1024;
typedef __attribute__((address_space(3))) void q_lds_t;
template <int N>
PTG_DEV void q_wait_vm() {  // at most N vector loads in flight, no LDS read
  static_assert(N >= 0 && N < 64, "vmcnt");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
}
template <int GS, bool HASZ>
__global__ __launch_bounds__(512) void int4_tile_k(Args4 a, int mb, int nbk, int splits) {
  constexpr int NG = 4 / GS;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, q = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), half = wid >> 2, wn = wid & 3;
  // the tiles of one split are neighbours on one XCD: its L2 reads that split's inputs and weights once
  const int item = xcd_remap(blockIdx.x, gridDim.x), sp = item / (mb * nbk), rest = item - sp * (mb * nbk);
  const int m0 = (rest % mb) * QT_M, nb = (rest / mb) * (QT_N / 16), ntiles = (a.N + 15) / 16, kt = a.kt;
  const int t0 = (int)((long)kt * sp / splits), nk = (int)((long)kt * (sp + 1) / splits) - t0;
  const Rsrc rx = make_rsrc(a.x + (long)m0 * a.K, (uint32_t)min(a.M - m0, QT_M) * (uint32_t)a.K * 2u);
  const Rsrc rw = make_rsrc(a.w + (long)nb * kt * 1024, (uint32_t)min(ntiles - nb, QT_N / 16) * (uint32_t)kt * 1024u);
  // a wave loads 8 rows of inputs (4 at a time) and 2 weight tiles of each stage
  uint32_t xo[2], wo[2];
  int xt[2];  // stages whose chunk exists
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = (wid * 2 + j) * 4 + q, k = t0 * QT_K + (n16 ^ (row & 15)) * 8;
    xo[j] = ((uint32_t)row * (uint32_t)a.K + (uint32_t)k) * 2u;
    xt[j] = min(nk, (a.K - k + QT_K - 1) / QT_K);
    wo[j] = ((uint32_t)(wid * 2 + j) * (uint32_t)kt + (uint32_t)t0) * 1024u + (uint32_t)lane * 16u;
  }
  // stages past the end are issued too, out of range (zeros, no traffic): the count of loads in flight stays known.
  // So does their order, by the barrier behind each: q_wait_vm counts on the stages arriving one after another,
  // and to the scheduler their places in LDS have nothing to do with each other.
  auto issue = [&](int t, unsigned char* base) {
    base += wid * 2048;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (q_lds_t*)(base + j * 1024), 16,
                                               t < xt[j] ? xo[j] + (uint32_t)t * (QT_K * 2u) : PTG_OOB, 0, 0, 0);
    const uint32_t wt = t < nk ? (uint32_t)t * 1024u : PTG_OOB;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (q_lds_t*)(base + Q_XB + j * 1024), 16, wo[j] + wt, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  const bf16_t* sp_[4];  // this lane's scales and zero points of the next stage
  const uint8_t* zp_[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int nt = nb + wn * 4 + n;
    const long at = (((long)(nt < ntiles ? nt : ntiles - 1) * kt + t0) * 16 + n16) * NG;
    sp_[n] = a.s + at;
    if (HASZ) zp_[n] = a.z + at;
  }
  Group<GS> gn[4];
  auto scales = [&](int t) {
    t = t < nk ? t : nk - 1;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      __builtin_memcpy(gn[n].s, sp_[n] + t * 16 * NG, 2 * NG);
      if (HASZ) __builtin_memcpy(gn[n].z, zp_[n] + t * 16 * NG, NG);
    }
  };
  f32x4_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[i][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  U4 ones;
  ones.x = 0x3F803F80u; ones.y = ones.x; ones.z = ones.x; ones.w = ones.x;
  uint32_t e16 = 0x41804180u;
  asm volatile("" : "+v"(e16));  // in a vector register: and-or takes one scalar
  scales(half);
#pragma unroll
  for (int t = 0; t < QR - 2; ++t) issue(t, smem + t * Q_STAGE);
  // One pair of stages.  `st` is what this wave works on, f0 and f1 where stages t + QR - 2 and t + QR - 1 go:
  // as separate restricted arguments, or the compiler would drain the loads in flight before an LDS read.
  auto pair = [&](int t, const unsigned char* __restrict__ st, unsigned char* __restrict__ f0,
                  unsigned char* __restrict__ f1) __attribute__((always_inline)) {
    Group<GS> gc[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) gc[n] = gn[n];
    scales(t + 2 + half);
    issue(t + QR - 2, f0);
    issue(t + QR - 1, f1);
    const unsigned char* sx = st + n16 * 256;
    U4 wv[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) wv[n] = *(const U4*)(st + Q_XB + wn * 4096 + lane * 16 + n * 1024);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t xs[4], d[4][4];
      const f32x4_t z4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < GS; ++j) {
        const int jj = g * GS + j;
        U4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const U4*)(sx + i * 4096 + ((jj * 4 + q) ^ n16) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) xs[i] = mfma32(x[i], ones, j ? xs[i] : z4);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t ww[4] = {wv[n].x, wv[n].y, wv[n].z, wv[n].w};
          const U4 b = dec8(ww[jj], e16);
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i][n] = mfma32(x[i], b, j ? d[i][n] : z4);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float s = bf2f(gc[n].s[g]), zs = s * (HASZ ? -16.f - (float)gc[n].z[g] : -24.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i][n] += d[i][n] * s;
          acc[i][n] += xs[i] * zs;
        }
      }
    }
  };
  int slot = 0, fill = QR - 2;  // of stage t; of stage t + QR - 2
  for (int t = 0; t < nk; t += 2) {
    q_wait_vm<4 * (QR - 4)>();     // this wave's part of stages t and t + 1 has landed
    __builtin_amdgcn_s_barrier();  // and every wave's; all have left the buffers of the two before
    asm volatile("" ::: "memory");
    const int slot1 = slot + 1 == QR ? 0 : slot + 1, fill1 = fill + 1 == QR ? 0 : fill + 1;
    pair(t, smem + (half ? slot1 : slot) * Q_STAGE, smem + fill * Q_STAGE, smem + fill1 * Q_STAGE);
    slot = slot1 + 1 == QR ? 0 : slot1 + 1;
    fill = fill1 + 1 == QR ? 0 : fill1 + 1;
  }
  // The halves meet in LDS, [half][64 rows][256 + 4 outputs]; then all 512 threads write rows of 4 outputs.
  q_wait_vm<0>();
  __syncthreads();
  float* red = (float*)smem;
  constexpr int RS = QT_N + 4, RH = QT_M * RS;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        red[half * RH + (i * 16 + q * 4 + r) * RS + (wn * 4 + n) * 16 + n16] = acc[i][n][r];
  __syncthreads();
  const int c = lane * 4, col = nb * 16 + c, cols = min(a.N - col, 4);
#pragma unroll 1
  for (int r = wid; r < min(a.M - m0, QT_M); r += 8) {
    const f32x4_t v = *(const f32x4_t*)(red + r * RS + c) + *(const f32x4_t*)(red + RH + r * RS + c);
    if (a.part) {
      float* o = a.part + ((long)sp * a.M + m0 + r) * a.N + col;
      if (cols == 4) __builtin_memcpy(o, &v, 16);
      else
        for (int k = 0; k < cols; ++k) o[k] = v[k];
    } else {
      for (int k = 0; k < cols; ++k) int4_finish<GS>(a, m0 + r, col + k, v[k]);
    }
  }
}

// y = act(sum of the splits + bias), V outputs of a row a thread
template <int GS, int V>
__global__ __launch_bounds__(256) void int4_join_k(Args4 a, int splits) {
  const long total = (long)a.M * a.N, i = ((long)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= total) return;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    float p[V];
    __builtin_memcpy(p, a.part + k * total + i, 4 * V);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] += p[j];
  }
  const int m = (int)(i / a.N), n = (int)(i - (long)m * a.N);
#pragma unroll
  for (int j = 0; j < V; ++j) int4_finish<GS>(a, m, n + j, s[j]);
}

namespace {
constexpr int Q_NW = 16;  // waves of int4_mm_k
// Outputs alone give one workgroup a CU only where N is large; otherwise K is split, up to one workgroup a
// CU (two: 16 x 8192 x 8192 17.0 instead of 13.4 us, 12 x 2048 x 20480 13.9 instead of 10.9).  A split costs
// the join, about 2.2 us, so a wave keeps at least 4 tiles (one row: 4 x 2048 x 8192 7.2 us whole, 9.4 in two)
// or 2 where it works on two columns of tiles at a time (12 x 2048 x 20480 10.9 us in four, 22.5 whole).
//
// Above 32 rows the tile kernel, unless int4_mm_k is through after `steps` = 2 tiles of a wave (4 for groups
// below 128, whose sums cost the tile kernel more): 128 x 1024 x 1024 (1 step) 7.4 instead of 12.0 us, 256 x 2048
// x 2048 (2) 16.3 instead of 16.7, 128 x 8192 x 1024 (4) 18.9 instead of 16.1, 64 x 8192 x 8192 (8) 40.1 instead of
// 22.4; groups of 32, 256 x 1024 x 4096 (2) 13.9 instead of 19.1, 128 x 2048 x 8192 (4) 22.4 instead of 23.8, 256 x
// 8192 x 512 (8) 39.8 instead of 17.0.  Up to 32 rows it has the fewer rows for its 64: 12 x 8192 x 8192
// 17.3 instead of 12.1 us.
struct Plan4 { int tile, mt, nt, mb, nb, splits; };
Plan4 plan4(int M, int N, int K, int group) {
  Plan4 p;
  const long kt = (K + QT_K - 1) / QT_K;
  p.tile = 0;
  p.mt = M <= 16 ? 1 : 2;
  p.nt = M <= 8 ? 1 : 2;  // two: half the reads of the inputs; 16 x 8192 x 8192 13.4 us instead of 19.5
  p.mb = (M + 16 * p.mt - 1) / (16 * p.mt);
  p.nb = (N + 16 * p.nt - 1) / (16 * p.nt);
  const long least = Q_NW * (p.nt == 1 ? 4 : 2);  // tiles of a split
  long wgs = (long)p.nb * p.mb, s = (256 + wgs - 1) / wgs;
  s = s < kt / least ? s : kt / least;
  s = s < 1 ? 1 : s;
  const long steps = (wgs * s + 255) / 256 * ((kt + s * Q_NW - 1) / (s * Q_NW));
  if (M > 32 && steps > (group == 128 ? 2 : 4)) {
    p.tile = 1;
    p.mb = (M + QT_M - 1) / QT_M;
    p.nb = (N + QT_N - 1) / QT_N;
    wgs = (long)p.nb * p.mb;
    s = 256 / wgs < kt / 4 ? 256 / wgs : kt / 4;
    s = s < 1 ? 1 : s;
  }
  p.splits = (int)s;
  return p;
}
template <int MT, int NT, int NW, int GS>
void go4(const Plan4& p, const Args4& a, hipStream_t st) {
  const dim3 grid((unsigned)p.splits * p.nb, p.mb);
  if (a.z) int4_mm_k<MT, NT, NW, GS, true><<<grid, NW * 64, 0, st>>>(a, p.splits);
  else int4_mm_k<MT, NT, NW, GS, false><<<grid, NW * 64, 0, st>>>(a, p.splits);
}
template <int GS>
void go4t(const Plan4& p, const Args4& a, hipStream_t st) {
  auto kern = a.z ? int4_tile_k<GS, true> : int4_tile_k<GS, false>;
  constexpr int lds = QR * Q_STAGE;
  static uint64_t set[2];  // devices whose limit is raised, for each of the two kernels
  ptg_allow_lds((const void*)kern, lds, set[a.z != nullptr]);
  kern<<<p.mb * p.nb * p.splits, 512, lds, st>>>(a, p.mb, p.nb, p.splits);
}
template <int GS>
int go4g(const Plan4& p, const Args4& a, hipStream_t st) {
  if (p.tile) go4t<GS>(p, a, st);
  else if (p.mt == 1 && p.nt == 1) go4<1, 1, Q_NW, GS>(p, a, st);
  else if (p.mt == 1) go4<1, 2, Q_NW, GS>(p, a, st);
  else go4<2, 2, Q_NW, GS>(p, a, st);
  if (a.part) {
    const long total = (long)a.M * a.N;
    if (a.N % 4 == 0) int4_join_k<GS, 4><<<(int)((total / 4 + 255) / 256), 256, 0, st>>>(a, p.splits);
    else int4_join_k<GS, 1><<<(int)((total + 255) / 256), 256, 0, st>>>(a, p.splits);
  }
  PTG_RETURN_LAUNCH();
}
}  // namespace

extern "C" {

// *floats: workspace of a product of M rows (0 where none is needed)
int ptg_int4_ws(int M, int N, int K, int group, void* floats) {
  const int splits = M > 0 ? plan4(M, N, K, group).splits : 1;
  *(long*)floats = splits > 1 ? (long)splits * M * N : 0;
  return 0;
}

// Arguments, 64 bits each.  x: 16-byte aligned; w, scale, zero: tile layout; group 32, 64 or 128; zero null: 8
// everywhere; act 0 linear, 1 ReLU
struct Int4Call {
  const bf16_t* x;
  const uint8_t* w;
  const bf16_t* scale;
  const uint8_t* zero;
  const float* bias;
  void* y;
  float* ws;
  int64_t M, N, K, group, act, f32;
};
int ptg_int4_dense(const void* call, hipStream_t stream) {
  const Int4Call& c = *(const Int4Call*)call;
  if (c.M <= 0 || c.N <= 0) return 0;
  if (c.M > INT_MAX || c.N > INT_MAX || c.K > INT_MAX) return (int)hipErrorInvalidValue;
  const int M = (int)c.M, N = (int)c.N, K = (int)c.K, group = (int)c.group;
  // a block of rows or of outputs stays below 2 GiB
  if ((group != 32 && group != 64 && group != 128) || K < group || K % group || K > (1 << 22) || ((uintptr_t)c.x & 15))
    return (int)hipErrorInvalidValue;
  const Plan4 p = plan4(M, N, K, group);
  if (p.splits > 1 && !c.ws) return (int)hipErrorInvalidValue;
  const Args4 a{c.x, c.w, c.scale, c.zero, c.bias, c.y, p.splits > 1 ? c.ws : nullptr, M, N, K, (K + QT_K - 1) / QT_K,
                (int)c.act, (int)c.f32};
  if (group == 32) return go4g<1>(p, a, stream);
  if (group == 64) return go4g<2>(p, a, stream);
  return go4g<4>(p, a, stream);
}

}  // extern "C"
