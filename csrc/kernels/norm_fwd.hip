// Block norm, forward (norm.h): d = drop(scale * gate * post(x)); h = res + d; u = pre(h).
//
// Bound by HBM: x and res in, h and u out, each once; statistics, the gate, the dropout mask and both
// affine maps live in registers between the load and the stores of a row.  u is taken from the
// unrounded h.  Statistics are fp32 and kept for the backward pass ([4][M]).
#include "norm.h"

template <typename T, int LPR, int NT, bool ALN>
__global__ __launch_bounds__(NT) void block_norm_fwd_k(BlkArgs a) {
  __shared__ float2 xch[2 * (NT / 64)];
  const int tid = threadIdx.x, tpr = LPR < 64 ? LPR : a.tpr, slots = NT / tpr, slot = tid / tpr;
  const int c0 = (tid % tpr) * 8, C = a.C, nv = ALN ? (c0 < C ? 8 : 0) : min(max(C - c0, 0), 8);
  RowX rx{xch, 0, tid >> 6, NT / 64, LPR < 64 ? 0 : (slot * tpr) >> 6, tpr >> 6};
  const uint64_t step = a.drop ? drop_step(a.d) : 0;
  float g1[8], b1[8], g2[8], b2[8], gt[8];
  vec8(g1, a.g1, c0, nv, 1.f);
  vec8(b1, a.b1, c0, nv, 0.f);
  vec8(g2, a.g2, c0, nv, 1.f);
  vec8(b2, a.b2, c0, nv, 0.f);
  vec8(gt, a.gate_mode == GATE_VEC ? (const float*)a.gate : nullptr, c0, nv, 1.f);
  for (long r0 = (long)blockIdx.x * slots; r0 < a.M; r0 += (long)gridDim.x * slots) {
    const long row = r0 + slot;
    const bool on = row < a.M && nv > 0;
    Raw8<T> rx8, rr8, rg8;
    float f[8], r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { f[j] = 0.f; r[j] = 0.f; }
    if (on) {
      load8<ALN>(rx8, a.x, row, C, c0, nv);
      if (a.res) load8<ALN>(rr8, a.res, row, C, c0, nv);
      if (a.gate_mode == GATE_GROUP) load8<ALN>(rg8, a.gate, row / a.rpg, C, c0, nv);
      rx8.get(f);
      if (a.res) rr8.get(r);
      if (a.gate_mode == GATE_GROUP) rg8.get(gt);
    }
    float m1 = 0.f, s1 = 1.f, m2 = 0.f, s2 = 1.f;
    if (a.kind1) {
      row_stats<LPR>(f, nv, C, a.kind1, a.eps1, rx, m1, s1);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf((f[j] - m1) * s1, g1[j], b1[j]);
    }
    const uint32_t keep = a.drop && on ? row_keep<ALN>(a, step, row, c0) : 0xFFu;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = f[j] * gt[j] * a.scale;
      const float k = a.drop ? ((keep >> j) & 1u ? d * a.d.scale : 0.f) : d;
      f[j] = j < nv ? r[j] + k : 0.f;
    }
    if (a.h && on) {
      rx8.set(f);
      store8<ALN>(rx8, a.h, row, C, c0, nv);
    }
    if (a.kind2) {
      row_stats<LPR>(f, nv, C, a.kind2, a.eps2, rx, m2, s2);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf((f[j] - m2) * s2, g2[j], b2[j]);
      if (on) {
        rx8.set(f);
        store8<ALN>(rx8, a.u, row, C, c0, nv);
      }
    }
    if (a.stats && row < a.M && c0 == 0) {
      a.stats[row] = m1;
      a.stats[a.M + row] = s1;
      a.stats[2 * a.M + row] = m2;
      a.stats[3 * a.M + row] = s2;
    }
  }
}

namespace {
template <typename T, bool ALN>
int fwd_launch(const BlkArgs& a, hipStream_t stream) {
  auto go = [&](auto kern, int nt, int tpr) {
    BlkArgs b = a;
    b.tpr = tpr;
    const long slots = nt / tpr, wgs = (a.M + slots - 1) / slots, cap = 2048L * 256 / nt;
    kern<<<(int)(wgs < cap ? wgs : cap), nt, 0, stream>>>(b);
  };
  const int C = a.C;
  if (C <= 16) go(block_norm_fwd_k<T, 2, 256, ALN>, 256, 2);
  else if (C <= 64) go(block_norm_fwd_k<T, 8, 256, ALN>, 256, 8);
  else if (C <= 256) go(block_norm_fwd_k<T, 32, 256, ALN>, 256, 32);
  else if (C <= 512) go(block_norm_fwd_k<T, 64, 256, ALN>, 256, 64);
  else if (C <= 1024) go(block_norm_fwd_k<T, 64, 256, ALN>, 256, 128);
  else if (C <= 2048) go(block_norm_fwd_k<T, 64, 256, ALN>, 256, 256);
  else if (C <= 4096) go(block_norm_fwd_k<T, 64, 512, ALN>, 512, 512);
  else go(block_norm_fwd_k<T, 64, 1024, ALN>, 1024, 1024);
  PTG_RETURN_LAUNCH();
}
}  // namespace

extern "C" {

// aligned: every tensor starts on 16 bytes and C % 8 == 0.  Rows per gate group: rpg.
int ptg_block_norm_fwd(const void* x, const void* res, const void* gate, void* h, void* u, const void* g1,
                       const void* b1, const void* g2, const void* b2, void* stats, long M, int C, int f32,
                       int aligned, int kind1, float eps1, int kind2, float eps2, int gate_mode, long rpg, float scale,
                       int drop, int thr, float dscale, long seed, long step, const void* step_dev,
                       hipStream_t stream) {
  if (M <= 0) return 0;
  if (C < 1 || C > 8192) return (int)hipErrorInvalidValue;
  BlkArgs a{};
  a.x = x; a.res = res; a.gate = gate; a.h = h; a.u = u;
  a.g1 = (const float*)g1; a.b1 = (const float*)b1; a.g2 = (const float*)g2; a.b2 = (const float*)b2;
  a.stats = (float*)stats;
  a.M = M; a.C = C; a.kind1 = kind1; a.kind2 = kind2; a.eps1 = eps1; a.eps2 = eps2;
  a.gate_mode = gate_mode; a.rpg = rpg > 0 ? rpg : 1; a.scale = scale; a.drop = drop;
  a.d = drop_args(thr, dscale, seed, step, step_dev);
  if (f32) return aligned ? fwd_launch<float, true>(a, stream) : fwd_launch<float, false>(a, stream);
  return aligned ? fwd_launch<bf16_t, true>(a, stream) : fwd_launch<bf16_t, false>(a, stream);
}

}  // extern "C"
