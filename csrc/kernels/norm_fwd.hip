// Block norm, forward (norm.h): d = drop(scale * gate * post(x)); h = res + d; u = pre(h).
//
// Bound by HBM (32768 x 2048 bf16: 99 us, 5.4 TB/s; 4096 x 1024, 12.7 us, by its start and its end): x and res
// in, h and u out, each once; statistics, the gate, the dropout mask and both
// affine maps live in registers between the load and the stores of a row.  The next row's loads are
// issued before the current row is worked on, so the row sums (and the barrier of rows of several waves)
// run while memory is busy.  u is taken from the unrounded h.  Statistics are fp32 and kept for the
// backward pass ([4][M]).
#include "norm.h"

template <typename T, int LPR, int NT, bool ALN, bool PO, bool PR, bool DROP>
__global__ __launch_bounds__(NT) void block_norm_fwd_k(BlkArgs a) {
  __shared__ float2 xch[2 * (NT / 64)];
  extern __shared__ float4 dyn[];
  float* vecs = (float*)dyn;
  const int tid = threadIdx.x, tpr = LPR < 64 ? LPR : a.tpr, slots = NT / tpr, slot = tid / tpr;
  const int C = a.C, c0 = (tid % tpr) * 8;
  const Lane<T, ALN, LPR == 2> ln(slot, c0, C);
  const int nv = ln.nv, cc = nv ? c0 : 0;
  RowX rx;
  rx.init(xch, tid, NT, LPR, tpr, C);
  const uint64_t step = DROP ? drop_step(a.d) : 0;
  ColVecs<NT, 5> cv;
  enum { G1, B1, G2, B2, GV };
  long r0 = (long)blockIdx.x * slots;
  const long stride = (long)gridDim.x * slots;
  auto rows_at = [&](long r) { return (uint32_t)(a.M - r < slots ? (a.M > r ? a.M - r : 0) : slots); };
  uint32_t rows = rows_at(r0);
  bool on = slot < (int)rows && nv > 0;
  Raw8<T> nx, nr, t;
  ln.load(nx, a.x, r0 * C, rows, C, on);
  ln.load(nr, a.res, r0 * C, rows, C, on);
  cv.v[G1] = {PO ? a.g1 : nullptr, 1.f, 1.f};
  cv.v[B1] = {PO ? a.b1 : nullptr, 0.f, 1.f};
  cv.v[G2] = {PR ? a.g2 : nullptr, 1.f, 1.f};
  cv.v[B2] = {PR ? a.b2 : nullptr, 0.f, 1.f};
  const float sc = DROP ? a.scale * a.d.scale : a.scale;  // scale and keep scale, times the gate
  cv.v[GV] = {a.gate_mode == GATE_VEC ? (const float*)a.gate : nullptr, 1.f, sc};
  cv.init(vecs, C, tid, a.vecs);
  const float lay1 = a.kind1 == NORM_LAYER ? 1.f : 0.f, lay2 = a.kind2 == NORM_LAYER ? 1.f : 0.f;
  const bool full = C == tpr * 8;
  __syncthreads();
  while (r0 < a.M) {
    asm volatile("" ::: "memory");  // the column vectors stay in LDS
    float f[8], r[8], v[8], w[8];
    ln.get(nx, f, on);
    ln.get(nr, r, on);
    const long cur = r0, at = r0 * C;
    const uint32_t crows = rows;
    const bool con = on;
    r0 += stride;
    rows = rows_at(r0);
    on = slot < (int)rows && nv > 0;
    ln.load(nx, a.x, r0 * C, rows, C, on);
    ln.load(nr, a.res, r0 * C, rows, C, on);
    float m1 = 0.f, s1 = 1.f, m2 = 0.f, s2 = 1.f;
    if (PO) {
      row_stats<LPR, ALN>(f, nv, lay1, a.eps1, rx, m1, s1);
      cv.get(vecs, G1, v, cc, nv);
      cv.get(vecs, B1, w, cc, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf((f[j] - m1) * s1, v[j], w[j]);
    }
    if (a.gate_mode == GATE_GROUP) {
      const Lane<T, false, LPR == 2> gl(0, c0, C);
      gl.load(t, a.gate, (cur + slot) / a.rpg * C, 0, C, con);
      gl.get(t, v, con);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= sc;
    } else {
      cv.get(vecs, GV, v, cc, nv);
    }
    if (DROP) {
      bool keep[8];
      row_keep<ALN>(a, step, at, ln.off, keep);
      // a dropped value is 0 whatever the branch holds
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = r[j] + (keep[j] ? f[j] * v[j] : 0.f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf(f[j], v[j], r[j]);
    }
    if (!ALN || !full) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = j < nv ? f[j] : 0.f;
    }
    meet<LPR, ALN>(a, PO);
    if (a.h) {
      t.set(f);
      ln.store(t, a.h, at, crows, C, con);
    }
    if (PR) {
      row_stats<LPR, ALN>(f, nv, lay2, a.eps2, rx, m2, s2);
      cv.get(vecs, G2, v, cc, nv);
      cv.get(vecs, B2, w, cc, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf((f[j] - m2) * s2, v[j], w[j]);
      t.set(f);
      ln.store(t, a.u, at, crows, C, con);
    }
    if (a.stats && con && c0 == 0) {
      float* st = a.stats + cur + slot;
      st[0] = m1;
      st[a.M] = s1;
      st[2 * a.M] = m2;
      st[3 * a.M] = s2;
    }
  }
}

namespace {
// Four waves a SIMD; three for rows above 1024 columns, which read more rows at a time as it is (32768 x 2048,
// forward and backward together: 276 us with four, 259 with three; 401408 x 64: 56.9 with four, 58.2 with three).
// Above 2048 columns a workgroup is 16 waves, one a CU (4096 x 8192 forward: 73.7 us; 76.6 with two a CU, 93.9 on
// three quarters of the CUs).
template <typename T, bool ALN, bool PO, bool PR, bool DROP>
int fwd_launch(const BlkArgs& a, hipStream_t stream) {
  auto go = [&](auto kern, int nt, int tpr) {
    BlkArgs b = a;
    b.tpr = tpr;
    const long slots = nt / tpr, wgs = (a.M + slots - 1) / slots, cap = a.C <= 1024 ? 1024 : a.C <= 2048 ? 768 : 256;
    const bool there[5] = {a.kind1 && a.g1, a.kind1 && a.b1, a.kind2 && a.g2, a.kind2 && a.b2, a.gate_mode == GATE_VEC};
    const int lds = col_vec_bytes(nt, a.C, 5, there, VECS_MOST);
    b.vecs = lds / 4;
    static uint64_t set = 0;  // devices whose limit is raised (only 16-wave workgroups get there)
    if (lds > 64 * 1024) ptg_allow_lds((const void*)kern, VECS_MOST, set);
    kern<<<(int)(wgs < cap ? wgs : cap), nt, lds, stream>>>(b);
  };
  const int C = a.C;
  if (C <= 16) go(block_norm_fwd_k<T, 2, 256, ALN, PO, PR, DROP>, 256, 2);
  else if (C <= 64) go(block_norm_fwd_k<T, 8, 256, ALN, PO, PR, DROP>, 256, 8);
  else if (C <= 256) go(block_norm_fwd_k<T, 32, 256, ALN, PO, PR, DROP>, 256, 32);
  else if (C <= 2048) go(block_norm_fwd_k<T, 64, 256, ALN, PO, PR, DROP>, 256, C <= 512 ? 64 : C <= 1024 ? 128 : 256);
  else go(block_norm_fwd_k<T, 64, 1024, ALN, PO, PR, DROP>, 1024, C <= 4096 ? 512 : 1024);
  PTG_RETURN_LAUNCH();
}
template <typename T, bool ALN, bool DROP>
int fwd_kind(const BlkArgs& a, hipStream_t stream) {
  if (a.kind1 && a.kind2) return fwd_launch<T, ALN, true, true, DROP>(a, stream);
  if (a.kind1) return fwd_launch<T, ALN, true, false, DROP>(a, stream);
  return a.kind2 ? fwd_launch<T, ALN, false, true, DROP>(a, stream) : fwd_launch<T, ALN, false, false, DROP>(a, stream);
}
template <typename T, bool ALN>
int fwd_drop(const BlkArgs& a, hipStream_t stream) {
  return a.drop ? fwd_kind<T, ALN, true>(a, stream) : fwd_kind<T, ALN, false>(a, stream);
}
}  // namespace

extern "C" {

// call: a FwdCall.  aligned: every tensor starts on 16 bytes, C % 8 == 0 and first % 8 == 0.  Rows per gate group: rpg.
int ptg_block_norm_fwd(const void* call, hipStream_t stream) {
  const FwdCall& c = *(const FwdCall*)call;
  if (c.M <= 0) return 0;
  if (c.C < 1 || c.C > 8192) return (int)hipErrorInvalidValue;
  BlkArgs a{};
  a.x = c.x; a.res = c.res; a.gate = c.gate; a.h = c.h; a.u = c.u;
  a.g1 = c.g1; a.b1 = c.b1; a.g2 = c.g2; a.b2 = c.b2;
  a.stats = c.stats;
  a.M = c.M; a.C = (int)c.C; a.kind1 = (int)c.kind1; a.kind2 = (int)c.kind2;
  a.eps1 = (float)c.eps1; a.eps2 = (float)c.eps2;
  a.gate_mode = (int)c.gate_mode; a.rpg = c.rpg > 0 ? c.rpg : 1; a.scale = (float)c.scale; a.drop = (int)c.drop;
  a.d = drop_args((int)c.thr, (float)c.dscale, c.seed, c.step, c.step_dev, c.first);
  a.over = !c.aligned && c.h && (c.h == c.x || c.h == c.res);
  if (c.f32) return c.aligned ? fwd_drop<float, true>(a, stream) : fwd_drop<float, false>(a, stream);
  return c.aligned ? fwd_drop<bf16_t, true>(a, stream) : fwd_drop<bf16_t, false>(a, stream);
}

}  // extern "C"
