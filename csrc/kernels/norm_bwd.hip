// Block norm, backward (norm.h).  From du = dL/du and dh = dL/dh (the residual stream's gradient):
//
//   dh' = dh + pre'(du)       pre'(g) = rstd * (g*gamma - mean(g*gamma) [layer] - xhat * mean(g*gamma*xhat))
//   dres = dh';  dd = mask(dh') * dscale;  dgate = sum scale * post(x) * dd
//   dx = post'(scale * gate * dd);  dgamma = sum g * xhat;  dbeta = sum g      for both norms
//
// h and post(x) are computed again from x and res (and the mask drawn again), in fp32: the pass reads
// du, dh, x, res and writes dx, dres, each once, and h need not be kept.  Column sums stay in registers
// over all rows of a workgroup, are joined over its rows in LDS, and a second kernel adds the
// workgroups' partial sums in a fixed order: no atomics, the same bits every run.
#include "norm.h"

// Joins a thread's column sums over the rows (slots) of the workgroup and writes dst[0..C).
template <int LPR, int NT, typename D>
PTG_DEV void flush_cols(float* acc, float* lds, int tid, int tpr, int C, D* dst) {
  constexpr int NW = NT / 64;
  int rows, cols;
  if (LPR < 64) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) acc[j] += __shfl_xor(acc[j], o, 64);
    }
    rows = NW;
    cols = LPR * 8;
  } else {
    rows = NT / tpr;
    cols = tpr * 8;
  }
  __syncthreads();
  if (LPR == 64 || (tid & 63) < LPR) {
    const int r = LPR < 64 ? tid >> 6 : tid / tpr, c = LPR < 64 ? (tid & 63) * 8 : (tid % tpr) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) lds[r * cols + c + j] = acc[j];
  }
  __syncthreads();
  for (int c = tid; c < C; c += NT) {
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += lds[r * cols + c];
    if constexpr (sizeof(D) == 2) dst[c] = f2bf(s);
    else dst[c] = s;
  }
}

template <typename T, int LPR, int NT, bool ALN, bool PO, bool PR>
__global__ __launch_bounds__(NT) void block_norm_bwd_k(BlkArgs a) {
  __shared__ float2 xch[2 * (NT / 64)];
  __shared__ float cols[NT * 8];
  const int tid = threadIdx.x, tpr = LPR < 64 ? LPR : a.tpr, slots = NT / tpr, slot = tid / tpr;
  const int c0 = (tid % tpr) * 8, C = a.C, nv = ALN ? (c0 < C ? 8 : 0) : min(max(C - c0, 0), 8);
  RowX rx{xch, 0, tid >> 6, NT / 64, LPR < 64 ? 0 : (slot * tpr) >> 6, tpr >> 6};
  const uint64_t step = a.drop ? drop_step(a.d) : 0;
  const float invC = 1.f / (float)C;
  float g1[8], b1[8], g2[8], gt[8];
  float ag1[8], ab1[8], ag2[8], ab2[8], agt[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) { ag1[j] = 0.f; ab1[j] = 0.f; ag2[j] = 0.f; ab2[j] = 0.f; agt[j] = 0.f; }
  if (PO) {
    vec8(g1, a.g1, c0, nv, 1.f);
    vec8(b1, a.b1, c0, nv, 0.f);
  }
  if (PR) vec8(g2, a.g2, c0, nv, 1.f);
  vec8(gt, a.gate_mode == GATE_VEC ? (const float*)a.gate : nullptr, c0, nv, 1.f);
  RowIter it;
  it.item = blockIdx.x;
  it.enter(a, slot, slots);
  while (it.item < a.items) {
    const long row = it.row(a, slots);
    const bool on = it.valid(a, slots) && nv > 0;
    float x[8], r[8], gu[8], gh[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { x[j] = 0.f; r[j] = 0.f; gu[j] = 0.f; gh[j] = 0.f; }
    float m1 = 0.f, s1 = 0.f, m2 = 0.f, s2 = 0.f;
    Raw8<T> t;
    if (on) {
      load8<ALN>(t, a.x, row, C, c0, nv);
      t.get(x);
      if (PR && a.res) { load8<ALN>(t, a.res, row, C, c0, nv); t.get(r); }
      if (PR) { load8<ALN>(t, a.du, row, C, c0, nv); t.get(gu); }
      if (a.dh) { load8<ALN>(t, a.dh, row, C, c0, nv); t.get(gh); }
      if (a.gate_mode == GATE_GROUP && it.j == 0) { load8<ALN>(t, a.gate, it.g, C, c0, nv); t.get(gt); }
      if (PO && a.kind1) { m1 = a.stats[row]; s1 = a.stats[a.M + row]; }
      if (PR) { m2 = a.stats[2 * a.M + row]; s2 = a.stats[3 * a.M + row]; }
    }
    const uint32_t keep = a.drop && on ? row_keep<ALN>(a, step, row, c0) : 0xFFu;
    float n[8], xh[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xh[j] = PO && a.kind1 ? (x[j] - m1) * s1 : x[j];
      n[j] = PO && a.kind1 ? fmaf(xh[j], g1[j], b1[j]) : x[j];
    }
    if (PR) {
      float h2[8], gg[8], c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = n[j] * gt[j] * a.scale;
        const float k = a.drop ? ((keep >> j) & 1u ? d * a.d.scale : 0.f) : d;
        h2[j] = j < nv ? (r[j] + k - m2) * s2 : 0.f;
        gg[j] = gu[j] * g2[j];
        c1 += gg[j];
        c2 = fmaf(gg[j], h2[j], c2);
        ag2[j] = fmaf(gu[j], h2[j], ag2[j]);
        ab2[j] += gu[j];
      }
      const float2 c = row_sum2<LPR>(make_float2(c1, c2), rx);
      const float k1 = a.kind2 == NORM_LAYER ? c.x * invC : 0.f, k2 = c.y * invC;
#pragma unroll
      for (int j = 0; j < 8; ++j) gh[j] = fmaf(s2, gg[j] - k1 - h2[j] * k2, gh[j]);
    }
    if (a.dres && on) {
      t.set(gh);
      store8<ALN>(t, a.dres, row, C, c0, nv);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float dd = (a.drop ? ((keep >> j) & 1u ? gh[j] * a.d.scale : 0.f) : gh[j]) * a.scale;
      agt[j] = fmaf(dd, n[j], agt[j]);
      gh[j] = dd * gt[j];
    }
    if (PO && a.kind1) {
      float gg[8], c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        gg[j] = j < nv ? gh[j] * g1[j] : 0.f;
        c1 += gg[j];
        c2 = fmaf(gg[j], xh[j], c2);
        if (on) {
          ag1[j] = fmaf(gh[j], xh[j], ag1[j]);
          ab1[j] += gh[j];
        }
      }
      const float2 c = row_sum2<LPR>(make_float2(c1, c2), rx);
      const float k1 = a.kind1 == NORM_LAYER ? c.x * invC : 0.f, k2 = c.y * invC;
#pragma unroll
      for (int j = 0; j < 8; ++j) gh[j] = s1 * (gg[j] - k1 - xh[j] * k2);
    }
    if (a.dx && on) {
      t.set(gh);
      store8<ALN>(t, a.dx, row, C, c0, nv);
    }
    if (a.gate_mode == GATE_GROUP && it.j == it.jn - 1) {
      if (a.slotwise) {  // this slot has its whole group: the sums are final
        if (on) {
          t.set(agt);
          store8<ALN>(t, a.dgate, it.g, C, c0, nv);
        }
      } else if (a.sub > 1) {
        flush_cols<LPR, NT>(agt, cols, tid, tpr, C, a.gpart + it.item * C);
      } else {
        flush_cols<LPR, NT>(agt, cols, tid, tpr, C, (T*)a.dgate + it.item * C);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) agt[j] = 0.f;
    }
    it.next(a, slot, slots);
  }
  // partial column sums: [vector][workgroup][C], vectors in the order dgamma2, dbeta2, dgamma1,
  // dbeta1, dgate as far as they are there (nvec)
  const long wg = (long)gridDim.x * C;
  float* p = a.part + (long)blockIdx.x * C;
  if (PR) {
    flush_cols<LPR, NT>(ag2, cols, tid, tpr, C, p);
    p += wg;
    if (a.kind2 == NORM_LAYER) { flush_cols<LPR, NT>(ab2, cols, tid, tpr, C, p); p += wg; }
  }
  if (PO && a.kind1) {
    flush_cols<LPR, NT>(ag1, cols, tid, tpr, C, p);
    p += wg;
    if (a.kind1 == NORM_LAYER) { flush_cols<LPR, NT>(ab1, cols, tid, tpr, C, p); p += wg; }
  }
  if (a.gate_mode == GATE_VEC) flush_cols<LPR, NT>(agt, cols, tid, tpr, C, p);
}

// Sums of up to 5 [rows][C] matrices over their rows, in a fixed order: 32 columns and 32 strips of
// rows a workgroup.  A gradient that is not asked for has a null destination.
struct ColSums {
  const float* src;
  float* dst[5];
};
__global__ __launch_bounds__(1024) void col_sums_k(ColSums a, int rows, int C) {
  __shared__ float s[32][33];
  if (!a.dst[blockIdx.y]) return;
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  const float* p = a.src + (long)blockIdx.y * rows * C;
  float v = 0.f;
  if (c < C)
    for (int r = k; r < rows; r += 32) v += p[(long)r * C + c];
  s[k][threadIdx.x & 31] = v;
  __syncthreads();
  if (k == 0 && c < C) {
    v = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) v += s[r][threadIdx.x];
    a.dst[blockIdx.y][c] = v;
  }
}
// dgate[g][c] = sum of the `sub` partial rows of group g
template <typename T>
__global__ __launch_bounds__(256) void gate_sums_k(const float* src, T* dst, long n, int C, int sub) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long g = i / C;
  const float* p = src + g * sub * C + (i - g * C);
  float v = 0.f;
  for (int k = 0; k < sub; ++k) v += p[(long)k * C];
  if constexpr (sizeof(T) == 2) dst[i] = f2bf(v);
  else dst[i] = v;
}

namespace {

constexpr int BWD_WGS = 512;  // workgroups of a backward pass at most: rows of its partial sums

struct Shape { int lpr, nt, tpr; };
Shape shape_of(int C) {
  if (C <= 16) return {2, 256, 2};
  if (C <= 64) return {8, 256, 8};
  if (C <= 256) return {32, 256, 32};
  if (C <= 512) return {64, 256, 64};
  if (C <= 1024) return {64, 256, 128};
  if (C <= 2048) return {64, 256, 256};
  if (C <= 4096) return {64, 512, 512};
  return {64, 1024, 1024};
}
// Work items: bundles of `slots` groups while groups are short; a long group is an item of its own, or
// is split (`sub`) where there are too few groups to fill the workgroups.
void plan(BlkArgs& a, const Shape& s, int& grid) {
  const long slots = s.nt / s.tpr, G = a.M / a.rpg;
  a.slotwise = a.rpg <= 4 * slots || a.rpg <= 16;
  a.sub = 1;
  if (a.slotwise) {
    a.items = (G + slots - 1) / slots;
  } else {
    const long want = BWD_WGS / (G < BWD_WGS ? G : BWD_WGS), most = a.rpg / (4 * slots);
    a.sub = (int)(want < most ? want : most);
    if (a.sub < 1) a.sub = 1;
    a.items = G * a.sub;
  }
  grid = (int)(a.items < BWD_WGS ? a.items : BWD_WGS);
}

template <typename T, bool ALN, bool PO, bool PR>
void bwd_go(const BlkArgs& a, const Shape& s, int grid, hipStream_t st) {
  if (s.lpr == 2) block_norm_bwd_k<T, 2, 256, ALN, PO, PR><<<grid, 256, 0, st>>>(a);
  else if (s.lpr == 8) block_norm_bwd_k<T, 8, 256, ALN, PO, PR><<<grid, 256, 0, st>>>(a);
  else if (s.lpr == 32) block_norm_bwd_k<T, 32, 256, ALN, PO, PR><<<grid, 256, 0, st>>>(a);
  else if (s.nt == 256) block_norm_bwd_k<T, 64, 256, ALN, PO, PR><<<grid, 256, 0, st>>>(a);
  else if (s.nt == 512) block_norm_bwd_k<T, 64, 512, ALN, PO, PR><<<grid, 512, 0, st>>>(a);
  else block_norm_bwd_k<T, 64, 1024, ALN, PO, PR><<<grid, 1024, 0, st>>>(a);
}
template <typename T, bool ALN>
void bwd_kind(const BlkArgs& a, const Shape& s, int grid, hipStream_t st) {
  if (!a.kind2) bwd_go<T, ALN, true, false>(a, s, grid, st);
  else if (!a.kind1) bwd_go<T, ALN, false, true>(a, s, grid, st);
  else bwd_go<T, ALN, true, true>(a, s, grid, st);
}

}  // namespace

extern "C" {

// *floats: the workspace that a backward pass of these sizes takes at most (any kinds, any gate).
int ptg_block_norm_ws(long M, int C, long groups, void* floats) {
  *(long*)floats = 0;
  if (M <= 0 || C < 1 || C > 8192 || groups < 1 || M % groups) return 0;
  BlkArgs a{};
  a.M = M; a.C = C; a.rpg = M / groups;
  int grid;
  const Shape s = shape_of(C);
  plan(a, s, grid);
  const long split = a.sub > 1 ? a.items : 0;
  long wgs = grid;
  a.rpg = 1;  // a gate vector or no gate
  plan(a, s, grid);
  if (grid > wgs) wgs = grid;
  *(long*)floats = (5 * wgs + split) * C;
  return 0;
}

int ptg_block_norm_bwd(const void* x, const void* res, const void* gate, const void* du, const void* dh, void* dx,
                       void* dres, const void* g1, const void* b1, const void* g2, const void* stats, void* dg1,
                       void* db1, void* dg2, void* db2, void* dgate, void* ws, long M, int C, int f32, int aligned,
                       int kind1, int kind2, int gate_mode, long rpg, float scale, int drop, int thr, float dscale,
                       long seed, long step, const void* step_dev, hipStream_t stream) {
  if (M <= 0) return 0;
  if (C < 1 || C > 8192 || (gate_mode == GATE_GROUP && (rpg < 1 || M % rpg))) return (int)hipErrorInvalidValue;
  BlkArgs a{};
  a.x = x; a.res = res; a.gate = gate; a.du = du; a.dh = dh; a.dx = dx; a.dres = dres;
  a.g1 = (const float*)g1; a.b1 = (const float*)b1; a.g2 = (const float*)g2;
  a.stats = (float*)stats;
  a.M = M; a.C = C; a.kind1 = kind1; a.kind2 = kind2;
  a.gate_mode = gate_mode; a.rpg = gate_mode == GATE_GROUP ? rpg : 1; a.scale = scale; a.drop = drop;
  a.d = drop_args(thr, dscale, seed, step, step_dev);
  a.dgate = dgate;
  const Shape s = shape_of(C);
  int grid;
  plan(a, s, grid);
  a.tpr = s.tpr;
  ColSums cs{};
  if (kind2) {
    cs.dst[a.nvec++] = (float*)dg2;
    if (kind2 == NORM_LAYER) cs.dst[a.nvec++] = (float*)db2;
  }
  if (kind1) {
    cs.dst[a.nvec++] = (float*)dg1;
    if (kind1 == NORM_LAYER) cs.dst[a.nvec++] = (float*)db1;
  }
  if (gate_mode == GATE_VEC) cs.dst[a.nvec++] = (float*)dgate;
  a.part = (float*)ws;
  a.gpart = (float*)ws + (long)a.nvec * grid * C;
  cs.src = a.part;
  if (f32) { if (aligned) bwd_kind<float, true>(a, s, grid, stream); else bwd_kind<float, false>(a, s, grid, stream); }
  else { if (aligned) bwd_kind<bf16_t, true>(a, s, grid, stream); else bwd_kind<bf16_t, false>(a, s, grid, stream); }
  if (a.nvec) col_sums_k<<<dim3((C + 31) / 32, a.nvec), 1024, 0, stream>>>(cs, grid, C);
  if (gate_mode == GATE_GROUP && a.sub > 1) {
    const long n = (M / rpg) * C;
    const int blocks = (int)((n + 255) / 256);
    if (f32) gate_sums_k<float><<<blocks, 256, 0, stream>>>(a.gpart, (float*)dgate, n, C, a.sub);
    else gate_sums_k<bf16_t><<<blocks, 256, 0, stream>>>(a.gpart, (bf16_t*)dgate, n, C, a.sub);
  }
  PTG_RETURN_LAUNCH();
}

}  // extern "C"
