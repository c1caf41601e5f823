// Block norm, backward (norm.h).  From du = dL/du and dh = dL/dh (the residual stream's gradient):
//
//   dh' = dh + pre'(du)       pre'(g) = rstd * (g*gamma - mean(g*gamma) [layer] - xhat * mean(g*gamma*xhat))
//   dres = dh';  dd = mask(dh') * dscale;  dgate = sum scale * post(x) * dd
//   dx = post'(scale * gate * dd);  dgamma = sum g * xhat;  dbeta = sum g      for both norms
//
// h and post(x) are computed again from x and res (and the mask drawn again), in fp32: the pass reads
// du, dh, x, res and writes dx, dres, each once, and h need not be kept.  Column sums stay in registers
// over all rows of a workgroup, are joined over its rows in LDS, and a second kernel adds the
// workgroups' partial sums in a fixed order: no atomics, the same bits every run.  As in the forward pass
// the next row's loads are in flight while a row is worked on.
//
// Bound by HBM where it has rows enough (32768 x 2048 bf16: 155 to 159 us, 5.1 TB/s).  On the way there a wave sees few
// rows, so its start (vectors to LDS, first loads) and its end (five vectors joined) weigh as much as the rows: 4096 x
// 1024 with both norms, gate and dropout, 4 rows a wave, takes 17.8 us, in which the vector pipes are 52 % busy
// and the waves wait for 46 % of their time; 1537 x 771 fp32 with 53 gate rows, 2 rows a wave, 15.2 us, 33 % and 54 %.
// Rows above 2048 columns take 16 waves of 128 registers, which are too few: 34 of the 48 such variants spill, up to
// 89 registers with both norms (4096 x 8192 with all parts: bf16 173 us, 2.3 TB/s, fp32 332 us, 2.4 TB/s).
#include "norm.h"

// A thread's column sums over the rows (slots) of the workgroup: put_cols leaves them in LDS, [rows][cols]
// (col_floats in all), and sum_cols adds dst[0..C) up after a barrier.
template <int LPR, int NT>
PTG_DEV int col_rows(int tpr) { return LPR < 64 ? NT / 64 : NT / tpr; }
template <int LPR, int NT>
constexpr int col_floats() { return LPR < 64 ? NT / 64 * LPR * 8 : NT * 8; }
template <int LPR, int NT>
PTG_DEV void put_cols(float* acc, float* lds, int tid, float mul) {
  if (LPR < 64) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) acc[j] += __shfl_xor(acc[j], o, 64);
    }
  }
  if (LPR == 64 || (tid & 63) < LPR) {
    float* p = lds + (LPR < 64 ? (tid >> 6) * LPR * 8 + (tid & 63) * 8 : tid * 8);
    *(float4*)p = make_float4(acc[0] * mul, acc[1] * mul, acc[2] * mul, acc[3] * mul);
    *(float4*)(p + 4) = make_float4(acc[4] * mul, acc[5] * mul, acc[6] * mul, acc[7] * mul);
  }
}
template <int LPR, int NT, typename D>
PTG_DEV void sum_cols(const float* lds, int tid, int tpr, int C, D* dst) {
  const int rows = col_rows<LPR, NT>(tpr), cols = LPR < 64 ? LPR * 8 : tpr * 8;
  for (int c = tid; c < C; c += NT) {
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += lds[r * cols + c];
    if constexpr (sizeof(D) == 2) dst[c] = f2bf(s);
    else dst[c] = s;
  }
}
// vectors joined at a time at the end; 16-wave workgroups join them in the place of the column vectors too
template <int NT>
constexpr int flush_vecs() { return NT <= 512 ? 5 : 3; }

template <typename T>
struct RowIn {  // a row on its way in
  Raw8<T> x, r, gu, gh;
  float m1, s1, m2, s2;
};
template <bool PO, bool PR, typename T, typename L>
PTG_DEV void load_row(RowIn<T>& in, const BlkArgs& a, const L& ln, long base, uint32_t rows, bool on) {
  const long at = base * a.C;
  ln.load(in.x, a.x, at, rows, a.C, on);
  if (PR) ln.load(in.r, a.res, at, rows, a.C, on);
  if (PR) ln.load(in.gu, a.du, at, rows, a.C, on);
  ln.load(in.gh, a.dh, at, rows, a.C, on);
  // a row that does not exist, and a lane without columns, take 0 for 1/std: nothing of theirs counts
  auto stat = [&](int k) {
    return __uint_as_float(bload4(make_rsrc(a.stats + k * a.M + base, rows * 4), ln.soff));
  };
  if (PO) {
    in.m1 = a.kind1 ? stat(0) : 0.f;
    in.s1 = a.kind1 ? stat(1) : 1.f;
  }
  if (PR) {
    in.m2 = stat(2);
    in.s2 = stat(3);
  }
}

template <typename T, int LPR, int NT, bool ALN, bool PO, bool PR, bool GG, bool DROP>
__global__ __launch_bounds__(NT, 2) void block_norm_bwd_k(BlkArgs a) {
  __shared__ float2 xch[2 * (NT / 64)];
  extern __shared__ float4 dyn[];
  float* vecs = (float*)dyn;  // column vectors, then [NT * 8] of the joins
  const int tid = threadIdx.x, tpr = LPR < 64 ? LPR : a.tpr, slots = NT / tpr, slot = tid / tpr;
  const int C = a.C, c0 = (tid % tpr) * 8, lag = RowIter<GG>::lag(a, slot);
  const Lane<T, ALN, LPR == 2> ln(lag, c0, C);
  const int nv = ln.nv, cc = nv ? c0 : 0;
  RowX rx;
  rx.init(xch, tid, NT, LPR, tpr, C);
  const uint64_t step = DROP ? drop_step(a.d) : 0;
  RowIn<T> in;
  RowIter<GG> it;
  it.item = blockIdx.x;
  it.enter(a, slots);
  uint32_t rows = it.rows(a, slots);
  bool on = lag < (int)rows && nv > 0;
  load_row<PO, PR>(in, a, ln, it.base, rows, on);
  ColVecs<NT, 4> cv;
  enum { G1, B1, G2, GV };
  cv.v[G1] = {PO ? a.g1 : nullptr, 1.f, 1.f};
  cv.v[B1] = {PO ? a.b1 : nullptr, 0.f, 1.f};
  cv.v[G2] = {PR ? a.g2 : nullptr, 1.f, 1.f};
  const float fs = DROP ? a.scale * a.d.scale : a.scale;  // scale and keep scale, times the gate: gt
  cv.v[GV] = {a.gate_mode == GATE_VEC ? (const float*)a.gate : nullptr, 1.f, fs};
  cv.init(vecs, C, tid, a.vecs);
  float* cols = vecs + a.vecs;
  float ag1[8], ab1[8], ag2[8], ab2[8], agt[8], gt[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) { ag1[j] = 0.f; ab1[j] = 0.f; ag2[j] = 0.f; ab2[j] = 0.f; agt[j] = 0.f; gt[j] = fs; }
  // the sums' shares: mean(g) of a LayerNorm only, mean(g * xhat) of a norm only
  const float p1 = a.kind1 == NORM_LAYER ? rx.invC : 0.f, q1 = a.kind1 ? rx.invC : 0.f;
  const float p2 = a.kind2 == NORM_LAYER ? rx.invC : 0.f;
  __syncthreads();
  while (it.item < a.items) {
    asm volatile("" ::: "memory");  // keeps the column vectors in LDS: hoisted, they cost 32 registers
    const long at = it.base * C, g = it.g, item = it.item;
    const uint32_t crows = rows;
    const bool con = on, first = it.j == 0, last = it.j == it.jn - 1;
    float xh[8], r[8], gu[8], gh[8], n[8], v[8];
    bool keep[8];
    ln.get(in.x, xh, on);
    if (PR) ln.get(in.r, r, on);
    if (PR) ln.get(in.gu, gu, on);
    ln.get(in.gh, gh, on);
    const float m1 = in.m1, s1 = in.s1, m2 = in.m2, s2 = in.s2;
    it.next(a, slots);
    rows = it.item < a.items ? it.rows(a, slots) : 0;
    on = lag < (int)rows && nv > 0;
    load_row<PO, PR>(in, a, ln, it.base, rows, on);
    if (DROP) row_keep<ALN>(a, step, at, ln.off, keep);
    Raw8<T> t;
    const Lane<T, false, LPR == 2> gl(0, c0, C);
    if (GG && first) {
      gl.load(t, a.gate, (g + (a.slotwise ? slot : 0)) * C, 0, C, con);
      gl.get(t, gt, con);
#pragma unroll
      for (int j = 0; j < 8; ++j) gt[j] *= fs;
    }
    if (PO) {
      float b[8];
      cv.get(vecs, G1, v, cc, nv);
      cv.get(vecs, B1, b, cc, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[j] = (xh[j] - m1) * s1;
        n[j] = fmaf(xh[j], v[j], b[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] = xh[j];
    }
    if (!GG) cv.get(vecs, GV, gt, cc, nv);
    if (PR) {
      float c1 = 0.f, c2 = 0.f;
      cv.get(vecs, G2, v, cc, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float k = n[j] * gt[j];
        r[j] = (r[j] + (!DROP || keep[j] ? k : 0.f) - m2) * s2;  // xhat of h
        if (!ALN) r[j] = j < nv ? r[j] : 0.f;
        ag2[j] = fmaf(gu[j], r[j], ag2[j]);
        ab2[j] += gu[j];
        gu[j] *= v[j];
        c1 += gu[j];
        c2 = fmaf(gu[j], r[j], c2);
      }
      const float2 c = row_sum2<LPR>(make_float2(c1, c2), rx);
      const float k1 = c.x * p2, k2 = c.y * rx.invC;
#pragma unroll
      for (int j = 0; j < 8; ++j) gh[j] = fmaf(s2, gu[j] - fmaf(r[j], k2, k1), gh[j]);
    }
    meet<LPR, ALN>(a, PR);
    if (a.dres) {
      t.set(gh);
      ln.store(t, a.dres, at, crows, C, con);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float dd = !DROP || keep[j] ? gh[j] : 0.f;  // times fs: in gt, and in agt where it is flushed
      agt[j] = fmaf(dd, n[j], agt[j]);
      gh[j] = dd * gt[j];
    }
    if (PO) {
      float c1 = 0.f, c2 = 0.f;
      cv.get(vecs, G1, v, cc, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ag1[j] = fmaf(gh[j], xh[j], ag1[j]);
        ab1[j] += gh[j];
        gh[j] *= v[j];
        if (!ALN) gh[j] = j < nv ? gh[j] : 0.f;
        c1 += gh[j];
        c2 = fmaf(gh[j], xh[j], c2);
      }
      const float2 c = row_sum2<LPR>(make_float2(c1, c2), rx);
      const float k1 = c.x * p1, k2 = c.y * q1;
#pragma unroll
      for (int j = 0; j < 8; ++j) gh[j] = fmaf(xh[j], -s1 * k2, fmaf(gh[j], s1, -s1 * k1));
    }
    if (a.dx) {
      t.set(gh);
      ln.store(t, a.dx, at, crows, C, con);
    }
    if (GG && last) {
      if (a.slotwise) {  // this slot has its whole group: the sums are final
#pragma unroll
        for (int j = 0; j < 8; ++j) agt[j] *= fs;
        t.set(agt);
        gl.store(t, a.dgate, (g + slot) * C, 0, C, con);
      } else {
        __syncthreads();
        put_cols<LPR, NT>(agt, cols, tid, fs);
        __syncthreads();
        if (a.sub > 1) sum_cols<LPR, NT>(cols, tid, tpr, C, a.gpart + item * C);
        else sum_cols<LPR, NT>(cols, tid, tpr, C, (T*)a.dgate + item * C);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) agt[j] = 0.f;
    }
  }
  // partial column sums: [vector][workgroup][C], vectors in the order dgamma2, dbeta2, dgamma1,
  // dbeta1, dgate as far as they are there (nvec)
  float* p = a.part + (long)blockIdx.x * C;
  int v = 0;
  // 4 columns of one vector a thread, all vectors at once
  auto drain = [&] {
    __syncthreads();
    const int quads = (C + 3) >> 2, jrows = col_rows<LPR, NT>(tpr), jcols = LPR < 64 ? LPR * 8 : tpr * 8;
    for (int e = tid; e < v * quads; e += NT) {
      const int k = e / quads, c = (e - k * quads) * 4;
      const float* q = cols + k * col_floats<LPR, NT>() + c;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int r = 0; r < jrows; ++r) {
        const float4 t = *(const float4*)(q + r * jcols);
        s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
      }
      float* o = p + (long)k * gridDim.x * C + c;
      if (c + 4 <= C) {
        __builtin_memcpy(o, &s, 16);
      } else {
        const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < C) o[j] = f[j];
      }
    }
    p += (long)v * gridDim.x * C;
    v = 0;
  };
  auto flush = [&](float* acc, float mul) {
    if (v == flush_vecs<NT>()) {
      drain();
      __syncthreads();
    }
    put_cols<LPR, NT>(acc, cols + v++ * col_floats<LPR, NT>(), tid, mul);
  };
  __syncthreads();
  if (NT > 512) cols = vecs;  // no longer needed
  if (PR) {
    flush(ag2, 1.f);
    if (a.kind2 == NORM_LAYER) flush(ab2, 1.f);
  }
  if (PO && a.kind1) {
    flush(ag1, 1.f);
    if (a.kind1 == NORM_LAYER) flush(ab1, 1.f);
  }
  if (a.gate_mode == GATE_VEC) flush(agt, fs);
  drain();
}

// The sums of the workgroups' parts, in a fixed order.  First `cblocks` workgroups a vector: sums of up to
// 5 [rows][C] matrices over their rows, 32 columns and 32 strips of rows a workgroup (a gradient that is
// not asked for has a null destination).  Then dgate[g][c] = sum of the `sub` partial rows of group g.
struct ColSums {
  const float* src;
  float* dst[5];
  const float* gsrc;
  void* gdst;
  long gn;
  int rows, C, cblocks, nvec, sub;
};
template <typename T>
__global__ __launch_bounds__(1024) void col_sums_k(ColSums a) {
  __shared__ float s[32][33];
  const int C = a.C;
  if ((int)blockIdx.x >= a.cblocks * a.nvec) {
    const long i = (long)(blockIdx.x - a.cblocks * a.nvec) * 1024 + threadIdx.x;
    if (i >= a.gn) return;
    const long g = i / C;
    const float* p = a.gsrc + g * a.sub * C + (i - g * C);
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < a.sub; ++k) v += p[(long)k * C];
    if constexpr (sizeof(T) == 2) ((T*)a.gdst)[i] = f2bf(v);
    else ((T*)a.gdst)[i] = v;
    return;
  }
  const int y = blockIdx.x / a.cblocks;
  if (!a.dst[y]) return;
  const int c = (blockIdx.x - y * a.cblocks) * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  const float* p = a.src + (long)y * a.rows * C;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int r = k; r < a.rows; r += 32) v += p[(long)r * C + c];
  }
  s[k][threadIdx.x & 31] = v;
  __syncthreads();
  if (k == 0 && c < C) {
    v = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) v += s[r][threadIdx.x];
    a.dst[y][c] = v;
  }
}

namespace {

constexpr int BWD_WGS = 256;  // workgroups of a backward pass at most: rows of its partial sums

struct Shape { int lpr, nt, tpr; };
Shape shape_of(int C) {
  if (C <= 16) return {2, 512, 2};
  if (C <= 64) return {8, 512, 8};
  if (C <= 256) return {32, 512, 32};
  if (C <= 512) return {64, 512, 64};
  if (C <= 1024) return {64, 512, 128};
  if (C <= 2048) return {64, 512, 256};
  return {64, 1024, C <= 4096 ? 512 : 1024};
}
// Work items: bundles of `slots` groups, each slot going through a group of its own; or a long group is an
// item whose rows the slots share, split (`sub`) where there are too few groups to fill the workgroups.
// The fewer rows one after another win; an item of shared rows ends in a join, worth about two rows (62 x 24, one
// group: 90 us as 62 rows of one slot).  Slots of long groups would stand too far apart for 32-bit offsets.
void plan(BlkArgs& a, const Shape& s, int& grid) {
  const long slots = s.nt / s.tpr, G = a.M / a.rpg;
  auto up = [](long x, long y) { return (x + y - 1) / y; };
  const long want = BWD_WGS / (G < BWD_WGS ? G : BWD_WGS), most = a.rpg / slots;
  const long sub = most < 1 ? 1 : want < most ? want : most;
  const long own = up(up(G, slots), BWD_WGS) * a.rpg;
  const long shared = up(G * sub, BWD_WGS) * (up(up(a.rpg, sub), slots) + 2);
  a.slotwise = a.rpg <= (4 * slots > 16 ? 4 * slots : 16) && own <= shared;
  a.sub = a.slotwise ? 1 : (int)sub;
  a.items = a.slotwise ? up(G, slots) : G * sub;
  grid = (int)(a.items < BWD_WGS ? a.items : BWD_WGS);
}

template <typename T, int LPR, int NT, bool ALN, bool PO, bool PR, bool GG, bool DROP>
void bwd_run(const BlkArgs& a, int grid, hipStream_t st) {
  auto kern = block_norm_bwd_k<T, LPR, NT, ALN, PO, PR, GG, DROP>;
  const bool there[4] = {PO && a.g1, PO && a.b1, PR && a.g2, a.gate_mode == GATE_VEC};
  constexpr int one = col_floats<LPR, NT>() * 4;  // a vector's join
  const int vb = col_vec_bytes(NT, a.C, 4, there, VECS_MOST - one), fb = flush_vecs<NT>() * one;
  const int lds = NT <= 512 ? vb + fb : vb + one > fb ? vb + one : fb;
  BlkArgs b = a;
  b.vecs = vb / 4;
  static uint64_t set = 0;  // devices whose limit is raised
  if (LPR == 64) ptg_allow_lds((const void*)kern, VECS_MOST, set);
  kern<<<grid, NT, lds, st>>>(b);
}
template <typename T, bool ALN, bool PO, bool PR, bool GG, bool DROP>
void bwd_go(const BlkArgs& a, const Shape& s, int grid, hipStream_t st) {
  if (s.lpr == 2) bwd_run<T, 2, 512, ALN, PO, PR, GG, DROP>(a, grid, st);
  else if (s.lpr == 8) bwd_run<T, 8, 512, ALN, PO, PR, GG, DROP>(a, grid, st);
  else if (s.lpr == 32) bwd_run<T, 32, 512, ALN, PO, PR, GG, DROP>(a, grid, st);
  else if (s.nt == 512) bwd_run<T, 64, 512, ALN, PO, PR, GG, DROP>(a, grid, st);
  else bwd_run<T, 64, 1024, ALN, PO, PR, GG, DROP>(a, grid, st);
}
// no norm at all: the post-norm kernel, whose kind1 == 0 is the identity
template <typename T, bool ALN, bool GG, bool DROP>
void bwd_kind(const BlkArgs& a, const Shape& s, int grid, hipStream_t st) {
  if (!a.kind2) bwd_go<T, ALN, true, false, GG, DROP>(a, s, grid, st);
  else if (!a.kind1) bwd_go<T, ALN, false, true, GG, DROP>(a, s, grid, st);
  else bwd_go<T, ALN, true, true, GG, DROP>(a, s, grid, st);
}
template <typename T, bool ALN>
void bwd_mode(const BlkArgs& a, const Shape& s, int grid, hipStream_t st) {
  if (a.gate_mode == GATE_GROUP) {
    if (a.drop) bwd_kind<T, ALN, true, true>(a, s, grid, st);
    else bwd_kind<T, ALN, true, false>(a, s, grid, st);
  } else {
    if (a.drop) bwd_kind<T, ALN, false, true>(a, s, grid, st);
    else bwd_kind<T, ALN, false, false>(a, s, grid, st);
  }
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

// call: a BwdCall, `aligned` and `rpg` as in the forward pass
int ptg_block_norm_bwd(const void* call, hipStream_t stream) {
  const BwdCall& c = *(const BwdCall*)call;
  const long M = c.M, rpg = c.rpg;
  const int C = (int)c.C, kind1 = (int)c.kind1, kind2 = (int)c.kind2, gate_mode = (int)c.gate_mode;
  const bool f32 = c.f32, aligned = c.aligned;
  float *dg1 = c.dg1, *db1 = c.db1, *dg2 = c.dg2, *db2 = c.db2;
  void *dgate = c.dgate, *ws = c.ws;
  if (M <= 0) return 0;
  if (c.C < 1 || c.C > 8192 || (gate_mode == GATE_GROUP && (rpg < 1 || M % rpg))) return (int)hipErrorInvalidValue;
  BlkArgs a{};
  a.x = c.x; a.res = c.res; a.gate = c.gate; a.du = c.du; a.dh = c.dh; a.dx = c.dx; a.dres = c.dres;
  a.g1 = c.g1; a.b1 = c.b1; a.g2 = c.g2;
  a.stats = c.stats;
  a.M = M; a.C = C; a.kind1 = kind1; a.kind2 = kind2;
  a.gate_mode = gate_mode; a.rpg = gate_mode == GATE_GROUP ? rpg : 1; a.scale = (float)c.scale; a.drop = (int)c.drop;
  a.d = drop_args((int)c.thr, (float)c.dscale, c.seed, c.step, c.step_dev, c.first);
  a.dgate = dgate;
  auto over = [&](const void* o) { return o && (o == c.x || o == c.res || o == c.du || o == c.dh); };
  a.over = !aligned && (over(c.dx) || over(c.dres));
  const Shape s = shape_of(C);
  int grid;
  plan(a, s, grid);
  a.tpr = s.tpr;
  ColSums cs{};
  if (kind2) {
    cs.dst[a.nvec++] = dg2;
    if (kind2 == NORM_LAYER) cs.dst[a.nvec++] = db2;
  }
  if (kind1) {
    cs.dst[a.nvec++] = dg1;
    if (kind1 == NORM_LAYER) cs.dst[a.nvec++] = db1;
  }
  if (gate_mode == GATE_VEC) cs.dst[a.nvec++] = (float*)dgate;
  a.part = (float*)ws;
  a.gpart = (float*)ws + (long)a.nvec * grid * C;
  cs.src = a.part;
  if (f32) { if (aligned) bwd_mode<float, true>(a, s, grid, stream); else bwd_mode<float, false>(a, s, grid, stream); }
  else { if (aligned) bwd_mode<bf16_t, true>(a, s, grid, stream); else bwd_mode<bf16_t, false>(a, s, grid, stream); }
  cs.rows = grid; cs.C = C; cs.nvec = a.nvec; cs.cblocks = (C + 31) / 32;
  if (gate_mode == GATE_GROUP && a.sub > 1) {
    cs.gsrc = a.gpart; cs.gdst = dgate; cs.gn = (M / rpg) * C; cs.sub = a.sub;
  }
  const long blocks = (long)cs.cblocks * cs.nvec + (cs.gn + 1023) / 1024;
  if (blocks) {
    if (f32) col_sums_k<float><<<(int)blocks, 1024, 0, stream>>>(cs);
    else col_sums_k<bf16_t><<<(int)blocks, 1024, 0, stream>>>(cs);
  }
  PTG_RETURN_LAUNCH();
}

}  // extern "C"
