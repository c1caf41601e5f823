// Shared pieces of the block norm kernels (norm_fwd.hip, norm_bwd.hip).
//
//   d = drop(scale * gate * post(x));   h = res + d;   u = pre(h)        over rows of C columns
//
// post / pre: none, LayerNorm (mean and variance) or RMSNorm, with affine vectors.  A thread owns 8
// consecutive columns of a row for the whole kernel, so affine vectors are loaded once and column sums
// stay in registers.  A row takes LPR lanes of a wave (2, 8, 32), one wave, or 2..16 waves (C <= 8192),
// and a workgroup works on NT / (threads of a row) rows at a time.
#pragma once
#include "rng.h"

enum { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
enum { GATE_NONE = 0, GATE_VEC = 1, GATE_GROUP = 2 };

struct BlkArgs {
  const void *x, *res, *du, *dh, *gate;
  void *h, *u, *dx, *dres;
  const float *g1, *b1, *g2, *b2;
  float* stats;  // [4][M]: mean and 1/std of x, mean and 1/std of h
  float* part;   // backward: column sums, [vector][workgroup][C]
  void* dgate;   // GATE_GROUP: [G][C] in the tensors' type
  float* gpart;  // GATE_GROUP with groups split over workgroups: [item][C]
  int kind1, kind2, gate_mode, drop;
  float eps1, eps2, scale;
  DropArgs d;
  long M, rpg, items;  // rows per gate group; work items (see RowIter)
  int C, tpr, slotwise, sub, nvec;
};

// ---- sums over the LPR lanes of a row (every lane gets the sum) --------------------------------
template <int CTRL>
PTG_DEV float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int LPR>
PTG_DEV float lanes_sum(float v) {
  v = dpp_add<0xB1>(v);                    // lane ^ 1
  if (LPR >= 4) v = dpp_add<0x4E>(v);      // lane ^ 2
  if (LPR >= 8) v = dpp_add<0x141>(v);     // mirrored within 8: the other quad
  if (LPR >= 16) v = dpp_add<0x140>(v);    // mirrored within 16: the other 8
  if (LPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (LPR >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sums of two values over a row of `tpr` threads.  Rows of several waves meet in LDS; `phase`
// alternates between two buffers, so one barrier an exchange is enough: a buffer is written again
// only after the barrier of the exchange in between.
struct RowX {
  float2* lds;  // [2][NT / 64]
  int phase, w, nw, w0, wper;  // wave, waves of the workgroup, first wave of this row, waves of a row
  PTG_DEV float2* put(float2 v) {
    float2* buf = lds + (phase & 1) * nw;
    ++phase;
    if ((threadIdx.x & 63) == 0) buf[w] = v;
    __syncthreads();
    return buf + w0;
  }
};
template <int LPR>
PTG_DEV float2 row_sum2(float2 v, RowX& rx) {
  v.x = lanes_sum<LPR>(v.x);
  v.y = lanes_sum<LPR>(v.y);
  if (LPR == 64 && rx.wper > 1) {
    const float2* p = rx.put(v);
    v = make_float2(0.f, 0.f);
    for (int k = 0; k < rx.wper; ++k) { v.x += p[k].x; v.y += p[k].y; }
  }
  return v;
}

// Mean and 1/std of a row held 8 values a thread (`nv` of them real, the others 0).  LayerNorm takes
// the squared deviations from each wave's own mean and joins the waves by
//   M2 = sum_w M2_w + n_w * (mean_w - mean)^2
// so no sum of squares around zero cancels, whatever the row's offset; one exchange either way.
template <int LPR>
PTG_DEV void row_stats(const float* f, int nv, int C, int kind, float eps, RowX& rx, float& mean, float& rstd) {
  float s = 0.f, q = 0.f;
  if (kind == NORM_RMS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q = fmaf(f[j], f[j], q);
    mean = 0.f;
    rstd = rsqrtf(row_sum2<LPR>(make_float2(0.f, q), rx).y / (float)C + eps);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) s += f[j];
  s = lanes_sum<LPR>(s);
  const bool multi = LPR == 64 && rx.wper > 1;
  const int cw = multi ? min(max(C - (rx.w - rx.w0) * 512, 0), 512) : C;
  float m = cw > 0 ? s / (float)cw : 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e = f[j] - m;
    q = j < nv ? fmaf(e, e, q) : q;
  }
  q = lanes_sum<LPR>(q);
  if (multi) {
    const float2* p = rx.put(make_float2(m, q));
    m = 0.f;
    for (int k = 0; k < rx.wper; ++k) m = fmaf((float)min(max(C - k * 512, 0), 512), p[k].x, m);
    m /= (float)C;
    q = 0.f;
    for (int k = 0; k < rx.wper; ++k) {
      const float e = p[k].x - m;
      q += p[k].y + (float)min(max(C - k * 512, 0), 512) * e * e;
    }
  }
  mean = m;
  rstd = rsqrtf(q / (float)C + eps);
}

// ---- 8 consecutive values of a row ---------------------------------------------------------------
// ALN: 16-byte aligned and always whole.  Otherwise whole groups use unaligned vector accesses and the
// last group of a row goes value by value.
template <typename T> struct Raw8;
template <> struct Raw8<bf16_t> {
  U4 v;
  PTG_DEV void get(float* f) const { unpack8(v, f); }
  PTG_DEV void set(const float* f) { v = pack8(f); }
};
template <> struct Raw8<float> {
  float v[8];
  PTG_DEV void get(float* f) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v[j];
  }
  PTG_DEV void set(const float* f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[j];
  }
};
template <bool ALN, typename T>
PTG_DEV void load8(Raw8<T>& r, const void* base, long row, int C, int c0, int nv) {
  const T* p = (const T*)base + row * C + c0;
  if (ALN) {
    __builtin_memcpy(&r.v, __builtin_assume_aligned(p, 16), sizeof(r.v));
  } else if (nv == 8) {
    __builtin_memcpy(&r.v, p, sizeof(r.v));
  } else {
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = j < nv ? p[j] : (T)0;
    __builtin_memcpy(&r.v, t, sizeof(r.v));
  }
}
template <bool ALN, typename T>
PTG_DEV void store8(const Raw8<T>& r, void* base, long row, int C, int c0, int nv) {
  T* p = (T*)base + row * C + c0;
  if (ALN) {
    __builtin_memcpy(__builtin_assume_aligned(p, 16), &r.v, sizeof(r.v));
  } else if (nv == 8) {
    __builtin_memcpy(p, &r.v, sizeof(r.v));
  } else {
    T t[8];
    __builtin_memcpy(t, &r.v, sizeof(r.v));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < nv) p[j] = t[j];
  }
}
PTG_DEV void vec8(float* f, const float* p, int c0, int nv, float dflt) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = p && j < nv ? p[c0 + j] : dflt;
}

template <bool ALN>
PTG_DEV uint32_t row_keep(const BlkArgs& a, uint64_t step, long row, int c0) {
  const uint64_t i = (uint64_t)row * (uint64_t)a.C + (uint64_t)c0;
  return ALN ? keep8(philox(i >> 3, step, a.d.seed), a.d.thr) : keep8_at(i, step, a.d);
}

// ---- rows of a workgroup -------------------------------------------------------------------------
// A work item is a bundle of row groups, one for each slot (`slotwise`, groups of rpg rows; rpg = 1
// unless the gate has a row per group), or a part of one long group whose rows the slots share.
struct RowIter {
  long item;
  int j, jn;
  long g, r0, r1;
  PTG_DEV void enter(const BlkArgs& a, int slot, int slots) {
    j = 0;
    if (a.slotwise) {
      g = item * slots + slot;
      r0 = g * a.rpg;
      r1 = item < a.items && r0 < a.M ? r0 + a.rpg : r0;
      jn = (int)a.rpg;
    } else {
      g = item / a.sub;
      const long len = (a.rpg + a.sub - 1) / a.sub, k = item - g * a.sub;
      r0 = g * a.rpg + k * len + slot;
      r1 = item < a.items ? min(g * a.rpg + (k + 1) * len, (g + 1) * a.rpg) : r0;
      jn = (int)((len + slots - 1) / slots);
    }
  }
  PTG_DEV long row(const BlkArgs& a, int slots) const { return r0 + (a.slotwise ? (long)j : (long)j * slots); }
  PTG_DEV bool valid(const BlkArgs& a, int slots) const { return row(a, slots) < r1; }
  PTG_DEV void next(const BlkArgs& a, int slot, int slots) {
    if (++j >= jn) {
      item += gridDim.x;
      enter(a, slot, slots);
    }
  }
};
