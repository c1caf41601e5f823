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
  int vecs;  // floats of the column vectors in LDS (wide rows: 0 where they are read from L2)
  int over;  // an output lies on an input and rows are unaligned: see meet()
};

// Arguments of the C entries, one block of 64-bit fields (a call with as many arguments of its own costs the
// host about 2 us more).  Addresses of tensors that are not there are 0.
struct FwdCall {
  const void *x, *res, *gate;
  void *h, *u;
  const float *g1, *b1, *g2, *b2;
  float* stats;
  const void* step_dev;
  int64_t M, C, f32, aligned, kind1, kind2, gate_mode, rpg, drop, thr, seed, step, first;
  double eps1, eps2, scale, dscale;
};
struct BwdCall {
  const void *x, *res, *gate, *du, *dh;
  void *dx, *dres;
  const float *g1, *b1, *g2;
  float *stats, *dg1, *db1, *dg2, *db2;
  void* dgate;
  float* ws;
  const void* step_dev;
  int64_t M, C, f32, aligned, kind1, kind2, gate_mode, rpg, drop, thr, seed, step, first;
  double scale, dscale;
};
static_assert(sizeof(FwdCall) == 28 * 8 && sizeof(BwdCall) == 33 * 8, "64-bit fields");

typedef __attribute__((ext_vector_type(4))) unsigned int vu4_t;

// The last group of an unaligned row reads columns of the lane before it as well (Lane::load).  Those may belong to
// another wave, which must not write an output on top of them before they are read: where an output lies on an
// input the waves of a workgroup meet once a row, between its loads and its first store.  A kernel whose row sums
// come before that store (`summed`) has met there.
template <int LPR, bool ALN>
PTG_DEV void meet(const BlkArgs& a, bool summed) {
  if (LPR == 64 && !ALN && !summed && a.over) __syncthreads();
}

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

// Rows of several waves meet in LDS.  `phase` alternates between two buffers, so one barrier an exchange is
// enough: a buffer is written again only after the barrier of the exchange in between.  Every lane then
// takes the entry of wave (lane % waves of a row) and the 16 lanes of a DPP row add up, each wave counted
// 16 / waves times: no loop over the waves.
struct RowX {
  float2* lds;  // [2][NT / 64]
  int phase, w, nw, w0, wper;  // wave, waves of the workgroup, first wave of this row, waves of a row
  float invC, inv_cw;          // 1 / C; 1 / columns of this wave (of the row for LPR < 64)
  float rep, nk;               // waves of a row / 16; that times the columns of wave (lane % wper)
  PTG_DEV void init(float2* buf, int tid, int nt, int lpr, int tpr, int C) {
    lds = buf;
    phase = 0;
    w = __builtin_amdgcn_readfirstlane(tid >> 6);
    nw = nt / 64;
    wper = tpr >> 6;
    w0 = lpr < 64 ? 0 : __builtin_amdgcn_readfirstlane((tid / tpr) * wper);
    const bool multi = lpr == 64 && wper > 1;
    const int n = multi ? min(max(C - (w - w0) * 512, 0), 512) : C;
    invC = 1.f / (float)C;
    inv_cw = n > 0 ? 1.f / (float)n : 0.f;
    rep = (float)wper * 0.0625f;
    nk = multi ? (float)min(max(C - (tid & (wper - 1)) * 512, 0), 512) * rep : 0.f;
  }
  PTG_DEV float2 put(float2 v) {
    float2* buf = lds + (phase & 1) * nw;
    ++phase;
    if ((threadIdx.x & 63) == 0) buf[w] = v;
    __syncthreads();
    return buf[w0 + (threadIdx.x & (wper - 1))];
  }
};
template <int LPR>
PTG_DEV float2 row_sum2(float2 v, RowX& rx) {
  v.x = lanes_sum<LPR>(v.x);
  v.y = lanes_sum<LPR>(v.y);
  if (LPR == 64 && rx.wper > 1) {
    v = rx.put(v);
    v.x = lanes_sum<16>(v.x * rx.rep);
    v.y = lanes_sum<16>(v.y * rx.rep);
  }
  return v;
}

// Mean and 1/std of a row held 8 values a thread (`nv` of them real, the others 0).  The squared
// deviations are taken from each wave's own mean and joined by
//   M2 = sum_w M2_w + n_w * (mean_w - mean)^2
// so no sum of squares around zero cancels, whatever the row's offset; one exchange.  An RMSNorm (layer ==
// 0) is the same with every mean 0.
template <int LPR, bool ALN>
PTG_DEV void row_stats(const float* f, int nv, float layer, float eps, RowX& rx, float& mean, float& rstd) {
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += f[j];
  float m = lanes_sum<LPR>(s) * (rx.inv_cw * layer);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e = f[j] - m;
    q = ALN || j < nv ? fmaf(e, e, q) : q;
  }
  q = lanes_sum<LPR>(!ALN || nv ? q : 0.f);
  if (LPR == 64 && rx.wper > 1) {
    // a wave's own mean is rounded; the identity above holds for any value near it
    const float2 p = rx.put(make_float2(m, q));
    m = lanes_sum<16>(p.x * rx.nk) * rx.invC;
    const float e = p.x - m;
    q = lanes_sum<16>(fmaf(rx.nk * e, e, p.y * rx.rep));
  }
  mean = m;
  rstd = rsqrtf(q * rx.invC + eps);
}

// ---- 8 consecutive values of a row ---------------------------------------------------------------
// Aligned rows (ALN: 16-byte aligned, C % 8 == 0) go through buffer descriptors that stand at the
// workgroup's current rows: a lane's offset never changes, rows and columns that do not exist read 0 and
// are not written, and so does a tensor that is not there (0 bytes): no branch, no 64-bit arithmetic a
// lane.  Otherwise a group is one unaligned vector load as well: the last group of a row reads the row's
// last 8 values and is shifted down where it is used, a lane without columns or row reads the tensor's
// first 8 and takes 0.  A branch around the load would wait for it there and then (1537 x 771 fp32
// backward: 15.6 instead of 15.0 us).  Rows below 8 columns have no 8 values to read; they are among those of two
// lanes (TINY, up to 16 columns), which load value by value.
template <typename T> struct Raw8;
template <> struct Raw8<bf16_t> {
  U4 v;
  PTG_DEV void get(float* f) const { unpack8(v, f); }
  // drops the first n values, 0 follows
  PTG_DEV void shift(int n) {
    if (n & 4) { v.x = v.z; v.y = v.w; v.z = 0; v.w = 0; }
    if (n & 2) { v.x = v.y; v.y = v.z; v.z = v.w; v.w = 0; }
    if (n & 1) {
      v.x = (v.x >> 16) | (v.y << 16);
      v.y = (v.y >> 16) | (v.z << 16);
      v.z = (v.z >> 16) | (v.w << 16);
      v.w >>= 16;
    }
    if (n >= 8) v = zero4();
  }
  PTG_DEV void set(const float* f) { v = pack8(f); }
  PTG_DEV void load(Rsrc r, uint32_t off) { v = bload16(r, off); }
  PTG_DEV void store(Rsrc r, uint32_t off) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(vu4_t, v), r, off, 0, 0);
  }
};
template <> struct Raw8<float> {
  float v[8];
  PTG_DEV void get(float* f) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v[j];
  }
  PTG_DEV void shift(int n) {
#pragma unroll
    for (int b = 4; b; b >>= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = n & b ? (j + b < 8 ? v[j + b] : 0.f) : v[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = n >= 8 ? 0.f : v[j];
  }
  PTG_DEV void set(const float* f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[j];
  }
  PTG_DEV void load(Rsrc r, uint32_t off) {
    const U4 a = bload16(r, off), b = bload16(r, off + 16);
    __builtin_memcpy(v, &a, 16);
    __builtin_memcpy(v + 4, &b, 16);
  }
  PTG_DEV void store(Rsrc r, uint32_t off) const {
    vu4_t a, b;
    __builtin_memcpy(&a, v, 16);
    __builtin_memcpy(&b, v + 4, 16);
    __builtin_amdgcn_raw_buffer_store_b128(a, r, off, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(b, r, off + 16, 0, 0);
  }
};
// Where a lane stands: columns c0.. of the row `lag` rows behind the workgroup's base row.
template <typename T, bool ALN, bool TINY>
struct Lane {
  int nv;        // real values of its 8
  uint32_t off;  // elements from the base row's start
  uint32_t boff, soff;  // bytes for the descriptors: values, and a float of the row
  int back;             // unaligned: how far before `off` its 8 values are read
  PTG_DEV Lane(int lag, int c0, int C) {
    nv = ALN ? (c0 < C ? 8 : 0) : min(max(C - c0, 0), 8);
    off = (uint32_t)lag * C + c0;
    boff = nv ? off * (uint32_t)sizeof(T) : PTG_OOB;
    soff = nv ? (uint32_t)lag * 4 : PTG_OOB;
    back = 8 - nv;
  }
  // rows: how many rows from the base row on exist (at most as far as the lanes reach)
  PTG_DEV static Rsrc rsrc(const void* p, long at, uint32_t rows, int C) {
    return make_rsrc((const T*)p + at, p ? rows * (uint32_t)C * (uint32_t)sizeof(T) : 0u);
  }
  // on: there is such a row, and nv > 0.  What was loaded is taken with get().
  PTG_DEV void load(Raw8<T>& r, const void* base, long at, uint32_t rows, int C, bool on) const {
    if (ALN) {
      r.load(rsrc(base, at, rows, C), boff);
      return;
    }
    T t[8];
    if (!base) {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = (T)0;
    } else if (TINY) {
      const T* p = (const T*)base + (on ? at + off : 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = p[on ? min(j, nv - 1) : 0];
    } else {
      __builtin_memcpy(t, (const T*)base + (on ? at + off - back : 0), sizeof(t));
    }
    __builtin_memcpy(&r.v, t, sizeof(t));
  }
  PTG_DEV void get(const Raw8<T>& r, float* f, bool on) const {
    if (ALN) {
      r.get(f);
    } else if (TINY) {
      r.get(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = on && j < nv ? f[j] : 0.f;
    } else {
      const int n = on ? back : 8;
      Raw8<T> q = r;
      if (__ballot(n != 0)) q.shift(n);  // most waves have none
      q.get(f);
    }
  }
  PTG_DEV void store(const Raw8<T>& r, void* base, long at, uint32_t rows, int C, bool on) const {
    if (ALN) {
      r.store(rsrc(base, at, rows, C), boff);
    } else if (on && base) {
      T* p = (T*)base + at + off;
      if (nv == 8) {
        __builtin_memcpy(p, &r.v, sizeof(r.v));
      } else {
        T t[8];
        __builtin_memcpy(t, &r.v, sizeof(r.v));
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < nv) p[j] = t[j];
      }
    }
  }
};

// Column vectors (affine parameters, a gate row) are in LDS (dynamic, [vector][2][C/2 rounded up]), as two
// planes of 4 values a thread so that a wave reads 16 bytes a lane without bank conflicts: in registers they
// would cost up to 40 of the 128 that leave four waves a SIMD.  Rows of up to 2048 columns have a place for
// every vector; wider ones (NT = 1024) only for those that are there, and if those do not fit they are
// read from L2, a wait for each (3892 x 4520 pre-norm forward: 43.0 us from L2, 34.7 from LDS).
struct ColVec {
  const float* src;  // null: dflt everywhere
  float dflt;
  float mul;  // times this
};
template <int NT, int N>
struct ColVecs {
  static constexpr bool ALL = NT <= 512;
  ColVec v[N];
  int half, place[N];
  bool lds_on;
  // All vectors' loads are issued before the first store: one trip to memory, not one for each.
  PTG_DEV void init(float* lds, int C, int tid, bool on) {
    half = ((C + 7) & ~7) >> 1;
    lds_on = ALL || on;
    int used = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) place[k] = ALL ? k : v[k].src ? used++ : 0;
    if (!lds_on) return;
    for (int c = tid * 4; c < 2 * half; c += NT * 4) {
      float4 t[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        t[k] = make_float4(v[k].dflt, v[k].dflt, v[k].dflt, v[k].dflt);
        if (!v[k].src) continue;
        if (c + 4 <= C) {
          __builtin_memcpy(&t[k], v[k].src + c, 16);
        } else {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = c + j < C ? v[k].src[c + j] : v[k].dflt;
          t[k] = make_float4(e[0], e[1], e[2], e[3]);
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        t[k].x *= v[k].mul; t[k].y *= v[k].mul; t[k].z *= v[k].mul; t[k].w *= v[k].mul;
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (ALL || v[k].src) *(float4*)(lds + 2 * place[k] * half + ((c >> 2) & 1) * half + (c >> 3) * 4) = t[k];
    }
  }
  // c0 of a lane without columns: any that exist
  PTG_DEV void get(const float* lds, int k, float* f, int c0, int nv) const {
    if (ALL || (lds_on && v[k].src)) {
      const float* p = lds + 2 * place[k] * half + (c0 >> 1);
      const float4 a = *(const float4*)p, b = *(const float4*)(p + half);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else if (!v[k].src) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[k].dflt * v[k].mul;
    } else {
      if (nv == 8) {
        __builtin_memcpy(f, v[k].src + c0, 32);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = j < nv ? v[k].src[c0 + j] : v[k].dflt;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= v[k].mul;
    }
  }
};
constexpr int VECS_MOST = 128 * 1024;
// bytes of the vectors of a workgroup of nt threads; 0: read from L2 (more than `most`, or none there)
static inline int col_vec_bytes(int nt, int C, int n, const bool* there, int most) {
  const int one = ((C + 7) & ~7) * 4;
  if (nt <= 512) return n * one;
  int bytes = 0;
  for (int k = 0; k < n; ++k) bytes += there[k] ? one : 0;
  return bytes <= most ? bytes : 0;
}

template <bool ALN>
PTG_DEV void row_keep(const BlkArgs& a, uint64_t step, long at, uint32_t off, bool* k) {
  if (ALN) {
    keep8(philox((((uint64_t)at + a.d.first) >> 3) + (off >> 3), step, a.d.seed), a.d.thr, k);
  } else {
    const uint32_t b = keep8_at((uint64_t)at + a.d.first + off, step, a.d);
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = (b >> j) & 1u;
  }
}

// ---- rows of a workgroup -------------------------------------------------------------------------
// A work item is a bundle of rows, one for each slot; where the gate has a row per group (GG) a bundle of
// whole groups, one for each slot (`slotwise`), or a part of one long group whose rows the slots share.
// A slot stands at row base + lag, base being the same for the workgroup and lag never changing.
template <bool GG>
struct RowIter {
  long item, base, rem;  // rem: rows from base on that exist (slots with lag < rem have a row)
  long g;                // group of the item (slotwise: of slot 0)
  int j, jn;
  PTG_DEV static int lag(const BlkArgs& a, int slot) { return GG && a.slotwise ? slot * (int)a.rpg : slot; }
  // rows that the descriptors cover: as far as the last slot
  PTG_DEV uint32_t rows(const BlkArgs& a, int slots) const {
    const long reach = GG && a.slotwise ? (slots - 1) * a.rpg + 1 : slots;
    return (uint32_t)(rem < reach ? (rem > 0 ? rem : 0) : reach);
  }
  PTG_DEV void enter(const BlkArgs& a, int slots) {
    j = 0;
    if (!GG) {
      base = item * slots;
      rem = a.M - base;
      g = 0;
      jn = 1;
    } else if (a.slotwise) {
      g = item * slots;
      base = g * a.rpg;
      rem = a.M - base;
      jn = (int)a.rpg;
    } else {
      g = item / a.sub;
      const long len = (a.rpg + a.sub - 1) / a.sub, k = (item - g * a.sub) * len;
      base = g * a.rpg + k;
      rem = item < a.items ? min(len, a.rpg - k) : 0;
      jn = (int)((len + slots - 1) / slots);
    }
  }
  PTG_DEV void next(const BlkArgs& a, int slots) {
    if (GG && ++j < jn) {
      base += a.slotwise ? 1 : slots;
      rem -= a.slotwise ? 0 : slots;
    } else {
      item += gridDim.x;
      enter(a, slots);
    }
  }
};
