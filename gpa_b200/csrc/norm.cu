// Norms round a residual block (rows of `width` channels, all arithmetic in fp32):
//   u = y r_y wp           r_y = rsqrt(mean y^2 + eps)      (u = y without a post weight)
//   h' = h + c s(a) u      c: constant times an optional scale of every channel, s: sigmoid of an
//                          optional gate (one value per channel or one per row); h' is rounded
//                          once, to the stream's type
//   n  = h' r w            r = rsqrt(mean h'^2 + eps), from the rounded h'
// and, without a stream, n = y r w (plain RMS norm).  Backward, with G the gradient of h':
//   G  = dh' + r (w dn - h' r^2 mean(w dn h'))    dh = G      dw = sum_rows dn h' r
//   du = G c s     da = G c u s (1 - s)     dc = sum_rows G s u
//   dy = r_y (wp du - y r_y^2 mean(wp du y))      dwp = sum_rows du y r_y
// The statistics are formed again from the rows themselves, which the backward reads anyway.
//
// A group of G threads owns a row, each thread VEC consecutive channels at a time: sub-warp
// groups for narrow rows (several rows per warp), whole blocks for wide ones.  Rows are read
// once; the bound is the bytes moved.  Measured (GPU time, B200, copy 6.54 TB/s):
//   65536 x 1024, fp32 stream, bf16 update and result: forward 127 us = 6.3 TB/s, backward 163 us
//   (6.6), fold of the weight gradient 7 us;  262144 x 128 bf16, plain: 27 us (5.0) and 55 us (3.7);
//   8188 x 2560 bf16 with post weight, gate and scale: 61 us (3.4) and 96 us (3.5).
// Column sums of the backward stay in registers over a block's rows, go to one partial row per
// block and are added in block order by a second kernel, so results do not depend on scheduling.
#include "../../include/gpa_b200.h"
#include "common.cuh"
#include "norm.cuh"

#include <algorithm>
#include <atomic>

namespace gpa {
namespace {

struct Rows {  // row r of a strided [outer, inner, width] tensor, unit stride along the width
  int64_t so, si;
};

struct Fwd {
  const void *h, *y, *gate;
  const float *w, *wp, *scale;
  void *stream, *out;
  Rows rh, ry, rg;
  uint32_t rows, inner;
  int width, h_dt, y_dt, g_dt, out_dt, gate_full;
  float eps, c;
};

struct Bwd {
  Fwd f;                  // stream: the rounded h' of the forward (NULL for the plain norm)
  const void *dn, *ds;    // contiguous gradients of n and h' (either may be NULL)
  void *dh, *dy, *dgate;
  float *part;            // [blocks][sums][width], or NULL: one block, which writes the sums themselves
  float *sums_out[3];     // by slot
  int sum_w, sum_p, sum_c, sums;  // slot of dw / dwp / dc in a partial row, or -1
};

// 8 values as they lie in memory (one or two 16-byte loads), so that a load in flight holds few
// registers, and their conversion
struct Raw8 {
  uint4 a, b;
};
GPA_DEV Raw8 ldraw(const void* p, int64_t i, int dt) {
  Raw8 r;
  r.b = make_uint4(0, 0, 0, 0);
  if (dt == kF32) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
    r.a = q[0];
    r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
  }
  return r;
}
GPA_DEV void unraw(const Raw8& r, int dt, float (&v)[8]) {
  const uint32_t s[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dt == kF32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(s[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 f;
      if (dt == kBF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&s[k]));
      else f = __half22float2(*reinterpret_cast<const __half2*>(&s[k]));
      v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
  }
}

template <int VEC>
GPA_DEV void ldv(const void* p, int64_t i, int dt, float (&v)[VEC]) {
  if constexpr (VEC == 1) v[0] = load_in(p, i, dt);
  else unraw(ldraw(p, i, dt), dt, v);
}

// a value or 8 of them on their way from memory
template <int VEC>
struct Held {
  Raw8 r;
  GPA_DEV void load(const void* p, int64_t i, int dt) { r = ldraw(p, i, dt); }
  GPA_DEV void get(int dt, float (&v)[8]) const { unraw(r, dt, v); }
};
template <>
struct Held<1> {
  float r;
  GPA_DEV void load(const void* p, int64_t i, int dt) { r = load_in(p, i, dt); }
  GPA_DEV void get(int, float (&v)[1]) const { v[0] = r; }
};

template <int VEC>
GPA_DEV void stv(void* p, int64_t i, int dt, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    store_out(p, i, v[0], dt);
  } else {
    if (dt == kF32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (dt == kBF16) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
          s[k] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
          s[k] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(s[0], s[1], s[2], s[3]);
    }
  }
}

// 1 / rms of a row from its sum of squares.  The forward takes the correctly rounded division and
// root (one each per row and thread): what it is off by shifts every value of the row, and the
// stream is rounded to 16 bits next.
GPA_DEV float inv_rms(float sum, int width, float eps) { return 1.f / sqrtf(sum / (float)width + eps); }

// 1 / (1 + e^-a), to about 2^-22.  The exponent a log2 e is split into its rounded value, which the
// exp2 unit takes, and what the rounding left, which enters to first order; one Newton step
// follows the reciprocal unit.  (Full exp and division: 10 us of 66 for 8188 x 2560.)
GPA_DEV float gate_of(float a) {
  constexpr float kLog2e = 1.44269502f, kRest = 1.92596303e-8f, kLn2 = 0.693147182f;  // log2 e = kLog2e + kRest
  const float x = a < -87.f ? -87.f : a > 87.f ? 87.f : a;  // e^-x and the rests stay finite; NaN passes
  const float t = -x * kLog2e;
  const float rest = fmaf(-x, kRest, fmaf(-x, kLog2e, -t));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  const float d = 1.f + fmaf(e, rest * kLn2, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  r = r * fmaf(-d, r, 2.f);
  return a < -87.f ? 0.f : r;
}

// The gate in the backward.  16-bit gates: exp2 and reciprocal units alone (7 us less), whose error,
// 2^-24 |a| and so about a hundredth of the rounding of the gate's own gradient, moves no result next
// to a border of another tensor's.  fp32 ones, whose gradients are fp32: as in the forward.
GPA_DEV float gate_back(float a, int dt) {
  return dt == kF32 ? gate_of(a) : __fdividef(1.f, 1.f + __expf(-a));
}

GPA_DEV float round_to(float x, int dt) {
  if (dt == kBF16) return __bfloat162float(__float2bfloat16(x));
  if (dt == kF16) return __half2float(__float2half(x));
  return x;
}

// Sums of NV values over the group: shuffles inside a warp (G <= 32), or shuffles and one pass
// through shared memory (G == 0: the whole block).  `buf` alternates between two shared arrays,
// so one barrier per sum is enough.
template <int G, int NV>
GPA_DEV void group_sum(float (&v)[NV], float (*sm)[3][32], int& buf) {
  constexpr int kW = G == 0 ? 32 : G;
#pragma unroll
  for (int o = kW / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (G == 0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
    if (nw > 1) {
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < NV; ++k) sm[buf][k][warp] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float s = lane < nw ? sm[buf][k][lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        v[k] = s;
      }
      buf ^= 1;
    }
  }
}

GPA_DEV int64_t row_at(const Rows& r, uint32_t row, uint32_t inner) {
  if (r.so == r.si * (int64_t)inner) return (int64_t)row * r.si;
  const uint32_t o = row / inner;
  return (int64_t)o * r.so + (int64_t)(row - o * inner) * r.si;
}

// The types of a kernel's tensors: known where it is built (DT), or read from its arguments
// (DT < 0).  Built in, a load and its conversions are half the instructions of a row.
constexpr int kAny = -1;
constexpr int types_of(int stream, int update, int out) { return stream | update << 2 | out << 4; }
#define NORM_TYPES(DT)                                                   \
  const int h_dt = (DT) < 0 ? p.h_dt : (DT) & 3;                         \
  const int y_dt = (DT) < 0 ? p.y_dt : (DT) >> 2 & 3;                    \
  const int g_dt = (DT) < 0 ? p.g_dt : y_dt;                             \
  const int out_dt = (DT) < 0 ? p.out_dt : (DT) >> 4 & 3

template <int G, int VEC, int ITER, int MT, int DT>
__global__ void __launch_bounds__(MT) k_norm_fwd(const Fwd p) {
  NORM_TYPES(DT);
  __shared__ float sm[2][3][32];
  int buf = 0;
  const int g = G == 0 ? (int)blockDim.x : G;
  const int t = G == 0 ? (int)threadIdx.x : (int)(threadIdx.x % G);
  const uint32_t per = G == 0 ? 1u : blockDim.x / G;
  const uint32_t row = blockIdx.x * per + (G == 0 ? 0u : threadIdx.x / G);
  const bool live = row < p.rows;  // idle groups of a warp still take part in its shuffles
  const bool plain = p.h == nullptr;
  float x[ITER][VEC];
  Held<VEC> held_h[ITER], held_g[ITER];  // every load of the row in flight before its first sum
  const int64_t oy = live ? row_at(p.ry, row, p.inner) : 0;
  const int64_t oh = live && !plain ? row_at(p.rh, row, p.inner) : 0;
  const int64_t og = live && p.gate ? row_at(p.rg, row, p.inner) : 0;
  float s1[1] = {0.f};
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * g + t) * VEC;
    if (!live || c >= p.width) continue;
    if (!plain) held_h[i].load(p.h, oh + c, h_dt);
    if (p.gate && p.gate_full) held_g[i].load(p.gate, og + c, g_dt);
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * g + t) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[i][k] = 0.f;
    if (live && c < p.width) ldv<VEC>(p.y, oy + c, y_dt, x[i]);
  }
  const int64_t at = (int64_t)row * p.width;
  if (!plain) {
    float ry = 1.f;
    if (p.wp) {
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s1[0] += x[i][k] * x[i][k];
      group_sum<G, 1>(s1, sm, buf);
      ry = inv_rms(s1[0], p.width, p.eps);
    }
    float gr = p.c;
    if (live && p.gate && !p.gate_full) gr *= gate_of(load_in(p.gate, og, g_dt));
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * g + t) * VEC;
      if (!live || c >= p.width) continue;
      float h[VEC], m[VEC];
      held_h[i].get(h_dt, h);
#pragma unroll
      for (int k = 0; k < VEC; ++k) m[k] = gr;
      if (p.gate && p.gate_full) {
        float a[VEC];
        held_g[i].get(g_dt, a);
#pragma unroll
        for (int k = 0; k < VEC; ++k) m[k] *= gate_of(a[k]);
      }
      if (p.scale) {
        float a[VEC];
        ldv<VEC>(p.scale, c, kF32, a);
#pragma unroll
        for (int k = 0; k < VEC; ++k) m[k] *= a[k];
      }
      if (p.wp) {
        float a[VEC];
        ldv<VEC>(p.wp, c, kF32, a);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[i][k] *= ry * a[k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[i][k] = round_to(fmaf(m[k], x[i][k], h[k]), h_dt);
      stv<VEC>(p.stream, at + c, h_dt, x[i]);
    }
  }
  float s2[1] = {0.f};
#pragma unroll
  for (int i = 0; i < ITER; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) s2[0] += x[i][k] * x[i][k];
  group_sum<G, 1>(s2, sm, buf);
  const float r = inv_rms(s2[0], p.width, p.eps);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * g + t) * VEC;
    if (!live || c >= p.width) continue;
    float w[VEC];
    ldv<VEC>(p.w, c, kF32, w);
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] *= x[i][k] * r;
    stv<VEC>(p.out, at + c, out_dt, w);
  }
}

// where a block leaves its column sums of one weight
GPA_DEV float* sums_at(const Bwd& b, int slot) {
  return b.part ? b.part + ((int64_t)blockIdx.x * b.sums + slot) * b.f.width : b.sums_out[slot];
}

// Column sums of a block's rows into its partial row: registers of one group, or of the block's
// groups added through shared memory.
template <int G, int VEC, int ITER>
GPA_DEV void emit_sums(float* dst, const float (&a)[ITER][VEC], int width, int g, int t, uint32_t mine,
                       uint32_t per, float* fold) {
  if constexpr (G == 0) {
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int c = (i * g + t) * VEC + k;
        if (c < width) dst[c] = a[i][k];
      }
  } else {
    constexpr int kCols = G * VEC * ITER;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) fold[mine * kCols + (i * G + t) * VEC + k] = a[i][k];
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      float s = 0.f;
      for (uint32_t j = 0; j < per; ++j) s += fold[j * kCols + c];
      dst[c] = s;
    }
  }
}

// PARTS: with a post weight, a gate or a scale.  Without, the update and its sums take no registers,
// which blocks of 1024 threads are short of (1864 x 9001 in bf16, step: 807 -> 638 us, where plain
// PyTorch takes 662; with parts they spill still: 1307, 1631).
template <int G, int VEC, int ITER, int MT, bool PARTS>
__global__ void __launch_bounds__(MT, 1) k_norm_bwd(const Bwd b) {
  const Fwd& p = b.f;
  NORM_TYPES(kAny);
  __shared__ float sm[2][3][32];
  extern __shared__ float fold[];  // sub-warp groups: [blockDim / G][G * VEC * ITER]
  int buf = 0;
  const int g = G == 0 ? (int)blockDim.x : G;
  const int t = G == 0 ? (int)threadIdx.x : (int)(threadIdx.x % G);
  const uint32_t per = G == 0 ? 1u : blockDim.x / G;
  const uint32_t mine = G == 0 ? 0u : threadIdx.x / G;
  const bool plain = !PARTS && p.h_dt < 0;
  const float inv = 1.f / (float)p.width;
  constexpr int kP = PARTS ? ITER : 1;
  float aw[ITER][VEC], ap[kP][VEC], ac[kP][VEC];
#pragma unroll
  for (int i = 0; i < ITER; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      aw[i][k] = 0.f;
      if constexpr (PARTS) ap[i][k] = ac[i][k] = 0.f;
    }
  const uint32_t step = gridDim.x * per;
  for (uint32_t base = blockIdx.x * per; base < p.rows; base += step) {
    const uint32_t row = base + mine;
    const bool live = row < p.rows;
    const int64_t at = (int64_t)row * p.width;
    const int64_t oy = live ? row_at(p.ry, row, p.inner) : 0;
    const int64_t og = PARTS && live && p.gate ? row_at(p.rg, row, p.inner) : 0;
    float x[ITER][VEC], d[ITER][VEC], y[kP][VEC];
    float s[PARTS ? 3 : 2] = {};  // x^2, w dn x, y^2
    Held<VEC> held_s[ITER], held_g[kP];  // read after the sums, on their way before them
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * g + t) * VEC;
      if (!live || c >= p.width) continue;
      if (b.ds) held_s[i].load(b.ds, at + c, h_dt);
      if constexpr (PARTS)
        if (p.gate && p.gate_full) held_g[i].load(p.gate, og + c, g_dt);
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * g + t) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        x[i][k] = d[i][k] = 0.f;
        if constexpr (PARTS) y[i][k] = 0.f;
      }
      if (!live || c >= p.width) continue;
      if (plain) ldv<VEC>(p.y, oy + c, y_dt, x[i]);
      else ldv<VEC>(p.stream, at + c, h_dt, x[i]);
      if (b.dn) ldv<VEC>(b.dn, at + c, out_dt, d[i]);
      if constexpr (PARTS) ldv<VEC>(p.y, oy + c, y_dt, y[i]);
      float w[VEC];
      ldv<VEC>(p.w, c, kF32, w);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        s[0] += x[i][k] * x[i][k];
        s[1] += w[k] * d[i][k] * x[i][k];
        if constexpr (PARTS) s[2] += y[i][k] * y[i][k];
      }
    }
    group_sum<G, PARTS ? 3 : 2>(s, sm, buf);
    const float r = rsqrtf(s[0] * inv + p.eps), q = s[1] * inv * r * r;
    float ry = 1.f, gr = 1.f;
    if constexpr (PARTS) {
      if (p.wp) ry = rsqrtf(s[2] * inv + p.eps);
      if (live && p.gate && !p.gate_full) gr = gate_back(load_in(p.gate, og, g_dt), g_dt);
    }
    float s2[2] = {0.f, 0.f};  // wp du y, row-gate gradient
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * g + t) * VEC;
      if (!live || c >= p.width) continue;
      float w[VEC], a[VEC];
      ldv<VEC>(p.w, c, kF32, w);
      if (b.dn) {  // without: nothing reaches the row through its norm, whatever it holds
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          aw[i][k] += d[i][k] * x[i][k] * r;
          d[i][k] = r * (w[k] * d[i][k] - x[i][k] * q);
        }
      }
      if (b.ds) {
        held_s[i].get(h_dt, a);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[i][k] += a[k];
      }
      if (!plain && b.dh) stv<VEC>(b.dh, at + c, h_dt, d[i]);
      if constexpr (!PARTS) {
        if (!plain) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) d[i][k] *= p.c;
        }
        if (b.dy) stv<VEC>(b.dy, at + c, y_dt, d[i]);
      } else {
        float wp[VEC], cs[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) wp[k] = 1.f, cs[k] = p.c;
        if (p.wp) ldv<VEC>(p.wp, c, kF32, wp);
        if (p.scale) {
          ldv<VEC>(p.scale, c, kF32, a);
#pragma unroll
          for (int k = 0; k < VEC; ++k) cs[k] *= a[k];
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) a[k] = gr;
        if (p.gate && p.gate_full) {
          held_g[i].get(g_dt, a);
#pragma unroll
          for (int k = 0; k < VEC; ++k) a[k] = gate_back(a[k], g_dt);
        }
        float dg[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float u = y[i][k] * ry * wp[k], G_ = d[i][k];
          ac[i][k] += G_ * a[k] * u * p.c;
          dg[k] = G_ * cs[k] * u * a[k] * (1.f - a[k]);
          s2[1] += dg[k];
          const float du = G_ * cs[k] * a[k];
          ap[i][k] += du * y[i][k] * ry;
          d[i][k] = du * wp[k];
          s2[0] += d[i][k] * y[i][k];
        }
        if (p.gate && p.gate_full && b.dgate) stv<VEC>(b.dgate, at + c, g_dt, dg);
      }
    }
    if constexpr (PARTS) {
      const bool row_gate = p.gate && !p.gate_full && b.dgate;
      if (p.wp || row_gate) group_sum<G, 2>(s2, sm, buf);
      if (row_gate && live && t == 0) store_out(b.dgate, row, s2[1], g_dt);
      if (!b.dy) continue;
      const float qy = p.wp ? s2[0] * inv * ry * ry : 0.f;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = (i * g + t) * VEC;
        if (!live || c >= p.width) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[i][k] = ry * (d[i][k] - y[i][k] * qy);
        stv<VEC>(b.dy, at + c, y_dt, d[i]);
      }
    }
  }
  auto emit = [&](int slot, const float (&a)[ITER][VEC]) {
    if (slot >= 0) emit_sums<G, VEC, ITER>(sums_at(b, slot), a, p.width, g, t, mine, per, fold);
  };
  emit(b.sum_w, aw);
  if constexpr (PARTS) {
    emit(b.sum_p, ap);
    emit(b.sum_c, ac);
  }
}

// The plain norm over narrow rows: each group takes kNarrow rows at once, all their loads in
// flight together (262144 x 128 bf16: 39 -> 27 us).
constexpr int kNarrow = 4;
template <int G>
__global__ void __launch_bounds__(128) k_norm_narrow(const Fwd p) {
  const int t = threadIdx.x % G, c = t * 8;
  const uint32_t row0 = (blockIdx.x * (128 / G) + threadIdx.x / G) * kNarrow;
  Raw8 raw[kNarrow];
#pragma unroll
  for (int u = 0; u < kNarrow; ++u) {
    raw[u].a = raw[u].b = make_uint4(0, 0, 0, 0);
    if (row0 + u < p.rows && c < p.width) raw[u] = ldraw(p.y, row_at(p.ry, row0 + u, p.inner) + c, p.y_dt);
  }
  float w[8] = {};
  if (c < p.width) ldv<8>(p.w, c, kF32, w);
#pragma unroll
  for (int u = 0; u < kNarrow; ++u) {
    float x[8], s = 0.f;
    unraw(raw[u], p.y_dt, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) s += x[k] * x[k];
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float r = inv_rms(s, p.width, p.eps);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= r * w[k];
    if (row0 + u < p.rows && c < p.width) stv<8>(p.out, (int64_t)(row0 + u) * p.width + c, p.out_dt, x);
  }
}

// Backward where the update's share is the update times a constant (or the plain norm): no more
// than the stream and the two gradients are read.  A block's next row is loaded while the
// current one is reduced and written (65536 x 1024: 346 -> 163 us).  Types built in, as in the other
// block kernels, gave nothing here (163 -> 172 us).
template <int G, int MT>
__global__ void __launch_bounds__(MT) k_norm_bwd_light(const Bwd b) {
  const Fwd& p = b.f;
  __shared__ float sm[2][3][32];
  extern __shared__ float fold[];
  int buf = 0;
  const int g = G == 0 ? (int)blockDim.x : G;
  const int t = G == 0 ? (int)threadIdx.x : (int)(threadIdx.x % G);
  const uint32_t per = G == 0 ? 1u : blockDim.x / G;
  const uint32_t mine = G == 0 ? 0u : threadIdx.x / G;
  const bool plain = p.h_dt < 0;
  const int x_dt = plain ? p.y_dt : p.h_dt;
  const int c = t * 8;
  const bool in = c < p.width;
  const float inv = 1.f / (float)p.width;
  float w[8] = {}, aw[1][8] = {};
  if (in) ldv<8>(p.w, c, kF32, w);
  const uint32_t step = gridDim.x * per;
  Raw8 rx, rd, rs;
  auto load = [&](uint32_t row) {
    rx.a = rx.b = rd.a = rd.b = rs.a = rs.b = make_uint4(0, 0, 0, 0);
    if (row >= p.rows || !in) return;
    const int64_t at = (int64_t)row * p.width + c;
    rx = plain ? ldraw(p.y, row_at(p.ry, row, p.inner) + c, x_dt) : ldraw(p.stream, at, x_dt);
    if (b.dn) rd = ldraw(b.dn, at, p.out_dt);
    if (b.ds) rs = ldraw(b.ds, at, p.h_dt);
  };
  load(blockIdx.x * per + mine);
  for (uint32_t base = blockIdx.x * per; base < p.rows; base += step) {
    const uint32_t row = base + mine;
    float x[8], d[8], e[8];
    unraw(rx, x_dt, x);
    unraw(rd, p.out_dt, d);
    if (b.ds) unraw(rs, p.h_dt, e);
    load(row + step < row ? 0xffffffffu : row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s[0] += x[k] * x[k];
      s[1] += w[k] * d[k] * x[k];
    }
    group_sum<G, 2>(s, sm, buf);
    const float r = rsqrtf(s[0] * inv + p.eps), q = s[1] * inv * r * r;
    if (row >= p.rows || !in) continue;
    const int64_t at = (int64_t)row * p.width + c;
    if (b.dn) {  // without: nothing reaches the row through its norm, whatever it holds
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        aw[0][k] += d[k] * x[k] * r;
        d[k] = r * (w[k] * d[k] - x[k] * q);
      }
    }
    if (b.ds) {
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] += e[k];
    }
    if (b.dh) stv<8>(b.dh, at, p.h_dt, d);
    if (b.dy) {
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] *= p.c;
      stv<8>(b.dy, at, p.y_dt, d);
    }
  }
  if (b.sum_w >= 0) emit_sums<G, 8, 1>(sums_at(b, b.sum_w), aw, p.width, g, t, mine, per, fold);
}

// Backward with a post weight, a gate or a scale, over rows of whole blocks with 8 channels a
// thread.  Five tensors are read and a row is met three times (before the first sums, after them,
// and after the second), so each thread copies its share of the next row into shared memory
// (cp.async, two stages, 16 bytes a thread and slot: no other thread reads it, so no barrier) and
// reads the current row from there whenever it needs it, instead of holding it in registers.  The
// build for up to 320 threads (2560 channels) has 96 registers, with which two blocks run on an SM: 97
// us for 8188 x 2560 in bf16, 125 with the build for 512.  Wider rows get the latter, one block an SM
// (8162 x 2568: 133 us): two would have 64 registers, which spill (5117 x 4096: 106 -> 108 us, in fp32
// 238 -> 283).  What bounds it now is its own
// instructions (62 % of the issue slots busy, DRAM 36 % before the packed arithmetic): 96 us for
// 8188 x 2560 in bf16, against 104 us one channel to an instruction, 118 us with direct loads and
// 125 us with three blocks of 64 registers, which spill.
GPA_DEV void copy16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

template <int MT, int DT>
__global__ void __launch_bounds__(MT, MT == 320 ? 2 : 1) k_norm_bwd_parts(const Bwd b) {
  const Fwd& p = b.f;
  NORM_TYPES(DT);
  __shared__ float sm[2][3][32];
  extern __shared__ uint4 slots[];  // [stage][slot][thread]
  int buf = 0;
  const int n = blockDim.x, t = threadIdx.x, c = t * 8;
  const bool in = c < p.width, full = p.gate && p.gate_full;
  const float inv = 1.f / (float)p.width;
  const auto wide = [](int dt) { return dt == kF32 ? 2 : 1; };  // slots of 8 values
  const int sx = 0, sd = sx + wide(h_dt), ss = sd + wide(out_dt), sy = ss + wide(h_dt), sg = sy + wide(y_dt);
  const int stage = (sg + wide(g_dt)) * n;
  uint4* mine = slots + t;
  auto fetch = [&](int slot, const void* src, int64_t i, int dt) {
    const char* q = static_cast<const char*>(src) + i * (dt == kF32 ? 4 : 2);
    copy16(mine + slot, q);
    if (dt == kF32) copy16(mine + slot + n, q + 16);
  };
  auto fetch_row = [&](uint32_t row, int s) {
    if (row < p.rows && in) {
      const int64_t at = (int64_t)row * p.width + c;
      fetch(s + sx * n, p.stream, at, h_dt);
      if (b.dn) fetch(s + sd * n, b.dn, at, out_dt);
      if (b.ds) fetch(s + ss * n, b.ds, at, h_dt);
      fetch(s + sy * n, p.y, row_at(p.ry, row, p.inner) + c, y_dt);
      if (full) fetch(s + sg * n, p.gate, row_at(p.rg, row, p.inner) + c, g_dt);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // two channels to an instruction: the kernel is bound by its instructions
  struct V8 {
    float2 v[4];
  };
  auto read = [&](int slot, int dt) {
    Raw8 r;
    r.a = mine[slot];
    if (dt == kF32) r.b = mine[slot + n];
    else r.b = make_uint4(0, 0, 0, 0);
    V8 o;
    unraw(r, dt, reinterpret_cast<float(&)[8]>(o));
    return o;
  };
  auto load = [&](const float* q) {
    V8 o;
    ldv<8>(q, c, kF32, reinterpret_cast<float(&)[8]>(o));
    return o;
  };
  auto store = [&](void* q, int64_t i, int dt, const V8& o) {
    stv<8>(q, i, dt, reinterpret_cast<const float(&)[8]>(o));
  };
  auto both = [](float f) { return make_float2(f, f); };
  V8 aw = {}, ap = {}, ac = {};
  int s = 0;
  fetch_row(blockIdx.x, s);
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, s = stage - s) {
    fetch_row(row + gridDim.x < row ? 0xffffffffu : row + gridDim.x, stage - s);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const int64_t at = (int64_t)row * p.width + c;
    float sums[3] = {0.f, 0.f, 0.f};  // x^2, w dn x, y^2
    if (in) {
      float2 xx = both(0.f), wx = both(0.f), yy = both(0.f);
      const V8 x = read(s + sx * n, h_dt);
#pragma unroll
      for (int k = 0; k < 4; ++k) xx = __ffma2_rn(x.v[k], x.v[k], xx);
      if (b.dn) {
        const V8 d = read(s + sd * n, out_dt), w = load(p.w);
#pragma unroll
        for (int k = 0; k < 4; ++k) wx = __ffma2_rn(__fmul2_rn(w.v[k], d.v[k]), x.v[k], wx);
      }
      if (p.wp) {
        const V8 y = read(s + sy * n, y_dt);
#pragma unroll
        for (int k = 0; k < 4; ++k) yy = __ffma2_rn(y.v[k], y.v[k], yy);
      }
      sums[0] = xx.x + xx.y, sums[1] = wx.x + wx.y, sums[2] = yy.x + yy.y;
    }
    group_sum<0, 3>(sums, sm, buf);
    const float r = rsqrtf(sums[0] * inv + p.eps), q = sums[1] * inv * r * r;
    const float ry = p.wp ? rsqrtf(sums[2] * inv + p.eps) : 1.f;
    float gr = 1.f;
    if (p.gate && !full) gr = gate_back(load_in(p.gate, row_at(p.rg, row, p.inner), g_dt), g_dt);
    float two[2] = {0.f, 0.f};  // wp du y, row-gate gradient
    V8 d;
    if (in) {
      const V8 x = read(s + sx * n, h_dt);
#pragma unroll
      for (int k = 0; k < 4; ++k) d.v[k] = both(0.f);
      if (b.dn) {
        d = read(s + sd * n, out_dt);
        const V8 w = load(p.w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          aw.v[k] = __ffma2_rn(__fmul2_rn(d.v[k], x.v[k]), both(r), aw.v[k]);
          d.v[k] = __fmul2_rn(both(r), __ffma2_rn(x.v[k], both(-q), __fmul2_rn(w.v[k], d.v[k])));
        }
      }
      if (b.ds) {
        const V8 e = read(s + ss * n, h_dt);
#pragma unroll
        for (int k = 0; k < 4; ++k) d.v[k] = __fadd2_rn(d.v[k], e.v[k]);
      }
      if (b.dh) store(b.dh, at, h_dt, d);
      V8 a;
#pragma unroll
      for (int k = 0; k < 4; ++k) a.v[k] = both(gr);
      if (full) {
        a = read(s + sg * n, g_dt);
#pragma unroll
        for (int k = 0; k < 4; ++k) a.v[k] = make_float2(gate_back(a.v[k].x, g_dt), gate_back(a.v[k].y, g_dt));
      }
      V8 cs, wp;
#pragma unroll
      for (int k = 0; k < 4; ++k) wp.v[k] = both(1.f), cs.v[k] = both(p.c);
      if (p.scale) {
        cs = load(p.scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) cs.v[k] = __fmul2_rn(cs.v[k], both(p.c));
      }
      if (p.wp) wp = load(p.wp);
      const V8 y = read(s + sy * n, y_dt);
      float2 wy = both(0.f), gg = both(0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 yr = __fmul2_rn(y.v[k], both(ry)), u = __fmul2_rn(yr, wp.v[k]);
        const float2 ga = __fmul2_rn(d.v[k], a.v[k]);
        ac.v[k] = __ffma2_rn(__fmul2_rn(ga, u), both(p.c), ac.v[k]);
        const float2 du = __fmul2_rn(ga, cs.v[k]);
        ap.v[k] = __ffma2_rn(du, yr, ap.v[k]);
        // the gate's gradient, du u (1 - a)
        a.v[k] = __fmul2_rn(__fmul2_rn(du, u), __ffma2_rn(a.v[k], both(-1.f), both(1.f)));
        gg = __fadd2_rn(gg, a.v[k]);
        d.v[k] = __fmul2_rn(du, wp.v[k]);
        wy = __ffma2_rn(d.v[k], y.v[k], wy);
      }
      two[0] = wy.x + wy.y, two[1] = gg.x + gg.y;
      if (full && b.dgate) store(b.dgate, at, g_dt, a);
    }
    const bool row_gate = p.gate && !full && b.dgate;
    if (p.wp || row_gate) group_sum<0, 2>(two, sm, buf);
    if (row_gate && t == 0) store_out(b.dgate, row, two[1], g_dt);
    if (!b.dy || !in) continue;
    if (p.wp) {
      const V8 y = read(s + sy * n, y_dt);
      const float qy = two[0] * inv * ry * ry;
#pragma unroll
      for (int k = 0; k < 4; ++k) d.v[k] = __fmul2_rn(both(ry), __ffma2_rn(y.v[k], both(-qy), d.v[k]));
    }
    store(b.dy, at, y_dt, d);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!in) return;
  if (b.sum_w >= 0) store(sums_at(b, b.sum_w), c, kF32, aw);
  if (b.sum_p >= 0) store(sums_at(b, b.sum_p), c, kF32, ap);
  if (b.sum_c >= 0) store(sums_at(b, b.sum_c), c, kF32, ac);
}

// out[k][c] = sum over blocks of part[block][k][c] (k: blockIdx.y), always in the same order: 32
// lanes for 32 columns, each adding every 32nd block, then the lanes in a tree.
struct Sums {
  float* out[3];
};
__global__ void __launch_bounds__(1024) k_norm_fold(const float* part, int blocks, int sums, int cols, Sums out) {
  __shared__ float sm[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int64_t pitch = (int64_t)sums * cols;
  const float* p = part + (int64_t)blockIdx.y * cols + c;
  float s = 0.f;
  if (c < cols)
    for (int b = threadIdx.y; b < blocks; b += 32) s += p[b * pitch];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(sm[threadIdx.x][threadIdx.y]);  // column blockIdx.x * 32 + threadIdx.y
  const int mine = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && mine < cols) out.out[blockIdx.y][mine] = s;
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool strides8(const Rows& r) { return r.so % 8 == 0 && r.si % 8 == 0; }

// Threads of a row: 8 consecutive channels each where every row starts on a 16-byte boundary
// (one or two 16-byte accesses), else one channel each.
struct Shape {
  int vec, group, iter, threads;  // group 0: the block
};

Shape shape_of(const Fwd& f, bool vec) {
  Shape s;
  s.vec = vec ? 8 : 1;
  const int n = (f.width + s.vec - 1) / s.vec;  // thread-sized pieces of a row
  if (n <= 32) {
    s.group = 1;
    while (s.group < n) s.group *= 2;
    if (s.group < 4) s.group = 4;
    s.iter = 1;
    s.threads = 128;
  } else {
    // single channels: four a thread, so that a block is not all barrier
    s.group = 0;
    // and two turns of a smaller block where one of more than 512 threads would run out of registers
    s.iter = vec ? (n > 512 ? 2 : 1) : 4;
    while ((n + s.iter - 1) / s.iter > 1024) s.iter *= 2;
    s.threads = ((n + s.iter - 1) / s.iter + 31) / 32 * 32;
  }
  return s;
}

constexpr int kMaxWidth = 16384;

// Runs CALL(group, vec, iter, most threads, types) for the shape.  The types are built in for blocks
// over aligned rows with the mixes that models train in, and read from the arguments elsewhere
// (8188 x 2560 with parts: bf16 65 us forward and 97 backward, fp16 69 and 115).
#define NORM_TYPED(DT, CALL, M)                                                             \
  do {                                                                                      \
    if ((DT) == types_of(kF32, kBF16, kBF16)) { CALL(M, types_of(kF32, kBF16, kBF16)); }    \
    else if ((DT) == types_of(kBF16, kBF16, kBF16)) { CALL(M, types_of(kBF16, kBF16, kBF16)); } \
    else if ((DT) == types_of(kF32, kF32, kF32)) { CALL(M, types_of(kF32, kF32, kF32)); }   \
    else { CALL(M, kAny); }                                                                 \
  } while (0)
#define NORM_DISPATCH(S, CALL, BLOCK)                               \
  do {                                                              \
    if ((S).vec == 8) {                                             \
      if ((S).group == 4) { CALL(4, 8, 1, 128); }                   \
      else if ((S).group == 8) { CALL(8, 8, 1, 128); }              \
      else if ((S).group == 16) { CALL(16, 8, 1, 128); }            \
      else if ((S).group == 32) { CALL(32, 8, 1, 128); }            \
      else if ((S).iter == 1) { BLOCK; }                            \
      else if ((S).threads <= 512) { CALL(0, 8, 2, 512); }          \
      else { CALL(0, 8, 2, 1024); }                                 \
    } else {                                                        \
      if ((S).group == 4) { CALL(4, 1, 1, 128); }                   \
      else if ((S).group == 8) { CALL(8, 1, 1, 128); }              \
      else if ((S).group == 16) { CALL(16, 1, 1, 128); }            \
      else if ((S).group == 32) { CALL(32, 1, 1, 128); }            \
      else if ((S).iter == 4 && (S).threads <= 256) { CALL(0, 1, 4, 256); } \
      else if ((S).iter == 4) { CALL(0, 1, 4, 1024); }              \
      else if ((S).iter == 8) { CALL(0, 1, 8, 1024); }              \
      else { CALL(0, 1, 16, 1024); }                                \
    }                                                               \
  } while (0)

int built_types(const Fwd& f, int stream_dt) {
  return f.gate && f.g_dt != f.y_dt ? kAny : types_of(stream_dt, f.y_dt, f.out_dt);
}

const char* fill(const GpaNormArgs* a, Fwd* f) {
  if (!a) return "args is NULL";
  if (a->outer < 0 || a->inner < 0 || a->width < 1)
    return "outer, inner and width must not be negative, width at least 1";
  for (int dt : {a->stream_dtype, a->update_dtype, a->gate_dtype, a->out_dtype})
    if (dt < 0 || dt > 2) return "dtypes must be F32, BF16 or F16";
  if (!a->update && !a->residual) return "update must not be NULL";
  if (a->gate_mode < 0 || a->gate_mode > 2) return "gate_mode must be 0, 1 or 2";
  if (a->gate_mode && !a->gate) return "gate_mode needs a gate";
  if (!a->residual && (a->gate_mode || a->post_weight || a->scale))
    return "a norm without a residual takes no post weight, gate or scale";
  if (!a->weight) return "weight must not be NULL";
  f->h = a->residual;
  f->y = a->update;
  f->gate = a->gate_mode ? a->gate : nullptr;
  f->w = a->weight;
  f->wp = a->post_weight;
  f->scale = a->scale;
  f->stream = nullptr;
  f->out = nullptr;
  f->rh = {a->residual_stride[0], a->residual_stride[1]};
  f->ry = {a->update_stride[0], a->update_stride[1]};
  f->rg = {a->gate_stride[0], a->gate_stride[1]};
  f->rows = (uint32_t)(a->outer * a->inner);
  f->inner = (uint32_t)std::max<int64_t>(a->inner, 1);
  f->width = a->width;
  f->h_dt = a->residual ? a->stream_dtype : -1;
  f->y_dt = a->update_dtype;
  f->g_dt = a->gate_dtype;
  f->out_dt = a->out_dtype;
  f->gate_full = a->gate_mode == 2;
  f->eps = a->eps;
  f->c = a->scale_const;
  return nullptr;
}

bool too_large(const GpaNormArgs* a) {
  return a->width > kMaxWidth || (a->inner && a->outer > (int64_t)0x7fffffff / a->inner);
}

bool vec_ok(const Fwd& f) {
  return f.width % 8 == 0 && aligned8(f.h) && aligned8(f.y) && aligned8(f.w) && aligned8(f.wp) &&
         aligned8(f.scale) && aligned8(f.stream) && aligned8(f.out) &&
         (!f.h || strides8(f.rh)) && strides8(f.ry) &&
         (!f.gate_full || (aligned8(f.gate) && strides8(f.rg)));
}

// Blocks of the backward: as many as run at once, each with many rows, so that its column sums
// are added in registers and few partial rows are left.  At most 8 blocks of 128 threads an SM.
int most_blocks(const Shape& s) { return 148 * std::max(1, 1024 / s.threads); }
// Few rows go to one block, which writes the sums itself: up to 8 turns of narrow rows (28 x 96: 105
// -> 97 us eager, most of it the host's, 8.3 us replayed either way), 2 of wide ones (6 x 647 in one
// block: 139 -> 130 us eager, but 16 -> 35 us replayed).
uint32_t one_block(const Shape& s) { return s.group ? 8 : 2; }
// 0: the kernel cannot have its shared memory.  Known: a kernel's blocks per SM by device, warps of a
// block and 32-byte units of shared memory a thread (two stages of a slot; the types of a call set
// them), 0 where not asked yet.  The grid says how the column sums are grouped, so it follows from
// the call alone.
constexpr int kUnits = 11;
using Known = std::atomic<int>[8][33][kUnits];
int bwd_blocks(const Shape& s, uint32_t rows, const void* kernel, size_t smem, Known& known) {
  const uint32_t per = s.group ? s.threads / s.group : 1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const size_t units = smem / (32 * s.threads);
  const bool keep = dev < 8 && units < kUnits;
  int at_once = keep ? known[dev][s.threads / 32][units].load(std::memory_order_relaxed) : 0;
  if (!at_once) {
    // rows of whole blocks: up to 2 x 10 slots of 16 bytes for 512 threads, whatever the types of this call
    if (!s.group && smem &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != cudaSuccess)
      return 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&at_once, kernel, s.threads, smem) != cudaSuccess || at_once < 1)
      at_once = 1;
    if (keep) known[dev][s.threads / 32][units].store(at_once, std::memory_order_relaxed);
  }
  const uint32_t need = (rows + per - 1) / per;
  if (need <= one_block(s)) return 1;
  return (int)std::min(need, (uint32_t)std::min(148 * at_once, most_blocks(s)));
}

}  // namespace

int norm_forward(const GpaNormArgs* a, void* stream_out, void* normed, cudaStream_t st, const char** why) {
  Fwd f;
  if ((*why = fill(a, &f))) return GPA_B200_BAD_ARGUMENT;
  if (too_large(a)) {
    *why = "at most 16384 channels and 2^31 - 1 rows";
    return GPA_B200_UNSUPPORTED;
  }
  if (f.rows == 0) return GPA_B200_OK;
  if (!f.y || !normed || (f.h && !stream_out)) {
    *why = "update and the outputs must not be NULL";
    return GPA_B200_BAD_ARGUMENT;
  }
  f.stream = stream_out;
  f.out = normed;
  const Shape s = shape_of(f, vec_ok(f));
  uint32_t per = s.group ? s.threads / s.group : 1;
  Launch scope("norm_fwd", st);
  if (!f.h && s.vec == 8 && s.group) {
    per *= kNarrow;
    const uint32_t grid = (f.rows + per - 1) / per;
    if (s.group == 4) k_norm_narrow<4><<<grid, 128, 0, st>>>(f);
    else if (s.group == 8) k_norm_narrow<8><<<grid, 128, 0, st>>>(f);
    else if (s.group == 16) k_norm_narrow<16><<<grid, 128, 0, st>>>(f);
    else k_norm_narrow<32><<<grid, 128, 0, st>>>(f);
    if (cudaGetLastError() == cudaSuccess) return GPA_B200_OK;
    *why = "norm_fwd launch failed";
    return GPA_B200_LAUNCH_FAILURE;
  }
  const uint32_t grid = (f.rows + per - 1) / per;
  const int types = f.h ? built_types(f, f.h_dt) : kAny;
#define CALL(G, V, I, M) k_norm_fwd<G, V, I, M, kAny><<<grid, s.threads, 0, st>>>(f)
#define TYPED(M, T) k_norm_fwd<0, 8, 1, M, T><<<grid, s.threads, 0, st>>>(f)
#define BLOCK                                            \
  if (s.threads <= 256) NORM_TYPED(types, TYPED, 256);   \
  else NORM_TYPED(types, TYPED, 512)
  NORM_DISPATCH(s, CALL, BLOCK);
#undef BLOCK
#undef TYPED
#undef CALL
  if (cudaGetLastError() == cudaSuccess) return GPA_B200_OK;
  *why = "norm_fwd launch failed";
  return GPA_B200_LAUNCH_FAILURE;
}

namespace {
// whichever variant runs, its partial rows fit
size_t partial_floats(const Fwd& f) {
  size_t most = 0;
  for (bool vec : {true, false}) {
    const Shape s = shape_of(f, vec);
    const uint32_t per = s.group ? s.threads / s.group : 1, need = (f.rows + per - 1) / per;
    if (need > one_block(s)) most = std::max<size_t>(most, std::min<size_t>(need, most_blocks(s)));
  }
  return most * 3 * f.width;
}
}  // namespace

size_t norm_scratch_bytes(const GpaNormArgs* a) {
  Fwd f;
  if (fill(a, &f) || too_large(a)) return 0;
  return partial_floats(f) * sizeof(float);
}

int norm_backward(const GpaNormArgs* a, const void* stream_in, const void* dstream, const void* dnormed,
                  const GpaNormGrads* g, void* scratch, size_t scratch_bytes, cudaStream_t st,
                  const char** why) {
  Bwd b;
  if ((*why = fill(a, &b.f))) return GPA_B200_BAD_ARGUMENT;
  if (too_large(a)) {
    *why = "at most 16384 channels and 2^31 - 1 rows";
    return GPA_B200_UNSUPPORTED;
  }
  Fwd& f = b.f;
  const bool plain = f.h == nullptr;
  if (!g || (!plain && !stream_in) || (plain && (!f.y || !g->dupdate)) ||
      (!f.y && (f.wp || f.scale || f.gate))) {
    *why = "a tensor that the gradients need is NULL";
    return GPA_B200_BAD_ARGUMENT;
  }
  if ((g->dpost_weight && !f.wp) || (g->dscale && !f.scale) || (g->dgate && !f.gate)) {
    *why = "a gradient is asked for of a tensor that is not there";
    return GPA_B200_BAD_ARGUMENT;
  }
  b.sums = 0;
  b.sum_w = g->dweight ? b.sums++ : -1;
  b.sum_p = g->dpost_weight ? b.sums++ : -1;
  b.sum_c = g->dscale ? b.sums++ : -1;
  float* out[3] = {g->dweight, g->dpost_weight, g->dscale};
  if (f.rows == 0) {
    for (float* o : out)
      if (o && cudaMemsetAsync(o, 0, sizeof(float) * f.width, st) != cudaSuccess) {
        *why = "clearing the weight gradients failed";
        return GPA_B200_LAUNCH_FAILURE;
      }
    return GPA_B200_OK;
  }
  const size_t want = partial_floats(f) * sizeof(float);
  if (b.sums && want && (!scratch || scratch_bytes < want)) {
    *why = "scratch is smaller than gpa_b200_norm_scratch_bytes";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (b.sums && want && !aligned8(scratch)) {
    *why = "scratch must start on 16 bytes";
    return GPA_B200_BAD_ARGUMENT;
  }
  f.stream = const_cast<void*>(stream_in);
  f.h = nullptr;  // the backward reads the stream, not the residual that went in
  b.dn = dnormed;
  b.ds = dstream;
  b.dh = g->dresidual;
  b.dy = g->dupdate;
  b.dgate = g->dgate;
  for (int k = 0, slot = 0; k < 3; ++k)
    if (out[k]) b.sums_out[slot++] = out[k];
  const bool vec = vec_ok(f) && aligned8(dnormed) && aligned8(dstream) && aligned8(g->dresidual) &&
                   aligned8(g->dupdate) && (!f.gate_full || aligned8(g->dgate)) && aligned8(g->dweight) &&
                   aligned8(g->dpost_weight) && aligned8(g->dscale);
  const Shape s = shape_of(f, vec);
  const bool parts = f.wp || f.scale || f.gate, light = s.vec == 8 && s.iter == 1 && !parts;
  int blocks = 0;
  {
    Launch scope("norm_bwd", st);
#define RUN(K, SMEM)                                                             \
  do {                                                                           \
    static Known known;                                                          \
    const size_t smem = (SMEM);                                                  \
    blocks = bwd_blocks(s, f.rows, reinterpret_cast<const void*>(&K), smem, known); \
    b.part = blocks > 1 ? static_cast<float*>(scratch) : nullptr;                \
    if (blocks) K<<<blocks, s.threads, smem, st>>>(b);                           \
  } while (0)
#define LIGHT(G, M) RUN((k_norm_bwd_light<G, M>), fold_smem)
#define CALL(G, V, I, M)                                                   \
  do {                                                                     \
    /* 8 channels a thread in one turn without parts: k_norm_bwd_light */ \
    if (parts || ((V) == 8 && (I) == 1)) RUN((k_norm_bwd<G, V, I, M, true>), fold_smem); \
    else RUN((k_norm_bwd<G, V, I, M, (V) == 8 && (I) == 1>), fold_smem);   \
  } while (0)
#define TYPED(M, T) RUN((k_norm_bwd_parts<M, T>), slot_smem)
#define BLOCK                                            \
  if (s.threads <= 320) NORM_TYPED(types, TYPED, 320);   \
  else NORM_TYPED(types, TYPED, 512)
    const int types = built_types(f, f.h_dt);
    const size_t fold_smem = s.group ? sizeof(float) * s.threads * s.vec * s.iter : 0;
    auto slots = [](int dt) { return dt == kF32 ? 2 : 1; };
    const size_t slot_smem = (size_t)2 * s.threads * 16 *
                             (2 * slots(f.h_dt) + slots(f.out_dt) + slots(f.y_dt) + slots(f.gate ? f.g_dt : f.y_dt));
    if (light) {
      if (s.group == 4) LIGHT(4, 128);
      else if (s.group == 8) LIGHT(8, 128);
      else if (s.group == 16) LIGHT(16, 128);
      else if (s.group == 32) LIGHT(32, 128);
      else if (s.threads <= 256) LIGHT(0, 256);
      else LIGHT(0, 512);
    } else {
      NORM_DISPATCH(s, CALL, BLOCK);
    }
#undef BLOCK
#undef TYPED
#undef CALL
#undef LIGHT
#undef RUN
    if (cudaGetLastError() != cudaSuccess || !blocks) {
      *why = "norm_bwd launch failed";
      return GPA_B200_LAUNCH_FAILURE;
    }
  }
  if (!b.sums || blocks == 1) return GPA_B200_OK;
  Sums sums = {};
  for (int k = 0; k < 3; ++k) sums.out[k] = b.sums_out[k];
  Launch scope("norm_fold", st);
  k_norm_fold<<<dim3((f.width + 31) / 32, b.sums), dim3(32, 32), 0, st>>>(b.part, blocks, b.sums, f.width, sums);
  if (cudaGetLastError() != cudaSuccess) {
    *why = "norm_fold launch failed";
    return GPA_B200_LAUNCH_FAILURE;
  }
  return GPA_B200_OK;
}

}  // namespace gpa
