// Softmax cross entropy of z = x W^T over a large vocabulary, in pieces of it, without keeping z:
//   m_i = max_v z_iv    s_i = sum_v exp(z_iv - m_i)    loss_i = m_i - z_{i, y_i} + log s_i
//   P_iv = exp(z_iv - m_i) / s_i - [v = y_i]        dx_i = s r_i (P W)_i        dW = s P^T (r x)
// with the upstream gradient of row i written as s r_i (see Upstream).
//
// Rows without a label are dropped first: the labelled ones are packed (k_pack), so masked
// tokens cost nothing and whatever they hold (NaN included) reaches no product.
//   forward:  each tile of z leaves (max, sum of exp) per row, k_join puts the tiles together
//   backward: the vocabulary goes by in pieces; z of a piece is formed again and turned into P
//             (in the piece's buffer), then dx += P W over the piece and dW of the piece = P^T x.
// Every sum runs in a fixed order.  dx is added up in fp32 over the pieces (and over parts of a
// piece where the tiles of dx alone would not fill the GPU) and rounded once by k_finish.
#include "vocab_loss.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace gpa {
namespace vloss {
namespace {

// ------------------------------------------------------------------ rows
constexpr int kRun = 32;              // caller's rows per block of k_pack
constexpr int kCountDirectly = 4096;  // up to here each block counts the labels before its own

__global__ void k_count(const int64_t* labels, int n, int64_t ignore, int* count) {
  const int i = blockIdx.x * kRun + threadIdx.x;
  const unsigned b = __ballot_sync(0xffffffffu, i < n && labels[i] != ignore);
  if (threadIdx.x == 0) count[blockIdx.x] = __popc(b);
}

struct Pack {
  const int64_t* labels;
  int n;
  int64_t ignore, vocab;
  const int* count;        // labelled rows of each run before, or NULL: counted here
  int runs;
  int *info, *row, *label, *pos;  // info: see Call::n_rows
  int64_t so, si, inner;   // the caller's rows
  int width, pitch;
  int64_t plane;
  bool vec;
  Split split;
};

// A value as it goes to the tensor cores: itself, or for fp32 three bf16 parts of 8 bits each, in
// planes `plane` elements apart.
GPA_DEV void put(__nv_bfloat16* d, int64_t, __nv_bfloat16 v) { *d = v; }
GPA_DEV void put(__half* d, int64_t, __half v) { *d = v; }
GPA_DEV void put(__nv_bfloat16* d, int64_t plane, float v) {
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const __nv_bfloat16 b = __float2bfloat16(v);
    d[q * plane] = b;
    v -= __bfloat162float(b);
  }
}
template <typename T>
struct Part {
  using type = T;
};
template <>
struct Part<float> {
  using type = __nv_bfloat16;
};

// One row of `width` values to `pitch` places, by one warp; 8 at a time where both ends allow it.
template <typename T>
GPA_DEV void put_row(const T* __restrict__ s, typename Part<T>::type* __restrict__ d, int64_t plane, int width,
                     int pitch, bool vec, int lane) {
  if (vec) {
#pragma unroll 4
    for (int c = lane * 8; c < width; c += 256) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(d + c) = *reinterpret_cast<const uint4*>(s + c);
      } else {
        float v[8];
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(s + c);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(s + c + 4);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            const float2 f = __bfloat1622float2(b);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
            v[2 * i] -= f.x, v[2 * i + 1] -= f.y;
          }
          *reinterpret_cast<uint4*>(d + q * plane + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  } else {
#pragma unroll 8
    for (int c = lane; c < pitch; c += 32) put(d + c, plane, c < width ? s[c] : T(0.f));
  }
}

// Packs the labelled rows: row[j], label[j] (-1 outside the vocabulary) and the channels of the
// j-th of them, pos[i] its place or -1.  A block takes kRun rows; two more fill the places behind
// the last row with zeros up to a multiple of 64, the reduction block of dW.  Four blocks share a
// run's copies (blockIdx.y), a row for each of their warps.  Up to 4096 rows a block counts the
// labels before its own (at most 32 KB), which costs less than a launch of k_count; beyond, they
// are counted once.
template <typename T>
__global__ void __launch_bounds__(256) k_pack(const Pack p, const T* src, typename Part<T>::type* dst) {
  __shared__ int part[8];
  __shared__ int place[kRun];
  let_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = min((int)blockIdx.x, p.runs);
  int before = 0;
  if (p.count) {
    for (int i = threadIdx.x; i < run; i += 256) before += p.count[i];
  } else {
    const int stop = min(run * kRun, p.n);
    for (int i = threadIdx.x; i < stop; i += 256) before += p.labels[i] != p.ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) part[warp] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) before += part[k];
  if ((int)blockIdx.x >= p.runs) {  // `before` is the number of packed rows
    const int extra = blockIdx.x - p.runs;
    if (extra == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
      p.info[0] = before;
      p.info[1] = 0;
      p.info[2] = p.split.parts ? p.split.parts : parts_of(p.split, (before + kTile - 1) / kTile, &p.info[3]);
      if (p.split.parts) p.info[3] = p.split.k_part;
    }
    const int end = (before + 63) / 64 * 64;
    for (int j = before + extra * kRun + blockIdx.y; j < min(end, before + (extra + 1) * kRun); j += 4)
      for (int c = threadIdx.x; c < p.pitch; c += 256) put(dst + (int64_t)j * p.pitch + c, p.plane, T(0.f));
    return;
  }
  if (warp == 0) {
    const int i = blockIdx.x * kRun + lane;
    const int64_t y = i < p.n ? p.labels[i] : p.ignore;
    const bool has = i < p.n && y != p.ignore;
    const unsigned b = __ballot_sync(0xffffffffu, has);
    const int at = before + __popc(b & ((1u << lane) - 1));
    place[lane] = has ? at : -1;
    if (has && blockIdx.y == 0) {
      p.row[at] = i;
      p.label[at] = y >= 0 && y < p.vocab ? (int)y : -1;
    }
    if (i < p.n && blockIdx.y == 0) p.pos[i] = has ? at : -1;
  }
  __syncthreads();
  const int k = blockIdx.y * 8 + warp;
  if (place[k] < 0) return;
  const int64_t i = (int64_t)blockIdx.x * kRun + k;
  put_row(src + (i / p.inner) * p.so + (i % p.inner) * p.si, dst + (int64_t)place[k] * p.pitch, p.plane, p.width,
          p.pitch, p.vec, lane);
}

// The weight where the tensor cores cannot read the caller's: rows that do not start on 16 bytes,
// or fp32 (few rows: in the backward alone, see k_few).  A warp a row; rows behind the last (of a plane) become zero.
template <typename T>
__global__ void __launch_bounds__(256) k_weight(const T* src, int64_t stride, int64_t vocab, int64_t rows, int width,
                                                int pitch, int64_t plane, bool vec, typename Part<T>::type* dst) {
  const int64_t v = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (v >= rows) return;
  auto* d = dst + v * pitch;
  if (v < vocab) put_row(src + v * stride, d, plane, width, pitch, vec, lane);
  else
    for (int c = lane; c < pitch; c += 32) put(d + c, plane, T(0.f));
}

// dW of a piece where the caller's rows do not start on 16 bytes: from padded rows, a warp each.
// Stores of single values straight from the tile (a row a thread) measured four times as long as
// the whole step (14 x 314 x 85437).
template <typename T>
__global__ void __launch_bounds__(256) k_unpad(const T* __restrict__ src, int pitch, int64_t rows, int width,
                                               T* __restrict__ dst) {
  const int64_t v = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (v >= rows) return;
#pragma unroll 8
  for (int c = threadIdx.x & 31; c < width; c += 32) dst[v * width + c] = src[v * pitch + c];
}

// ------------------------------------------------------------------ joins
GPA_DEV void merge(float& m, float& s, float m2, float s2) {
  const float big = fmaxf(m, m2), safe = big == -INFINITY ? 0.f : big;
  s = s * expf(m - safe) + s2 * expf(m2 - safe);
  m = big;
}

// Maximum and 1 / sum of exp, and loss, of each packed row from the (max, sum) pairs of its
// tiles: blockDim.x rows a block, blockDim.y lanes of tiles each (256 threads).  The block that
// finishes last adds the losses of a mean or sum in double, in a fixed order.
__global__ void __launch_bounds__(256) k_join(const Call c, const float2* part, int tiles, const float* z_label,
                                              float2* lse, float* each, const int* pos, float* packed,
                                              float* total, bool mean, int* counter) {
  __shared__ float2 sm[256];
  __shared__ bool last;
  after_previous();
  const int rows = *c.n_rows, lanes = blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const bool live = j < rows;
  float m = -INFINITY, s = 0.f;
  if (live) {
    int t = threadIdx.y;
    for (; t + 3 * lanes < tiles; t += 4 * lanes) {
      float2 p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = part[(t + k * lanes) * c.n_pad + j];
#pragma unroll
      for (int k = 0; k < 4; ++k) merge(m, s, p[k].x, p[k].y);
    }
    for (; t < tiles; t += lanes) {
      const float2 p = part[t * c.n_pad + j];
      merge(m, s, p.x, p.y);
    }
  }
  sm[tid] = make_float2(m, s);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    __syncthreads();
    if (threadIdx.y < o) {
      const float2 p = sm[tid + o * blockDim.x];
      merge(m, s, p.x, p.y);
      sm[tid] = make_float2(m, s);
    }
  }
  if (threadIdx.y == 0 && live) {
    const float log_s = logf(s);
    lse[j] = make_float2(m, 1.f / s);
    const float l = c.label[j] < 0 ? NAN : (m - z_label[j]) + log_s;
    if (each) each[c.row[j]] = l;
    else packed[j] = l;
  }
  if (each) {  // rows without a label, by the caller's numbering
    if (threadIdx.y == 0 && j < c.n && pos[j] < 0) each[j] = 0.f;
    return;
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  __shared__ double sums[8];
  double v = 0.;
  for (int i = tid; i < rows; i += 256) v += (double)__ldcg(packed + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((tid & 31) == 0) sums[tid >> 5] = v;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < 8; ++k) v += sums[k];
    *total = (float)(mean ? v / (double)(rows > 0 ? rows : 1) : v);
    *counter = 0;
  }
}

// ------------------------------------------------------------------ z of few fp32 rows
// z for R of the packed rows a blockIdx.y, with fp32 multiply-adds on the weight as it is: (max, sum of
// exp) of each row, or P of a piece.  The tensor cores take fp32 as three bf16 parts, and writing and
// reading those (12 bytes a value beside the 4) is most of the time where rows are few.  Scores against
// 151936 entries of 1024 channels: 8 rows 584 -> 194 us, 16 -> 218, 32 -> 345; steps 1420 -> 1136 and
// 1191, with 32 rows 1440 as before.  64 rows would take two turns of W, as long as their parts.  P
// comes from here too, of the same bits of z: what it is measured by (P - 1 may be nothing) must not
// differ by so much as a rounding.
//
// A warp takes E entries at a time, its lanes four channels each of every 128; x lies in shared memory
// as pairs of rows, and two rows go to an instruction.  W's next values are on their way meanwhile: with
// 8 rows it comes by at 4.1 TB/s (eight warps of 200 registers an SM), with 32 instructions bound it
// (half a warp's lanes for either 16 rows, with half the reads of x: 308 -> 334 us).  The E R sums are
// added over the lanes 32 at a time, so that lane l ends up with row l % R of kMine neighbouring entries.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewShared = 224 * 1024;

struct Few {
  const float* w;         // the caller's weight
  int64_t w_stride;
  int pitch;              // channels up to a multiple of 128
  bool vec;               // rows of W start on 16 bytes
  int64_t v0, end;        // entries
  // statistics
  float2* part;
  float* z_label;
  // P of the entries, and zeros behind the last of the vocabulary
  const float2* lse;
  uint16_t* p;
  int64_t p_pitch;
};

GPA_DEV float4 few_load(const float* p, int d, int width, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec) {
    if (d < width) v = __ldcs(reinterpret_cast<const float4*>(p + d));  // width is a multiple of 4
  } else {
    if (d < width) v.x = p[d];
    if (d + 1 < width) v.y = p[d + 1];
    if (d + 2 < width) v.z = p[d + 2];
    if (d + 3 < width) v.w = p[d + 3];
  }
  return v;
}

template <int R, int E, bool PROBS>
__global__ void __launch_bounds__(kFewThreads, 1) k_few(const Call c, const Few f) {
  // [R / 2][channels 0, 1 or 2, 3 of four][pitch / 4]: {row, next row} of two channels; neighbouring
  // lanes read neighbouring 16 bytes
  extern __shared__ float4 xs[];
  __shared__ float2 joined[kFewWarps][R];
  constexpr int kMine = E * R / 32;  // entries of a lane in the end
  let_next();
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = blockIdx.y * R, quads = f.pitch / 4;
  const int rows = min(*c.n_rows - first, R);
  if (rows <= 0) return;
  const int row = lane % R;
  const bool live = row < rows;
  const int label = live ? c.label[first + row] : -1;
  const uint16_t* x = static_cast<const uint16_t*>(c.x) + (int64_t)first * c.pitch;
  const int64_t x_plane = c.n_pad * c.pitch;
  for (int i = threadIdx.x; i < R * quads; i += kFewThreads) {
    const int j = i / quads, q = i % quads;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (j < rows && q * 4 < c.pitch) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {  // the parts add up to the value, without a rounding
        const uint2 u = *reinterpret_cast<const uint2*>(x + k * x_plane + (int64_t)j * c.pitch + q * 4);
        v[0] += __uint_as_float(u.x << 16), v[1] += __uint_as_float(u.x & 0xffff0000u);
        v[2] += __uint_as_float(u.y << 16), v[3] += __uint_as_float(u.y & 0xffff0000u);
      }
    }
    float* to = reinterpret_cast<float*>(xs + (j >> 1) * 2 * quads + q) + (j & 1);
    to[0] = v[0], to[2] = v[1];
    to += 4 * quads;
    to[0] = v[2], to[2] = v[3];
  }
  __syncthreads();
  float m = -INFINITY, s = 0.f;  // of the row so far, or P's: its maximum and factor
  const float one = live && label < 0 ? NAN : 1.f;  // no such label: the row is NaN
  if (PROBS && live) m = f.lse[first + row].x, s = f.lse[first + row].y * one;
  const int64_t step = (int64_t)gridDim.x * kFewWarps * E;
  for (int64_t v0 = f.v0 + ((int64_t)blockIdx.x * kFewWarps + warp) * E; v0 < f.end; v0 += step) {
    const float* w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = f.w + (v0 + e < c.vocab ? v0 + e : c.vocab - 1) * f.w_stride;
    float2 acc[E][R / 2];
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int r = 0; r < R / 2; ++r) acc[e][r] = make_float2(0.f, 0.f);
    float4 next[E];
#pragma unroll
    for (int e = 0; e < E; ++e) next[e] = few_load(w[e], lane * 4, c.width, f.vec);
    for (int d = lane * 4; d < f.pitch; d += 128) {
      float4 now[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        now[e] = next[e];
        next[e] = few_load(w[e], d + 128, c.width, f.vec);
      }
#pragma unroll
      for (int r = 0; r < R / 2; ++r) {
        const float4 a = xs[2 * r * quads + d / 4], b = xs[(2 * r + 1) * quads + d / 4];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float2 v = acc[e][r];
          v = __ffma2_rn(make_float2(a.x, a.y), make_float2(now[e].x, now[e].x), v);
          v = __ffma2_rn(make_float2(a.z, a.w), make_float2(now[e].y, now[e].y), v);
          v = __ffma2_rn(make_float2(b.x, b.y), make_float2(now[e].z, now[e].z), v);
          acc[e][r] = __ffma2_rn(make_float2(b.z, b.w), make_float2(now[e].w, now[e].w), v);
        }
      }
    }
    const int64_t mine = v0 + lane / R * kMine;
    float z[kMine];
#pragma unroll
    for (int g = 0; g < kMine; ++g) {
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const float2 a = acc[i / R * kMine + g][i % R / 2];
        v[i] = a.x, v[i + 1] = a.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const bool high = lane & o;
          const float keep = high ? v[i + o] : v[i], send = high ? v[i] : v[i + o];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      z[g] = v[0];
    }
    if constexpr (PROBS) {
      float p[kMine];
#pragma unroll
      for (int g = 0; g < kMine; ++g) {
        p[g] = expf(z[g] - m) * s - (mine + g == label ? one : 0.f);
        if (!live || mine + g >= c.vocab) p[g] = 0.f;
      }
      uint16_t* out = f.p + (first + row) * f.p_pitch + (mine - f.v0);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        uint32_t b[kMine / 2];
#pragma unroll
        for (int g = 0; g < kMine; g += 2) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(p[g], p[g + 1]);
          const float2 r = __bfloat1622float2(h);
          b[g / 2] = *reinterpret_cast<const uint32_t*>(&h);
          p[g] -= r.x, p[g + 1] -= r.y;
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(out + k * c.n_pad * f.p_pitch);
        if constexpr (kMine == 4) *reinterpret_cast<uint2*>(to) = make_uint2(b[0], b[1]);
        else *to = b[0];
      }
    } else {
#pragma unroll
      for (int g = 0; g < kMine; ++g) {
        const bool is = mine + g < c.vocab;
        if (is && mine + g == label) f.z_label[first + row] = z[g];
        merge(m, s, is ? z[g] : -INFINITY, is ? 1.f : 0.f);
      }
    }
  }
  if constexpr (!PROBS) {
#pragma unroll
    for (int o = R; o < 32; o <<= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      merge(m, s, m2, s2);
    }
    if (lane < R) joined[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < rows) {
      float2 a = joined[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < kFewWarps; ++k) merge(a.x, a.y, joined[k][threadIdx.x].x, joined[k][threadIdx.x].y);
      f.part[blockIdx.x * c.n_pad + first + threadIdx.x] = a;
    }
  }
}

// fp16, a gradient for each row: s = the largest magnitude, r = its share (x times r would leave
// fp16's range otherwise).
__global__ void __launch_bounds__(1024) k_row_scale(const float* dloss, const Call c, float* r, float* scale) {
  __shared__ float sm[32];
  const int n = *c.n_rows;
  float big = 0.f;
  for (int j = threadIdx.x; j < n; j += 1024) big = fmaxf(big, fabsf(dloss[c.row[j]]));
  big = warp_max(big);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = big;
  __syncthreads();
  big = warp_max(sm[threadIdx.x & 31]);
  const float s = big > 0.f && big < INFINITY ? big : 1.f;
  for (int j = threadIdx.x; j < n; j += 1024) r[j] = dloss[c.row[j]] / s;
  if (threadIdx.x == 0) *scale = s;
}

// The packed rows times their r, as dW takes them where each has a gradient of its own: rounded
// once more to the inputs' type (fp32: its parts formed again).  A warp a row, zero behind the
// last one up to a multiple of 64.
template <typename T>
__global__ void __launch_bounds__(256) k_scale(const Call c, const Upstream up, typename Part<T>::type* dst) {
  using E = typename Part<T>::type;
  const int rows = *c.n_rows;
  const int64_t j = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), plane = c.n_pad * c.pitch;
  if (j >= (rows + 63) / 64 * 64) return;
  const float r = j < rows ? up.r(c, j) : 0.f;
  const E* src = static_cast<const E*>(c.x) + j * c.pitch;
  E* d = dst + j * c.pitch;
  for (int k = threadIdx.x & 31; k < c.pitch; k += 32) {
    if (j >= rows) {
      put(d + k, plane, T(0.f));
    } else if constexpr (sizeof(T) == 4) {
      put(d + k, plane, ((float)src[k] + (float)src[plane + k] + (float)src[2 * plane + k]) * r);
    } else {
      put(d + k, plane, T((float)src[k] * r));
    }
  }
}

// dx of the caller's rows: the parts added in order, times the row's gradient, rounded; zero for rows
// without a label.  kV channels a thread at a time.
template <typename T, int kV>
__global__ void k_finish(const float* __restrict__ part, int64_t part_stride, const Call c, const int* pos,
                         const Upstream up, float unit, T* __restrict__ dx) {
  after_previous();
  const int64_t i = blockIdx.x;
  const int j = pos[i], parts = c.n_rows[2];
  const float s = j < 0 ? 0.f : up.scale(*c.n_rows) * up.r(c, j) * unit;
  T* out = dx + i * c.width;
  const float* p = part + (int64_t)j * c.pitch;
  for (int k = threadIdx.x * kV; k < c.width; k += blockDim.x * kV) {
    float v[kV];
    T o[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = 0.f;
    if (j >= 0) {
#pragma unroll 8
      for (int q = 0; q < parts; ++q) {
        if constexpr (kV > 1) {  // rows of the parts start on 16 bytes
#pragma unroll
          for (int e = 0; e < kV; e += 4) {
            const float4 f = *reinterpret_cast<const float4*>(p + q * part_stride + k + e);
            v[e] += f.x, v[e + 1] += f.y, v[e + 2] += f.z, v[e + 3] += f.w;
          }
        } else {
          v[0] += p[q * part_stride + k];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kV; ++e) o[e] = T(j >= 0 ? v[e] * s : 0.f);
    if constexpr (kV > 1) {
      *reinterpret_cast<uint4*>(out + k) = *reinterpret_cast<const uint4*>(o);
    } else {
      out[k] = o[0];
    }
  }
}

// ------------------------------------------------------------------ plan of a call
constexpr int64_t kPieceBytes = int64_t(3) << 29;  // of P at a time
// Of dW in padded rows at a time, where it takes these: 128 MB would cost 32 x 1925 x 111314 fp32 5 %.
constexpr int64_t kPaddedBytes = int64_t(1) << 29;

struct Plan {
  Call c;
  bool copy_w;             // the weight is copied first (k_weight)
  int few_rows;            // z by k_few: its rows a block (8, 16 or 32); or 0
  int es;                  // bytes of an element of the caller's tensors
  int parts_v;             // (max, sum) pairs of a row
  int64_t piece;           // vocabulary entries of a piece (a multiple of kTile)
  int64_t padded;          // and of dW's padded rows (likewise)
  Split split;             // of the reduction of dx
  // saved
  int64_t s_row, s_label, s_pos, s_lse, s_x, s_w, s_bytes;
  // scratch
  int64_t count, part, z_label, loss, fwd_bytes;
  int64_t p, dxp, dwp, xr, r, scale, w, bwd_bytes;
};

int few_blocks(const Plan& p, int64_t entries) {
  const int turn = kFewWarps * (p.few_rows == 32 ? 4 : 8);  // of a block
  return (int)std::min<int64_t>((entries + turn - 1) / turn, 2 * tc_pairs());
}
// Rows that a block of k_few takes of n: all of them where their x fits shared memory, or half of up to
// 16; 0: none, their parts on the tensor cores take less.
int few_rows(int64_t n, int width) {
  const int64_t fit = kFewShared / (up(width, 128) * 4);
  for (int r : {8, 16, 32})
    if (r <= fit && (n <= r || (r == 8 && n <= 16 && fit < 16))) return r;
  return 0;
}

const char* plan_of(const GpaLossArgs* a, Plan* p, int* code) {
  *code = GPA_B200_BAD_ARGUMENT;
  if (!a) return "args is NULL";
  if (a->outer < 0 || a->inner < 0 || a->width < 1 || a->vocab < 1)
    return "outer and inner must not be negative, width and vocab at least 1";
  if (a->dtype < 0 || a->dtype > 2) return "dtype must be F32, BF16 or F16";
  if (a->reduction < 0 || a->reduction > 2) return "reduction must be GPA_B200_LOSS_MEAN, _SUM or _NONE";
  if (a->weight_stride < a->width && a->vocab > 1) return "weight rows must not overlap";
  *code = GPA_B200_UNSUPPORTED;
  if (a->width > 65536) return "at most 65536 channels";
  if (a->vocab > (int64_t(1) << 29)) return "at most 2^29 vocabulary entries";
  if (a->inner && a->outer > (int64_t(1) << 22) / a->inner) return "at most 2^22 rows in a call";
  Call& c = p->c;
  c.n = a->outer * a->inner;
  c.vocab = a->vocab;
  c.width = a->width;
  c.dtype = a->dtype;
  const bool f32 = a->dtype == GPA_B200_F32;
  p->es = f32 ? 4 : 2;
  c.planes = f32 ? 3 : 1;
  c.pitch = (int)up(a->width, 8);
  c.n_pad = up(std::max<int64_t>(c.n, 1), kTile);
  p->copy_w = f32 || a->width % 8 || a->weight_stride % 8 || (reinterpret_cast<uintptr_t>(a->weight) & 15);
  c.w = a->weight;
  c.w_pitch = p->copy_w || a->vocab == 1 ? c.pitch : a->weight_stride;
  const int at_once = tc_pairs();
  const int64_t tiles_v = up(c.vocab, kTile) / kTile, tiles_m = c.n_pad / kTile;
  const int64_t tiles_d = (c.pitch + kTile - 1) / kTile;
  if (tiles_v * tiles_m > (int64_t(1) << 30)) return "at most 2^30 tiles of 256 x 256 logits in a call";
  c.few = c.n <= 32 ? 32 : c.n <= 128 ? 128 : 0;
  p->few_rows = f32 ? few_rows(c.n, c.width) : 0;
  p->parts_v = p->few_rows ? few_blocks(*p, c.vocab) : tc_stats_parts(c);
  // A piece is as large as its buffer allows, or somewhat smaller where the tiles of dW then
  // come out in fewer turns of the whole GPU (the pieces' turns added up; one piece has the fewest).
  const int64_t most = std::max<int64_t>(1, kPieceBytes / (c.n_pad * 2 * c.planes) / kTile);
  int64_t best = std::min(tiles_v, most), turns = INT64_MAX;
  auto turns_of = [&](int64_t t) {
    auto one = [&](int64_t v) { return (v * tiles_d + at_once - 1) / at_once; };
    return tiles_v / t * one(t) + (tiles_v % t ? one(tiles_v % t) : 0);
  };
  if (tiles_v > most)
    for (int64_t t = best; t >= 1 && t >= most / 2; --t)
      if (turns_of(t) < turns) turns = turns_of(t), best = t;
  p->piece = best * kTile;
  // dx: at most one part for every 512 entries, and 256 MB of them in all beside the first; the last
  // one holds what is left.  Cut by the blocks that the first piece has, not by its tiles: every part
  // of it then holds a block and is written, and later pieces, which add to the parts, may leave some
  // out.  A turn over a piece goes at about 1.4 PFLOP/s, the parts in fp32 at about 5 TB/s.
  Split& d = p->split;
  d.tiles_d = (int)tiles_d;
  d.at_once = at_once;
  d.blocks = (int)((std::min(p->piece, c.vocab) + 63) / 64);
  const int64_t one = c.n_pad * c.pitch * 4;
  d.most = (int)std::max<int64_t>(1, std::min<int64_t>({tiles_m == 1 ? 2 * at_once : 16, p->piece / 512,
                                                        1 + (int64_t(1) << 28) / one}));
  d.turn = (float)(2.0 * kTile * kTile * at_once * (double)p->piece * (f32 ? 6 : 1) / 1.4e15);
  d.pass = (float)((double)kTile * c.pitch * 8 / 5e12);
  d.parts = d.k_part = 0;
  if (tiles_m == 1) d.parts = parts_of(d, 1, &d.k_part);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  take(256);  // packed rows, counter
  p->s_row = take(4 * c.n);
  p->s_label = take(4 * c.n);
  p->s_pos = take(4 * c.n);
  p->s_lse = take(8 * c.n);
  p->s_x = take(c.planes * c.n_pad * c.pitch * 2);
  const int64_t w_bytes = p->copy_w ? c.planes * up(c.vocab, kTile) * c.pitch * 2 : 0;
  p->s_w = take(p->few_rows ? 0 : w_bytes);
  p->s_bytes = at;
  at = 0;
  p->count = take(4 * (up(c.n, kRun) / kRun));
  p->part = take((int64_t)p->parts_v * c.n_pad * 8);
  p->z_label = take(4 * c.n);
  p->loss = take(4 * c.n);
  p->fwd_bytes = at;
  at = 0;
  p->p = take(c.planes * c.n_pad * p->piece * 2);
  p->dxp = take((int64_t)p->split.most * c.n_pad * c.pitch * 4);
  p->padded = std::min(p->piece, std::max<int64_t>(1, kPaddedBytes / (c.pitch * p->es) / kTile) * kTile);
  p->dwp = take(p->padded * c.pitch * p->es);
  p->xr = take(a->reduction == GPA_B200_LOSS_NONE ? c.planes * c.n_pad * c.pitch * 2 : 0);
  p->r = take(4 * c.n);
  p->scale = take(4);
  p->w = take(p->few_rows ? w_bytes : 0);
  p->bwd_bytes = at;
  return nullptr;
}

template <typename T>
void pack(const GpaLossArgs* a, const Plan& p, char* saved, char* scratch, cudaStream_t st) {
  const Call& c = p.c;
  Pack k;
  k.labels = a->labels;
  k.n = (int)c.n;
  k.ignore = a->ignore_index;
  k.vocab = c.vocab;
  k.count = nullptr;
  k.runs = (int)(up(c.n, kRun) / kRun);
  k.info = reinterpret_cast<int*>(saved);
  k.row = reinterpret_cast<int*>(saved + p.s_row);
  k.label = reinterpret_cast<int*>(saved + p.s_label);
  k.pos = reinterpret_cast<int*>(saved + p.s_pos);
  k.so = a->hidden_stride[0];
  k.si = a->hidden_stride[1];
  k.inner = std::max<int64_t>(a->inner, 1);
  k.width = c.width;
  k.pitch = c.pitch;
  k.split = p.split;
  k.plane = c.n_pad * c.pitch;
  k.vec = a->width % 8 == 0 && k.so % 8 == 0 && k.si % 8 == 0 && (reinterpret_cast<uintptr_t>(a->hidden) & 15) == 0;
  if (c.n > kCountDirectly) {
    int* count = reinterpret_cast<int*>(scratch + p.count);
    k.count = count;
    Launch scope("loss_count", st);
    k_count<<<k.runs, kRun, 0, st>>>(a->labels, k.n, k.ignore, count);
  }
  Launch scope("loss_pack", st);
  k_pack<T><<<dim3(k.runs + 2, 4), 256, 0, st>>>(
      k, static_cast<const T*>(a->hidden), reinterpret_cast<typename Part<T>::type*>(saved + p.s_x));
}

template <typename T>
void copy_weight(const GpaLossArgs* a, const Plan& p, char* to, cudaStream_t st) {
  const Call& c = p.c;
  const int64_t rows = c.planes > 1 ? up(c.vocab, kTile) : c.vocab;
  const bool vec = c.width % 8 == 0 && a->weight_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a->weight) & 15) == 0;
  Launch scope("loss_weight", st);
  k_weight<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(
      static_cast<const T*>(a->weight), a->weight_stride, c.vocab, rows, c.width, c.pitch, rows * c.pitch, vec,
      reinterpret_cast<typename Part<T>::type*>(to));
}

template <int R, int E, bool PROBS>
bool few_as(const Plan& p, const Few& f, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may take its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(k_few<R, E, PROBS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared) !=
        cudaSuccess)
      return false;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  Launch scope(PROBS ? "loss_probs_few" : "loss_stats_few", st);
  return launch_next(k_few<R, E, PROBS>, dim3(few_blocks(p, f.end - f.v0), (unsigned)((p.c.n + R - 1) / R)),
                     kFewThreads, (size_t)R * f.pitch * 4, st, p.c, f);
}

template <bool PROBS>
bool few(const GpaLossArgs* a, const Plan& p, Few f, cudaStream_t st) {
  f.w = static_cast<const float*>(a->weight);
  f.w_stride = a->weight_stride;
  f.pitch = (int)up(p.c.width, 128);
  f.vec = a->width % 4 == 0 && f.w_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(f.w) & 15) == 0;
  if (p.few_rows == 8) return few_as<8, 8, PROBS>(p, f, st);
  return p.few_rows == 16 ? few_as<16, 8, PROBS>(p, f, st) : few_as<32, 4, PROBS>(p, f, st);
}

bool few_stats(const GpaLossArgs* a, const Plan& p, float2* part, float* z_label, cudaStream_t st) {
  Few f = {};
  f.end = p.c.vocab;
  f.part = part;
  f.z_label = z_label;
  return few<false>(a, p, f, st);
}

bool few_probs(const GpaLossArgs* a, const Plan& p, int64_t v0, int64_t vn, const float2* lse, void* to,
               cudaStream_t st) {
  Few f = {};
  f.v0 = v0;
  f.end = v0 + up(vn, 64);  // dx adds up whole blocks of entries, and dW of rows
  f.lse = lse;
  f.p = static_cast<uint16_t*>(to);
  f.p_pitch = p.piece;
  if (cudaMemset2DAsync(to, p.c.n_pad * p.piece * 2, 0, 64 * p.piece * 2, 3, st) != cudaSuccess) return false;
  return few<true>(a, p, f, st);
}

template <typename T>
bool finish(const Plan& p, const float* dxp, int64_t stride, const int* pos, const Upstream& up, void* dx,
            cudaStream_t st) {
  constexpr int kV = 16 / sizeof(T);
  const Call& c = p.c;
  const float unit = 1.f / tc_p_scale(c.dtype);
  Launch scope("loss_finish", st);
  const bool vec = c.width % kV == 0 && (reinterpret_cast<uintptr_t>(dx) & 15) == 0;
  return launch_next(vec ? k_finish<T, kV> : k_finish<T, 1>, (unsigned)c.n, 128, 0, st, dxp, stride, c, pos, up, unit,
                     static_cast<T*>(dx));
}

// the kernels read and write the workspaces 32 bytes at a time
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }
const char* const kMisaligned = "saved and scratch must start on 32 bytes";

void bind(Plan* p, const void* saved) {
  const char* s = static_cast<const char*>(saved);
  p->c.n_rows = reinterpret_cast<const int*>(s);
  p->c.row = reinterpret_cast<const int*>(s + p->s_row);
  p->c.label = reinterpret_cast<const int*>(s + p->s_label);
  p->c.x = s + p->s_x;
  if (p->copy_w && !p->few_rows) p->c.w = s + p->s_w;
}

#define BY_TYPE(DT, CALL)                                  \
  do {                                                     \
    if ((DT) == GPA_B200_F32) { using T = float; CALL; }   \
    else if ((DT) == GPA_B200_BF16) { using T = __nv_bfloat16; CALL; } \
    else { using T = __half; CALL; }                       \
  } while (0)

#define FAIL(MSG)                     \
  do {                                \
    *why = MSG;                       \
    return GPA_B200_LAUNCH_FAILURE;   \
  } while (0)
#define OK_OR(MSG)                                   \
  do {                                               \
    if (cudaGetLastError() != cudaSuccess) FAIL(MSG); \
  } while (0)

}  // namespace
}  // namespace vloss

using namespace vloss;

size_t loss_saved_bytes(const GpaLossArgs* a) {
  Plan p;
  int code;
  return plan_of(a, &p, &code) ? 0 : p.s_bytes;
}

size_t loss_scratch_bytes(const GpaLossArgs* a, int backward) {
  Plan p;
  int code;
  return plan_of(a, &p, &code) ? 0 : backward ? p.bwd_bytes : p.fwd_bytes;
}

int loss_cut(const GpaLossArgs* a, int64_t labelled, int64_t* cut, const char** why) {
  Plan p;
  int code;
  if ((*why = plan_of(a, &p, &code))) return code;
  if (!cut || labelled < 0 || labelled > p.c.n) {
    *why = "cut is NULL, or labelled not between 0 and the rows";
    return GPA_B200_BAD_ARGUMENT;
  }
  int parts = p.split.parts, k_part = p.split.k_part;
  if (!parts) parts = parts_of(p.split, (int)((labelled + kTile - 1) / kTile), &k_part);
  cut[0] = std::min(p.piece, p.c.vocab);
  cut[1] = (cut[0] + 63) / 64;
  cut[2] = parts;
  cut[3] = k_part;
  return GPA_B200_OK;
}

int loss_forward(const GpaLossArgs* a, float* loss, void* saved, size_t saved_bytes, void* scratch,
                 size_t scratch_bytes, cudaStream_t st, const char** why) {
  Plan p;
  int code;
  if ((*why = plan_of(a, &p, &code))) return code;
  const Call& c = p.c;
  const bool none = a->reduction == GPA_B200_LOSS_NONE;
  if (!a->weight || !saved || !scratch || (c.n && (!a->hidden || !a->labels)) || (!loss && !(none && !c.n))) {
    *why = "a tensor is NULL";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (saved_bytes < (size_t)p.s_bytes || scratch_bytes < (size_t)p.fwd_bytes) {
    *why = "saved or scratch is smaller than its size query";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (!aligned(saved) || !aligned(scratch)) {
    *why = kMisaligned;
    return GPA_B200_BAD_ARGUMENT;
  }
  char* sv = static_cast<char*>(saved);
  char* sc = static_cast<char*>(scratch);
  bind(&p, saved);
  float* each = none ? loss : nullptr;
  float* z_label = reinterpret_cast<float*>(sc + p.z_label);
  float2* part = reinterpret_cast<float2*>(sc + p.part);
  BY_TYPE(a->dtype, pack<T>(a, p, sv, sc, st));
  OK_OR("loss_pack launch failed");
  if (p.copy_w && !p.few_rows && c.n) {
    BY_TYPE(a->dtype, copy_weight<T>(a, p, sv + p.s_w, st));
    OK_OR("loss_weight launch failed");
  }
  if (c.n && p.few_rows && !few_stats(a, p, part, z_label, st)) FAIL("loss_stats_few launch failed");
  if (c.n && !p.few_rows && !tc_stats(c, part, z_label, st)) FAIL("loss_stats_tc5 launch failed");
  if (c.n || !none) {
    // few rows: more lanes for the tiles of each
    const int rows = c.n >= 4096 ? 32 : c.n >= 256 ? 8 : 2;
    Launch scope("loss_join", st);
    if (!launch_next(k_join, (unsigned)std::max<int64_t>(1, (c.n + rows - 1) / rows), dim3(rows, 256 / rows), 0, st, c,
                     part, p.parts_v, z_label, reinterpret_cast<float2*>(sv + p.s_lse), each,
                     reinterpret_cast<const int*>(sv + p.s_pos), reinterpret_cast<float*>(sc + p.loss), loss,
                     a->reduction == GPA_B200_LOSS_MEAN, reinterpret_cast<int*>(sv) + 1))
      FAIL("loss_join launch failed");
  }
  return GPA_B200_OK;
}

int loss_backward(const GpaLossArgs* a, const void* saved, size_t saved_bytes, const float* dloss,
                  void* dhidden, void* dweight, void* scratch, size_t scratch_bytes, cudaStream_t st,
                  const char** why) {
  Plan p;
  int code;
  if ((*why = plan_of(a, &p, &code))) return code;
  const Call& c = p.c;
  if (!a->weight || !saved || !scratch || (c.n && (!dloss || (!dhidden && !dweight)))) {
    *why = "a tensor is NULL";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (saved_bytes < (size_t)p.s_bytes || scratch_bytes < (size_t)p.bwd_bytes) {
    *why = "saved or scratch is smaller than its size query";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (!aligned(saved) || !aligned(scratch)) {
    *why = kMisaligned;
    return GPA_B200_BAD_ARGUMENT;
  }
  if (!c.n) {
    if (dweight && cudaMemsetAsync(dweight, 0, (size_t)c.vocab * c.width * p.es, st) != cudaSuccess) {
      *why = "clearing dweight failed";
      return GPA_B200_LAUNCH_FAILURE;
    }
    return GPA_B200_OK;
  }
  const char* sv = static_cast<const char*>(saved);
  char* sc = static_cast<char*>(scratch);
  bind(&p, saved);
  const float2* lse = reinterpret_cast<const float2*>(sv + p.s_lse);
  if (p.few_rows && dhidden) {  // dx takes the weight in parts
    copy_weight<float>(a, p, sc + p.w, st);
    OK_OR("loss_weight launch failed");
    p.c.w = sc + p.w;
  }
  void* pr = sc + p.p;
  float* dxp = reinterpret_cast<float*>(sc + p.dxp);
  const bool none = a->reduction == GPA_B200_LOSS_NONE;
  const Upstream up = {none ? dloss : nullptr, true, none ? nullptr : dloss, a->reduction == GPA_B200_LOSS_MEAN};
  Upstream up_w = up;
  const void* x = c.x;
  if (none && dweight) {
    if (a->dtype == GPA_B200_F16) {
      float* r = reinterpret_cast<float*>(sc + p.r);
      float* s = reinterpret_cast<float*>(sc + p.scale);
      Launch scope("loss_row_scale", st);
      k_row_scale<<<1, 1024, 0, st>>>(dloss, c, r, s);
      OK_OR("loss_row_scale launch failed");
      up_w = {r, false, s, false};
    }
    Launch scope("loss_scale", st);
    BY_TYPE(a->dtype, (k_scale<T><<<(unsigned)(c.n_pad / 8), 256, 0, st>>>(
                          c, up_w, reinterpret_cast<typename Part<T>::type*>(sc + p.xr))));
    OK_OR("loss_scale launch failed");
    x = sc + p.xr;
  }
  const int64_t part_stride = c.n_pad * c.pitch;
  // pieces start at multiples of 256 rows: every row of dW on 16 bytes (32 for fp32), or none
  const bool in_place = c.width == c.pitch && (reinterpret_cast<uintptr_t>(dweight) & (p.es == 4 ? 31 : 15)) == 0;
  for (int64_t v0 = 0; v0 < c.vocab; v0 += p.piece) {
    const int64_t vn = std::min(p.piece, c.vocab - v0);
    if (p.few_rows ? !few_probs(a, p, v0, vn, lse, pr, st) : !tc_probs(c, v0, vn, lse, pr, p.piece, st))
      FAIL("loss_probs launch failed");
    if (dhidden && !tc_dx(c, pr, p.piece, v0, vn, p.split.most, v0 > 0, dxp, part_stride, st))
      FAIL("loss_dx_tc5 launch failed");
    if (!dweight) continue;
    const int64_t some = in_place ? vn : p.padded;
    for (int64_t u0 = 0; u0 < vn; u0 += some) {
      const int64_t un = std::min(some, vn - u0);
      char* dw = static_cast<char*>(dweight) + (v0 + u0) * c.width * p.es;
      if (!tc_dw(c, static_cast<char*>(pr) + 2 * u0, p.piece, v0 + u0, un, x, up_w, in_place ? dw : sc + p.dwp,
                 c.pitch, st))
        FAIL("loss_dw_tc5 launch failed");
      if (in_place) continue;
      Launch scope("loss_unpad", st);
      BY_TYPE(a->dtype, (k_unpad<T><<<(unsigned)((un + 7) / 8), 256, 0, st>>>(
                            reinterpret_cast<const T*>(sc + p.dwp), c.pitch, un, c.width, reinterpret_cast<T*>(dw))));
      OK_OR("loss_unpad launch failed");
    }
  }
  if (dhidden) {
    bool ok = false;
    BY_TYPE(a->dtype, ok = finish<T>(p, dxp, part_stride, reinterpret_cast<const int*>(sv + p.s_pos), up, dhidden, st));
    if (!ok) FAIL("loss_finish launch failed");
  }
  return GPA_B200_OK;
}

}  // namespace gpa
