// Softmax cross entropy of z = x W^T over a large vocabulary, in pieces of it, without keeping z:
//   lse_i = log sum_v exp z_iv        loss_i = lse_i - z_{i, y_i}
//   P_iv = (exp(z_iv - lse_i) - [v = y_i]) r_i        dx = s P W        dW = s P^T x
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
  int *info, *row, *label, *pos;  // info: [packed rows, counter of k_join]
  int64_t so, si, inner;   // the caller's rows
  int width, pitch;
  bool vec;
};

// Packs the labelled rows: row[j], label[j] (-1 outside the vocabulary) and the channels of the
// j-th of them, pos[i] its place or -1.  A block takes kRun rows; two more fill the places behind
// the last row with zeros up to a multiple of 64, the reduction block of dW.  Four blocks share a
// run's copies (blockIdx.y), a row for each of their warps.  In n <= 4096 rows
// one launch is cheaper than k_count before it (a block reads 32 KB of labels at most); beyond,
// the labels before a block are counted once.
template <typename T>
__global__ void __launch_bounds__(256) k_pack(const Pack p, const T* src, T* dst) {
  constexpr int kV = 16 / sizeof(T);
  __shared__ int part[8];
  __shared__ int place[kRun];
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
    if (extra == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.info[0] = before, p.info[1] = 0;
    const int end = (before + 63) / 64 * 64;
    for (int j = before + extra * kRun + blockIdx.y; j < min(end, before + (extra + 1) * kRun); j += 4)
      for (int c = threadIdx.x; c < p.pitch; c += 256) dst[(int64_t)j * p.pitch + c] = T(0.f);
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
  const T* s = src + (i / p.inner) * p.so + (i % p.inner) * p.si;
  T* d = dst + (int64_t)place[k] * p.pitch;
  if (p.vec) {
#pragma unroll 4
    for (int c = lane * kV; c < p.width; c += 32 * kV)
      *reinterpret_cast<uint4*>(d + c) = *reinterpret_cast<const uint4*>(s + c);
  } else {
    for (int c = lane; c < p.pitch; c += 32) d[c] = c < p.width ? s[c] : T(0.f);
  }
}

// Weight rows that cannot be read 16 bytes at a time: a copy with padded rows.
template <typename T>
__global__ void k_pad(const T* src, int64_t stride, int width, int pitch, T* dst) {
  const T* s = src + blockIdx.x * stride;
  T* d = dst + (int64_t)blockIdx.x * pitch;
  for (int c = threadIdx.x; c < pitch; c += blockDim.x) d[c] = c < width ? s[c] : T(0.f);
}

// ------------------------------------------------------------------ joins
GPA_DEV void merge(float& m, float& s, float m2, float s2) {
  const float big = fmaxf(m, m2), safe = big == -INFINITY ? 0.f : big;
  s = s * expf(m - safe) + s2 * expf(m2 - safe);
  m = big;
}

// lse and loss of each packed row from the (max, sum) pairs of its tiles: blockDim.x rows a block,
// blockDim.y lanes of tiles each (256 threads).  The block that finishes last adds the losses of
// a mean or sum in double, in a fixed order.
__global__ void __launch_bounds__(256) k_join(const Call c, const float2* part, int tiles, const float* z_label,
                                              float* lse, float* each, const int* pos, float* packed,
                                              float* total, bool mean, int* counter) {
  __shared__ float2 sm[256];
  __shared__ bool last;
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
    lse[j] = m + log_s;
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

// fp16, a gradient for each row: s = the largest magnitude, r = its share (fp16's range would lose
// the products otherwise).
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

// dx of the caller's rows: the parts added in order, scaled, rounded; zero for rows without a
// label.  kV channels a thread at a time.
template <typename T, int kV>
__global__ void k_finish(const float* part, int parts, int64_t part_stride, const Call c, const int* pos,
                         const Upstream up, float unit, T* dx) {
  const int64_t i = blockIdx.x;
  const int j = pos[i];
  const float s = up.scale(*c.n_rows) * unit;
  T* out = dx + i * c.width;
  const float* p = part + (int64_t)j * c.pitch;
  for (int k = threadIdx.x * kV; k < c.width; k += blockDim.x * kV) {
    float v[kV];
    T o[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = 0.f;
    if (j >= 0) {
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

// ------------------------------------------------------------------ products without tensor cores
// fp32 inputs: C (128 x 128 per block, 8 x 8 per thread) = A B over k, fp32 multiply-adds.  An
// operand is K-major (k contiguous) or MN-major; both are read 4 elements at a time.  Tensor cores
// would take three bf16 parts of each operand and six products for the same precision, and lose
// it again over reductions as long as the vocabulary.
constexpr int kB = 128, kBK = 16;

struct Operand {
  const float* p;
  int64_t pitch;
  int64_t mn, k;  // extents: reads outside give zero (whole groups of 4 along the contiguous axis)
};

template <bool KMAJOR>
GPA_DEV void fetch(const Operand& o, int64_t mn0, int64_t k0, float (&v)[2][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * 256;  // 512 groups of 4 of a 128 x 16 tile
    const int64_t mn = mn0 + (KMAJOR ? i >> 2 : (i & 31) * 4), k = k0 + (KMAJOR ? (i & 3) * 4 : i >> 5);
    v[h][0] = v[h][1] = v[h][2] = v[h][3] = 0.f;
    if (mn < o.mn && k < o.k) {
      const float4 f = *reinterpret_cast<const float4*>(o.p + (KMAJOR ? mn * o.pitch + k : k * o.pitch + mn));
      v[h][0] = f.x, v[h][1] = f.y, v[h][2] = f.z, v[h][3] = f.w;
    }
  }
}

template <bool KMAJOR>
GPA_DEV void put(float (*s)[kB + 4], const float (&v)[2][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * 256;
    if (KMAJOR) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[(i & 3) * 4 + e][i >> 2] = v[h][e];
    } else {
      *reinterpret_cast<float4*>(&s[i >> 5][(i & 31) * 4]) = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
    }
  }
}

// acc[i][j]: row m0 + (ty * 4 + i % 4) + 64 * (i / 4), column n0 + (tx * 4 + j % 4) + 64 * (j / 4)
template <bool AK, bool BK_>
GPA_DEV void product(const Operand& a, const Operand& b, int64_t m0, int64_t n0, int64_t k0,
                     int64_t k1, float (&acc)[8][8]) {
  __shared__ float sa[2][kBK][kB + 4], sb[2][kBK][kB + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  float va[2][4], vb[2][4];
  if (k0 < k1) {
    fetch<AK>(a, m0, k0, va);
    fetch<BK_>(b, n0, k0, vb);
  }
  int s = 0;
  for (int64_t k = k0; k < k1; k += kBK, s ^= 1) {
    put<AK>(sa[s], va);
    put<BK_>(sb[s], vb);
    __syncthreads();
    if (k + kBK < k1) {
      fetch<AK>(a, m0, k + kBK, va);
      fetch<BK_>(b, n0, k + kBK, vb);
    }
#pragma unroll
    for (int kk = 0; kk < kBK; ++kk) {
      float fa[8], fb[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<float4*>(fa + 4 * h) = *reinterpret_cast<const float4*>(&sa[s][kk][ty * 4 + 64 * h]);
        *reinterpret_cast<float4*>(fb + 4 * h) = *reinterpret_cast<const float4*>(&sb[s][kk][tx * 4 + 64 * h]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
    }
  }
}

GPA_DEV int at8(int t, int i) { return t * 4 + (i & 3) + 64 * (i >> 2); }

__global__ void __launch_bounds__(256, 2) k_stats(const Call c, float2* part, float* z_label) {
  const int64_t m0 = (int64_t)blockIdx.y * kB, n0 = (int64_t)blockIdx.x * kB;
  if (m0 >= *c.n_rows) return;
  float acc[8][8];
  product<true, true>({static_cast<const float*>(c.x), c.pitch, c.n_pad, c.pitch},
                            {static_cast<const float*>(c.w), c.w_pitch, c.vocab, c.pitch}, m0, n0, 0, c.pitch, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + at8(ty, i);
    const bool live = m < *c.n_rows;
    const int y = live ? c.label[m] : -1;
    float big = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t v = n0 + at8(tx, j);
      if (v >= c.vocab) acc[i][j] = -INFINITY;
      else if (v == y) z_label[m] = acc[i][j];
      big = fmaxf(big, acc[i][j]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    const float safe = big == -INFINITY ? 0.f : big;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += expf(acc[i][j] - safe);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (tx == 0 && live) part[blockIdx.x * c.n_pad + m] = make_float2(big, s);
  }
}

__global__ void __launch_bounds__(256, 2) k_probs(const Call c, int64_t v0, int64_t vn, const float* lse,
                                                  const Upstream up, float* p, int64_t p_pitch) {
  const int64_t m0 = (int64_t)blockIdx.y * kB, n0 = (int64_t)blockIdx.x * kB;
  if (m0 >= *c.n_rows) return;
  float acc[8][8];
  product<true, true>({static_cast<const float*>(c.x), c.pitch, c.n_pad, c.pitch},
                            {static_cast<const float*>(c.w) + v0 * c.w_pitch, c.w_pitch, vn, c.pitch}, m0, n0, 0,
                            c.pitch, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + at8(ty, i);
    const bool live = m < *c.n_rows;
    const float l = live ? lse[m] : 0.f, ri = live ? up.r(c, m) : 0.f;
    const int64_t y = live ? c.label[m] - v0 : -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t v = n0 + at8(tx, j);
      p[m * p_pitch + v] = live && v < vn ? (expf(acc[i][j] - l) - (v == y ? 1.f : 0.f)) * ri : 0.f;
    }
  }
}

// part[z] (+)= P[:, k of part z] W
__global__ void __launch_bounds__(256, 2) k_dx(const Call c, const float* p, int64_t p_pitch, int64_t v0,
                                               int64_t vn, int64_t k_part, bool add, float* part,
                                               int64_t part_stride) {
  const int64_t m0 = (int64_t)blockIdx.y * kB, n0 = (int64_t)blockIdx.x * kB;
  if (m0 >= *c.n_rows) return;
  const int64_t k0 = blockIdx.z * k_part, k1 = k0 + k_part < vn ? k0 + k_part : vn;
  float acc[8][8];
  product<true, false>({p, p_pitch, c.n_pad, p_pitch},
                                 {static_cast<const float*>(c.w) + v0 * c.w_pitch, c.w_pitch, c.pitch, vn}, m0, n0,
                                 k0, k1, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float* o = part + blockIdx.z * part_stride;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + at8(ty, i);
    if (m >= *c.n_rows) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t d = n0 + at8(tx, j);
      if (d < c.pitch) o[m * c.pitch + d] = add ? o[m * c.pitch + d] + acc[i][j] : acc[i][j];
    }
  }
}

__global__ void __launch_bounds__(256, 2) k_dw(const Call c, const float* p, int64_t p_pitch, int64_t v0,
                                               int64_t vn, const Upstream up, float* dw) {
  const int64_t m0 = (int64_t)blockIdx.y * kB, n0 = (int64_t)blockIdx.x * kB;
  const int64_t rows = *c.n_rows;
  float acc[8][8];
  product<false, false>({p, p_pitch, p_pitch, rows}, {static_cast<const float*>(c.x), c.pitch, c.pitch, rows},
                                  m0, n0, 0, rows, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float s = up.scale(*c.n_rows);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t v = m0 + at8(ty, i);
    if (v >= vn) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t d = n0 + at8(tx, j);
      if (d < c.width) dw[(v0 + v) * c.width + d] = acc[i][j] * s;
    }
  }
}

// ------------------------------------------------------------------ plan of a call
constexpr int64_t kPieceBytes = int64_t(3) << 29;  // of P at a time

struct Plan {
  Call c;
  bool copy_w;             // weight rows that cannot be read 16 bytes at a time are copied first
  int es;                  // bytes of an element of x and W
  bool tc;                 // tensor cores (16-bit inputs)
  int pes;                 // bytes of an element of P
  int tiles_v, tiles_m;    // tiles of z
  int64_t piece;           // vocabulary entries of a piece (a multiple of kTile)
  int parts;               // parts of dx
  int64_t k_part;          // vocabulary entries of a part
  // saved
  int64_t s_row, s_label, s_pos, s_lse, s_x, s_bytes;
  // scratch
  int64_t w, count, part, z_label, loss, fwd_bytes;
  int64_t p, dxp, r, scale, bwd_bytes;
};

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
  if (a->vocab > (int64_t(1) << 30)) return "at most 2^30 vocabulary entries";
  if (a->inner && a->outer > (int64_t(1) << 22) / a->inner) return "at most 2^22 rows in a call";
  Call& c = p->c;
  c.n = a->outer * a->inner;
  c.vocab = a->vocab;
  c.width = a->width;
  c.dtype = a->dtype;
  p->es = a->dtype == GPA_B200_F32 ? 4 : 2;
  const int unit = 16 / p->es;
  c.pitch = (int)up(a->width, unit);
  c.n_pad = up(std::max<int64_t>(c.n, 1), kTile);
  p->copy_w = a->width % unit || a->weight_stride % unit || (reinterpret_cast<uintptr_t>(a->weight) & 15);
  c.w = a->weight;
  c.w_pitch = p->copy_w ? c.pitch : a->vocab > 1 ? a->weight_stride : c.pitch;
  p->tc = a->dtype != GPA_B200_F32;
  p->pes = p->tc ? 2 : 4;
  const int tile = p->tc ? kTile : kB, at_once = p->tc ? tc_pairs() : 2 * 148;
  p->tiles_v = (int)((c.vocab + tile - 1) / tile);
  p->tiles_m = (int)(c.n_pad / tile);
  const int64_t tiles_d = (c.pitch + tile - 1) / tile;
  // A piece is as large as its buffer allows, or somewhat smaller where the tiles of dW then
  // come out in fewer turns of the whole GPU (the pieces' turns added up).
  const int64_t most = std::max<int64_t>(1, kPieceBytes / (c.n_pad * p->pes) / kTile);
  const int64_t all = up(c.vocab, kTile) / kTile;
  int64_t best = std::min(all, most), turns = INT64_MAX;
  auto turns_of = [&](int64_t t) {
    auto one = [&](int64_t v) { return (v * (kTile / tile) * tiles_d + at_once - 1) / at_once; };
    return all / t * one(t) + (all % t ? one(all % t) : 0);
  };
  for (int64_t t = std::min(all, most); t >= 1 && t >= std::min(all, most) / 2; --t)
    if (turns_of(t) < turns) turns = turns_of(t), best = t;
  p->piece = best * kTile;
  // dx: the reduction is cut into parts of at least 512 entries where that fills the GPU's turns
  // better; every part costs another pass over dx in fp32, so a gain of 10 % is asked for.
  p->parts = 1;
  const int64_t tiles_x = tiles_d * p->tiles_m;
  double cost = (double)((tiles_x + at_once - 1) / at_once);
  for (int n = 2; n <= 2 * at_once && n <= p->piece / 512; ++n) {
    const double now = (double)((tiles_x * n + at_once - 1) / at_once) / n;
    if (now < 0.9 * cost) cost = now, p->parts = n;
  }
  p->k_part = up((p->piece + p->parts - 1) / p->parts, 64);
  p->parts = (int)((p->piece + p->k_part - 1) / p->k_part);
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
  p->s_lse = take(4 * c.n);
  p->s_x = take(c.n_pad * c.pitch * p->es);
  p->s_bytes = at;
  at = 0;
  p->w = take(p->copy_w ? c.vocab * c.pitch * p->es : 0);
  const int64_t common = at;
  p->count = take(4 * up(c.n, kRun) / kRun);
  p->part = take((int64_t)p->tiles_v * c.n_pad * 8);
  p->z_label = take(4 * c.n);
  p->loss = take(4 * c.n);
  p->fwd_bytes = at;
  at = common;
  p->p = take(c.n_pad * p->piece * p->pes);
  p->dxp = take((int64_t)p->parts * c.n_pad * c.pitch * 4);
  p->r = take(4 * c.n);
  p->scale = take(4);
  p->bwd_bytes = at;
  return nullptr;
}

template <typename T>
void pack(const GpaLossArgs* a, const Plan& p, char* saved, char* scratch, cudaStream_t st) {
  const Call& c = p.c;
  constexpr int kV = 16 / sizeof(T);
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
  k.vec = a->width % kV == 0 && k.so % kV == 0 && k.si % kV == 0 &&
          (reinterpret_cast<uintptr_t>(a->hidden) & 15) == 0;
  if (c.n > kCountDirectly) {
    int* count = reinterpret_cast<int*>(scratch + p.count);
    k.count = count;
    Launch scope("loss_count", st);
    k_count<<<k.runs, kRun, 0, st>>>(a->labels, k.n, k.ignore, count);
  }
  Launch scope("loss_pack", st);
  k_pack<T><<<dim3(k.runs + 2, 4), 256, 0, st>>>(k, static_cast<const T*>(a->hidden), reinterpret_cast<T*>(saved + p.s_x));
}

template <typename T>
void pad_weight(const GpaLossArgs* a, const Plan& p, char* scratch, cudaStream_t st) {
  Launch scope("loss_pad", st);
  k_pad<T><<<(unsigned)p.c.vocab, 128, 0, st>>>(static_cast<const T*>(a->weight), a->weight_stride, p.c.width,
                                                p.c.pitch, reinterpret_cast<T*>(scratch + p.w));
}

template <typename T>
void finish(const Plan& p, const float* dxp, int64_t stride, const int* pos, const Upstream& up, void* dx,
            cudaStream_t st) {
  constexpr int kV = 16 / sizeof(T);
  const Call& c = p.c;
  const float unit = 1.f / (p.tc ? tc_p_scale(c.dtype) : 1.f);
  Launch scope("loss_finish", st);
  if (c.width % kV == 0 && (reinterpret_cast<uintptr_t>(dx) & 15) == 0)
    k_finish<T, kV><<<(unsigned)c.n, 128, 0, st>>>(dxp, p.parts, stride, c, pos, up, unit, static_cast<T*>(dx));
  else
    k_finish<T, 1><<<(unsigned)c.n, 128, 0, st>>>(dxp, p.parts, stride, c, pos, up, unit, static_cast<T*>(dx));
}

void bind(Plan* p, const void* saved, char* scratch) {
  const char* s = static_cast<const char*>(saved);
  p->c.n_rows = reinterpret_cast<const int*>(s);
  p->c.row = reinterpret_cast<const int*>(s + p->s_row);
  p->c.label = reinterpret_cast<const int*>(s + p->s_label);
  p->c.x = s + p->s_x;
  if (p->copy_w) p->c.w = scratch + p->w;
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
  char* sv = static_cast<char*>(saved);
  char* sc = static_cast<char*>(scratch);
  bind(&p, saved, sc);
  float* each = none ? loss : nullptr;
  float* z_label = reinterpret_cast<float*>(sc + p.z_label);
  float2* part = reinterpret_cast<float2*>(sc + p.part);
  BY_TYPE(a->dtype, pack<T>(a, p, sv, sc, st));
  OK_OR("loss_pack launch failed");
  if (p.copy_w && c.n) {
    BY_TYPE(a->dtype, pad_weight<T>(a, p, sc, st));
    OK_OR("loss_pad launch failed");
  }
  if (c.n) {
    if (p.tc) {
      if (!tc_stats(c, part, z_label, st)) FAIL("loss_stats_tc5 launch failed");
    } else {
      Launch scope("loss_stats", st);
      k_stats<<<dim3(p.tiles_v, p.tiles_m), 256, 0, st>>>(c, part, z_label);
      OK_OR("loss_stats launch failed");
    }
  }
  if (c.n || !none) {
    // few rows: more lanes for the tiles of each
    const int rows = c.n >= 4096 ? 32 : c.n >= 256 ? 8 : 2;
    Launch scope("loss_join", st);
    k_join<<<(unsigned)std::max<int64_t>(1, (c.n + rows - 1) / rows), dim3(rows, 256 / rows), 0, st>>>(
        c, part, p.tiles_v, z_label, reinterpret_cast<float*>(sv + p.s_lse), each,
        reinterpret_cast<const int*>(sv + p.s_pos), reinterpret_cast<float*>(sc + p.loss), loss,
        a->reduction == GPA_B200_LOSS_MEAN, reinterpret_cast<int*>(sv) + 1);
    OK_OR("loss_join launch failed");
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
  if (!a->weight || !saved || !scratch || (c.n && !dloss) || (!dhidden && !dweight)) {
    *why = "a tensor is NULL";
    return GPA_B200_BAD_ARGUMENT;
  }
  if (saved_bytes < (size_t)p.s_bytes || scratch_bytes < (size_t)p.bwd_bytes) {
    *why = "saved or scratch is smaller than its size query";
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
  bind(&p, saved, sc);
  const float* lse = reinterpret_cast<const float*>(sv + p.s_lse);
  void* pr = sc + p.p;
  float* dxp = reinterpret_cast<float*>(sc + p.dxp);
  if (p.copy_w) {
    BY_TYPE(a->dtype, pad_weight<T>(a, p, sc, st));
    OK_OR("loss_pad launch failed");
  }
  const bool none = a->reduction == GPA_B200_LOSS_NONE;
  Upstream up = {none ? dloss : nullptr, true, none ? nullptr : dloss, a->reduction == GPA_B200_LOSS_MEAN};
  if (none && a->dtype == GPA_B200_F16) {
    float* r = reinterpret_cast<float*>(sc + p.r);
    float* s = reinterpret_cast<float*>(sc + p.scale);
    Launch scope("loss_row_scale", st);
    k_row_scale<<<1, 1024, 0, st>>>(dloss, c, r, s);
    OK_OR("loss_row_scale launch failed");
    up = {r, false, s, false};
  }
  const int64_t part_stride = c.n_pad * c.pitch;
  const unsigned tiles_d = (unsigned)((c.pitch + kB - 1) / kB);
  for (int64_t v0 = 0; v0 < c.vocab; v0 += p.piece) {
    const int64_t vn = std::min(p.piece, c.vocab - v0);
    if (p.tc) {
      if (!tc_probs(c, v0, vn, lse, up, pr, p.piece, st)) FAIL("loss_probs_tc5 launch failed");
      if (dhidden && !tc_dx(c, pr, p.piece, v0, vn, p.parts, (int)(p.k_part / 64), v0 > 0, dxp, part_stride, st))
        FAIL("loss_dx_tc5 launch failed");
      if (dweight && !tc_dw(c, pr, p.piece, v0, vn, up, dweight, st)) FAIL("loss_dw_tc5 launch failed");
      continue;
    }
    const unsigned tv = (unsigned)(vloss::up(vn, kTile) / kB);
    float* pf = static_cast<float*>(pr);
    {
      Launch scope("loss_probs", st);
      k_probs<<<dim3(tv, p.tiles_m), 256, 0, st>>>(c, v0, vn, lse, up, pf, p.piece);
      OK_OR("loss_probs launch failed");
    }
    if (dhidden) {
      Launch scope("loss_dx", st);
      k_dx<<<dim3(tiles_d, p.tiles_m, p.parts), 256, 0, st>>>(c, pf, p.piece, v0, vn, p.k_part, v0 > 0, dxp,
                                                              part_stride);
      OK_OR("loss_dx launch failed");
    }
    if (dweight) {
      Launch scope("loss_dw", st);
      k_dw<<<dim3(tiles_d, tv), 256, 0, st>>>(c, pf, p.piece, v0, vn, up, static_cast<float*>(dweight));
      OK_OR("loss_dw launch failed");
    }
  }
  if (dhidden) {
    BY_TYPE(a->dtype, finish<T>(p, dxp, part_stride, reinterpret_cast<const int*>(sv + p.s_pos), up, dhidden, st));
    OK_OR("loss_finish launch failed");
  }
  return GPA_B200_OK;
}

}  // namespace gpa
