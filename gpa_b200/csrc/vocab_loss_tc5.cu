// The products of the vocabulary loss on the 5th-generation tensor cores (formulas in
// vocab_loss.cu): z = x W^T with the softmax statistics or with P in its epilogue, dx += P W, and
// dW = P^T x.
//
// One kernel shape serves all four: a pair of CTAs (cta_group::2) owns 256 x 256 tiles of the
// product, each CTA 128 of the rows.  A pair shares its operands: each CTA brings in its own 128
// rows of A and half of B's 256 columns (TMA, 128-byte swizzle, 64 of the reduction at a time, 6
// stages), so an SM's shared memory takes 64 bytes a cycle in and gives 64 out, which its 128
// allow; one CTA alone with the same tile would need 192.  K-major operands (x, W, P) come as
// boxes of 64 k x 128 rows, MN-major ones (W in dx, P and x in dW) as two boxes of 64 columns x
// 64 k: nothing is transposed in memory.  Two 256-column accumulators fill tensor memory: the
// epilogue warps empty one while the next tile's products go to the other.
//
//   warp 0: copies     warp 1: products (first CTA of the pair)     warp 2: tensor memory
//   warps 4-11: epilogue, two threads for each row of the tile (one: D of 135 channels leaves so few
//   products to a tile that its epilogue bounds it; 21010 x 135 x 9393 bf16 step 646 -> 612 us)
//
// Up to 128 rows of x would leave most of such a tile empty, and what counts then is how fast W
// comes by.  There z and dx are formed the other way round (kStatsT, kProbsT, kDxT): 256 vocabulary
// entries or channels by the 32 or 128 rows, so that a step of the products costs an eighth or
// half as much and more copies of W are on their way at a time.
//
// For fp32 the parts of W are then read once each instead of once for each product: a stage holds a
// part of W and every part of x that it meets (54 x 1024 x 86791: z 187 -> 173 us).
//
// fp32 inputs come as three bf16 parts, x = x0 + x1 + x2 (24 bits), in planes one behind the
// other, and each product is the six of them that matter, the smallest first: x2 y0, x1 y1, x0 y2,
// x1 y0, x0 y1, x0 y0.  The tensor core drops the bits below its accumulator's last with every
// step of 16, so a long reduction would lose what the parts gained: the accumulator is emptied
// after a segment of it and the segments are added in registers, in round-to-nearest fp32, by
// more epilogue warps (four threads a row of 256 columns, 64 registers each).  So is dW of 16-bit
// inputs over very many rows (see kSegmentDw), and so are the statistics of 16-bit inputs beyond
// 1024 channels: the loss is an fp32 result, and its error would grow with the width (2048
// channels: 1.1e-6 of the loss in one accumulator, 0.5e-6 in two).
//
// Measured (GPU time of one launch, B200): 65536 rows x 1024 channels x 151936 entries, bf16:
// statistics 16.4 ms = 1.24 PFLOP/s, P 16.7 ms, dx 15.5 ms, dW 15.3 ms (1.33 PFLOP/s; a library
// product of 8192^3 sustains 1.38 under the power limit, which bounds all four).  2048 x 2048 x
// 50000, fp16: dW 275 us = 1.53 PFLOP/s (1.65 in a burst).  1026 x 512 x 16001, fp32: dW 97 us =
// 173 TFLOP/s of fp32 products, 1040 of bf16 ones.  8 x 1024 x 151936, bf16: statistics 53 us =
// 5.9 TB/s of W.  One CTA instead of the pair was not built: its shared memory would bound it.
//
// Every wait is bounded (tc5.cuh); a wait that gives up sets the device status and the kernel
// drains and returns.
#include <cuda.h>

#include "tc5.cuh"
#include "vocab_loss.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>

namespace gpa {

__device__ int g_loss_status = 0;

namespace vloss {
namespace {

constexpr int kBK = 64;
constexpr int kHalf = 128;                        // rows of A that one CTA holds
constexpr uint32_t kOperand = kHalf * kBK * 2;    // their bytes in one stage
// Shared memory of a pair of tiles with BN columns: the stages, barriers, and for the transposed
// products a table of the rows and the square of one chunk of columns for either half.
constexpr int kSquare = 129;                      // pitch of its columns: no bank conflicts either way
template <int BN, bool SHARE>
struct Smem {
  static constexpr int kStages = BN == 256 ? 6 : BN == 128 ? (SHARE ? 4 : 7) : (SHARE ? 7 : 9);
  static constexpr uint32_t kColumns = BN / 2 * kBK * 2;
  static constexpr uint32_t kStage = kOperand + kColumns * (SHARE ? 3 : 1);
  static constexpr uint32_t kBars = kStages * kStage, kTable = kBars + 256, kSquares = kTable + BN * 16;
  static constexpr size_t kBytes = 1024 + (BN == 256 ? kTable : kSquares + 2 * 32 * kSquare * 4);
};
// Reduction blocks between two additions in registers: 512 for the six products of fp32 parts one
// after the other, 128 where the products of a part follow one another in every block (few rows,
// see below), 1024 for single products of z.
constexpr int kSegmentF32 = 8, kSegmentShare = 2, kSegment16 = 16;
// dW of 16-bit inputs: the reduction runs over the rows, and what the accumulator drops was measured
// at 1.04e-7 of the sum with every 16 of them (2^22 rows of one sign: 2.7e-2 of dW, 262144 of fp16:
// 2e-3).  Up to 65536 rows (fp16: 8192) that stays below an eighth of the half step to which dW is
// rounded; more are added up in registers 8192 at a time, which takes 3 % longer (65536 x 1024 x
// 151936: 14.8 -> 15.3 ms).
constexpr int kSegmentDw = 128;
bool long_dw(const Call& c) { return c.n > (c.dtype == GPA_B200_F16 ? 8192 : 65536); }
constexpr int kGroup = 16;  // row tiles that walk over the vocabulary together
constexpr float kLog2e = 1.4426950408889634f;

enum Mode { kStats, kProbs, kDx, kDw, kStatsT, kProbsT, kDxT };
// groups of four epilogue warps: threads that share a row of the tile
__host__ __device__ constexpr int groups_of(Mode m, bool f32) {
  return f32 ? (m >= kStatsT ? 2 : 4) : m >= kStatsT ? 1 : 2;
}
__host__ __device__ constexpr int threads_of(Mode m, bool f32) { return 128 + 128 * groups_of(m, f32); }

struct Args {
  Call c;
  Upstream up;
  int64_t v0, vn;
  int a_plane, b_plane;    // fp32: rows of a plane of the operands
  int tiles_n;             // tiles across the product's columns
  int k_blocks;            // reduction blocks of 64 (kDw: from the rows)
  // kStats
  float2* part;
  float* z_label;
  // kProbs
  const float2* lse;       // (max, 1 / sum of exp) of each row
  void* p;
  int64_t p_pitch;
  float p_scale;
  // kDx
  float* dx;
  int64_t dx_part;
  bool add;
  // kDw
  void* dw;                // of the piece
  int64_t dw_pitch;
  uint32_t idesc;
  bool f16;
};

// ------------------------------------------------------------------ pair primitives
GPA_DEV uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
GPA_DEV void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cluster address of `p` in the first CTA of the pair
GPA_DEV uint32_t in_first(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tc5::saddr(p)));
  return a;
}
GPA_DEV void tma_load(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(tc5::saddr(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
GPA_DEV void mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate));
}
// arrive on `bar` of both CTAs once the products issued so far are done
GPA_DEV void commit2(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          tc5::saddr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Hands an accumulator back.  It was read, and the reads waited for (ld32, ld8), so the arrival has no
// memory to publish; a release would first wait until the tile's results have reached memory, which
// held the accumulator 1900 cycles longer (16384 x 256 x 32000: statistics 309 -> 255 us, P 401 -> 312 us).
GPA_DEV void arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
GPA_DEV bool try_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(tc5::saddr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
GPA_DEV bool wait_cluster(uint64_t* bar, uint32_t parity) {
  if (try_cluster(bar, parity)) return true;
  const uint64_t t0 = tc5::gtime_ns();
  for (;;) {
    if (try_cluster(bar, parity)) return true;
    if (tc5::gtime_ns() - t0 > tc5::kWaitNs) return false;
  }
}

// Shared-memory descriptor of a 128-byte-swizzled operand.  K-major: rows of 128 bytes, 8-row
// groups 1024 bytes apart, a 16-wide step of k 32 bytes further.  MN-major: 128-byte rows of 64
// columns, one per k; 8-k groups 1024 bytes apart (stride), the next 64 columns 8192 bytes
// further (leading), a 16-wide step of k 2048 bytes further.
template <bool MN>
GPA_DEV uint64_t operand(uint32_t addr, int step) {
  const uint32_t a = addr + (uint32_t)step * (MN ? 2048u : 32u);
  return (uint64_t)((a & 0x3FFFFu) >> 4) | (uint64_t)(MN ? 8192u >> 4 : 1u) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

GPA_DEV void ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  __syncwarp();  // the load is the whole warp's; rows may have parted before it
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  tc5::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 8 at a time where 64 sums stay in registers: 16 would spill more of them (16384 x 1024 x 32000, fp32: P 1766
// -> 1712 us a piece).
GPA_DEV void ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  tc5::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

GPA_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The epilogues of 16-bit inputs are bound by instructions where channels are few: two values at an
// instruction where there is one, and P's factor as a term of its exponent (16384 x 256 x 32000: P 453 -> 401
// us, statistics 317 -> 309 us; with 1024 channels, under the power limit, P 848 -> 764 us).

// v log2(e) - off
GPA_DEV void scaled2(float& a, float& b, float off) {
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %2};\nmov.b64 z, {%3, %3};\n"
      "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(kLog2e), "f"(-off));
}
GPA_DEV void add2(float& a, float& b, float x, float y) {
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
GPA_DEV float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// Powers of 2 are taken of v log2(e) - base, base = m log2(e) as rounded, and so are all off by what
// that rounding left: 4e-5 at m = 1000, enough for a loss below 0.  base_rest is the factor that puts
// it right, once for a row; no m at all (-inf) has the base 0.
GPA_DEV float scaled(float m) { return __fmul_rn(m, kLog2e); }  // rounded: never part of an fma
GPA_DEV float base_of(float m) { return m == -INFINITY ? 0.f : scaled(m); }
GPA_DEV float base_rest(float m) { return m == -INFINITY ? 1.f : ex2(-fmaf(m, kLog2e, -scaled(m))); }
GPA_DEV uint32_t pack2(float a, float b, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 bytes at a time, a whole sector: an epilogue thread owns a row, so neighbouring threads do
// not share sectors and narrower accesses would move each one twice
GPA_DEV void st8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
GPA_DEV void ld8(const void* p, float* f) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
               : "l"(p)
               : "memory");
}

// ------------------------------------------------------------------ tiles
struct Tile {
  int m, n, part, k0, k1;
};

template <Mode M>
struct Walk {
  int mt, nt, total, n_rows, k_blocks, k_part;
  const Args& a;
  GPA_DEV Walk(const Args& args) : a(args) {
    n_rows = *args.c.n_rows;
    nt = args.tiles_n;
    if (M == kStatsT || M == kProbsT || M == kDxT) {
      mt = n_rows == 0 ? 0 : (int)(((M == kDxT ? args.c.pitch : args.vn) + kTile - 1) / kTile);
      nt = 1;
      k_blocks = args.k_blocks;
    } else if (M == kDw) {
      mt = (int)((args.vn + kTile - 1) / kTile);
      k_blocks = (n_rows + kBK - 1) / kBK;
    } else {
      mt = (n_rows + kTile - 1) / kTile;
      k_blocks = args.k_blocks;
    }
    constexpr bool kParts = M == kDx || M == kDxT;
    total = mt * nt * (kParts ? args.c.n_rows[2] : 1);
    k_part = kParts ? args.c.n_rows[3] : 0;
  }
  GPA_DEV Tile at(int t) const {
    Tile x;
    x.part = 0;
    x.k0 = 0;
    x.k1 = k_blocks;
    if (M == kStats || M == kProbs) {
      // kGroup row tiles side by side walk over the vocabulary, so that the tiles in flight
      // share a few tiles of x and of W in L2
      const int per = kGroup * nt, g = t / per, in = t - g * per;
      const int rows = mt - g * kGroup < kGroup ? mt - g * kGroup : kGroup;
      x.n = in / rows;
      x.m = g * kGroup + in - x.n * rows;
    } else {
      x.n = t % nt;
      x.m = t / nt;
      if (M == kDx || M == kDxT) {
        x.part = x.m / mt;
        x.m -= x.part * mt;
        x.k0 = x.part * k_part;
        x.k1 = x.k0 + k_part < k_blocks ? x.k0 + k_part : k_blocks;
      }
    }
    return x;
  }
};

// What a thread holds of its row of the tile when it is done: the columns in tensor memory (16-bit
// inputs), or the CW of them that it has added up in registers.
template <bool F32, int CW>
struct Row {
  uint32_t tmem;
  // chunk k of CH columns, to be used up: read into `buffer`, or the registers that hold it
  template <int CH>
  GPA_DEV float (&take(int k, float (&buffer)[CH]))[CH] {
    ld32(tc5::tmem_at(tmem, CH * k), buffer);
    return buffer;
  }
};
template <int CW>
struct Row<true, CW> {
  static constexpr int kCh = CW < 32 ? CW : 32;
  float acc[CW / kCh][kCh];
  template <int CH>
  GPA_DEV float (&take(int k, float (&)[CH]))[CH] {
    return acc[k];
  }
};

// What the statistics and P take from memory for a thread's row, read while the tile before is dealt
// with (16384 x 256 x 32000: statistics 255 -> 245 us, P 314 -> 308 us); not where sums fill the registers.
struct RowIn {
  int label;   // -1: no row, or no such label
  float2 lse;  // zero: no row
};
template <Mode M>
GPA_DEV RowIn row_in(const Args& a, const Tile& t, int n_rows, int rank) {
  const int64_t row = (int64_t)t.m * kTile + rank * kHalf + (threadIdx.x & 127);
  RowIn in = {-1, {0.f, 0.f}};
  if ((M == kStats || M == kProbs) && row < n_rows) {
    in.label = a.c.label[row];
    if (M == kProbs) in.lse = a.lse[row];
  }
  return in;
}

template <Mode M, bool F32, bool EXACT>
GPA_DEV void epilogue(const Args& a, const Tile& t, int n_rows, Row<F32, 64>& held, const RowIn& in, int rank,
                      bool empty) {
  constexpr int kGroups = groups_of(M, F32), kChunks = 8 / kGroups, kUnroll = F32 ? kChunks : 1;
  const int group = (threadIdx.x - 128) >> 7;  // of the tile's columns
  const int in_tile = rank * kHalf + (threadIdx.x & 127);
  const int64_t row = (int64_t)t.m * kTile + in_tile;
  const int64_t col0 = (int64_t)t.n * kTile + group * (kTile / kGroups);
  float buffer[32];
  if (M == kStats) {
    const bool live = row < n_rows;
    const int64_t y = in.label - col0;  // not in the tile when negative
    float big = -INFINITY, sum = 0.f;
#pragma unroll kUnroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 32 * k;
      float (&v)[32] = held.take(k, buffer);
      if (y >= c && y < c + 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (y == c + i) a.z_label[row] = v[i];
      }
      const int64_t left = a.c.vocab - col0 - c;
      if (left < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i >= left) v[i] = -INFINITY;
      }
      float m = big, m1 = v[0];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        m = max3(m, v[i], v[i + 1]);
        m1 = max3(m1, v[i + 2], v[i + 3]);
      }
      m = fmaxf(m, m1);
      const float safe = m == -INFINITY ? 0.f : m, off = base_of(m);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        if (F32) {  // one at a time: pairs would spill more of the sums (2048 x 2048 x 50000: 364 -> 341 us)
          s0 += EXACT ? expf(v[i] - safe) : ex2(fmaf(v[i], kLog2e, -off));
          s1 += EXACT ? expf(v[i + 1] - safe) : ex2(fmaf(v[i + 1], kLog2e, -off));
          continue;
        }
        scaled2(v[i], v[i + 1], off);
        add2(s0, s1, ex2(v[i]), ex2(v[i + 1]));
      }
      sum = fmaf(sum, EXACT ? expf(big - safe) : ex2(scaled(big) - off), s0 + s1);
      big = m;
    }
    if (!EXACT) sum *= base_rest(big);
    if (live) a.part[((int64_t)t.n * kGroups + group) * a.c.n_pad + row] = make_float2(big, sum);
  } else if (M == kProbs) {
    // P is rounded once to the type of its product's other operand, half a step of it (fp32: three
    // parts, 24 bits), without the row's gradient r: where the label's entry outweighs the others
    // it stays near -1 and its rounding is small.  fp16 takes P times 2^14 (tc_p_scale): a
    // probability of 2^-28 keeps its full precision.
    const bool live = row < n_rows;
    const float2 l = in.lse;
    const float one = live && in.label < 0 ? NAN : a.p_scale;  // no such label: the row is NaN
    const float f = l.y * one, off = EXACT ? l.x : fmaf(l.x, kLog2e, -log2f(f));
    const int64_t y = in.label - a.v0 - col0;
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p) + row * a.p_pitch + col0);
    const int64_t plane = a.c.n_pad * a.p_pitch / 2;
#pragma unroll kUnroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 32 * k;
      float (&v)[32] = held.take(k, buffer);
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        if (!EXACT) scaled2(v[i], v[i + 1], off);
        v[i] = EXACT ? expf(v[i] - off) * f : ex2(v[i]);
        v[i + 1] = EXACT ? expf(v[i + 1] - off) * f : ex2(v[i + 1]);
      }
      if (y >= c && y < c + 32) {
        // off is rounded, which moves all of a row alike: within P's own rounding, but not here, where
        // one goes off what may be nearly one
        const float base = scaled(l.x), rest = EXACT ? 1.f : ex2((off - base) + log2f(f) - fmaf(l.x, kLog2e, -base));
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (y == c + i) v[i] = fmaf(v[i], rest, -one);
      }
      const int64_t left = live ? a.vn - col0 - c : 0;
      if (left < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i >= left) v[i] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < (F32 ? 3 : 1); ++q) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          w[i] = pack2(v[2 * i], v[2 * i + 1], !F32 && a.f16);
          if (F32) {  // what this part leaves
            const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
            v[2 * i] -= g.x, v[2 * i + 1] -= g.y;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i += 8) st8(out + q * plane + c / 2 + i, w + i);
      }
    }
  } else if (M == kDx) {
    const bool live = row < n_rows;
    float* out = a.dx + t.part * a.dx_part + row * a.c.pitch + col0;
#pragma unroll kUnroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 32 * k;
      float (&v)[32] = held.take(k, buffer);
      if (!live) continue;
      const int64_t left = a.c.pitch - col0 - c;  // a multiple of 8
      if (a.add) {
        float g[32];
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          if (i < left) ld8(out + c + i, g + i);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] += g[i];
      }
#pragma unroll
      for (int i = 0; i < 32; i += 8)
        if (i < left) st8(out + c + i, reinterpret_cast<const uint32_t*>(v + i));
    }
  } else {
    const bool live = row < a.vn;
    const float s = a.up.scale(n_rows) / a.p_scale;
    const int64_t at = row * a.dw_pitch + col0;
#pragma unroll kUnroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 32 * k;
      float (&v)[32] = !F32 && empty ? buffer : held.take(k, buffer);
      if (!live) continue;
      const int64_t left = a.dw_pitch - col0 - c;  // a multiple of 8
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = empty ? 0.f : v[i] * s;
      if (EXACT) {
        float* out = static_cast<float*>(a.dw) + at + c;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          if (i < left) st8(out + i, reinterpret_cast<const uint32_t*>(v + i));
        continue;
      }
      uint16_t* out = static_cast<uint16_t*>(a.dw) + at + c;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], a.f16);
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        if (2 * i < left) *reinterpret_cast<uint4*>(out + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
}

// ---- transposed tiles: a thread's row is a vocabulary entry (or a channel), its columns are rows of x
template <bool F32, int BN>
struct Cols {
  static constexpr int kCw = F32 ? BN / 2 : BN;        // columns of a thread
  static constexpr int kCh = kCw < 32 ? kCw : 32;      // of a chunk
  static constexpr int kChunks = kCw / kCh;
  static constexpr int kLanes = 128 / kCh;             // threads that share a column of the square
};

GPA_DEV void half_sync(int half) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + half) : "memory"); }
// whether every warp of the half got its accumulator (they all wait for it, each for a limited time)
GPA_DEV bool half_all(int half, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.and.pred q, %2, 128, p;\nselp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(1 + half)
      : "memory");
  return r != 0;
}

// (max, sum of exp) of the columns over every tile of the CTA.  A chunk of columns goes through
// shared memory, so that a thread meets kCh entries of one column at a time.
template <bool F32, int BN, bool EXACT>
struct Stats {
  using C = Cols<F32, BN>;
  float big[C::kChunks], sum[C::kChunks];
  int64_t label[C::kChunks];
  int half, col, lane;  // this thread's column of a chunk, and its share of the rows

  GPA_DEV void start(const Args& a, int n_rows) {
    half = F32 ? (threadIdx.x - 128) >> 7 : 0;
    const int i = threadIdx.x & 127;
    col = i % C::kCh;
    lane = i / C::kCh;
#pragma unroll
    for (int k = 0; k < C::kChunks; ++k) {
      const int j = column(k);
      big[k] = -INFINITY, sum[k] = 0.f;
      label[k] = j < n_rows ? a.c.label[j] : -1;
    }
  }
  GPA_DEV int column(int k) const { return half * C::kCw + k * C::kCh + col; }
  GPA_DEV void tile(const Args& a, const Tile& t, Row<F32, C::kCw>& held, int rank, float* square) {
    const int r = threadIdx.x & 127;
    const int64_t base = (int64_t)t.m * kTile + rank * kHalf;
    const bool in = base + r < a.vn;
#pragma unroll
    for (int k = 0; k < C::kChunks; ++k) {
      float buffer[C::kCh];
      float (&v)[C::kCh] = held.take(k, buffer);
#pragma unroll
      for (int i = 0; i < C::kCh; ++i) square[i * kSquare + r] = in ? v[i] : -INFINITY;
      half_sync(half);
      const float* s = square + col * kSquare + lane * C::kCh;
      float m = big[k];
#pragma unroll
      for (int i = 0; i < C::kCh; ++i) {
        v[i] = s[i];
        m = fmaxf(m, v[i]);
      }
      const float safe = m == -INFINITY ? 0.f : m, off = base_of(m);
      float more = 0.f;
#pragma unroll
      for (int i = 0; i < C::kCh; ++i) more += EXACT ? expf(v[i] - safe) : ex2(fmaf(v[i], kLog2e, -off));
      sum[k] = fmaf(sum[k], EXACT ? expf(big[k] - safe) : ex2(scaled(big[k]) - off), more);
      big[k] = m;
      const int64_t y = label[k] - base - lane * C::kCh;
      if (label[k] >= 0 && y >= 0 && y < C::kCh) a.z_label[column(k)] = s[y];
      half_sync(half);
    }
  }
  GPA_DEV void finish(const Args& a, int n_rows) const {
#pragma unroll
    for (int k = 0; k < C::kChunks; ++k)
      if (column(k) < n_rows)
        a.part[((int64_t)blockIdx.x * C::kLanes + lane) * a.c.n_pad + column(k)] =
            make_float2(big[k], EXACT ? sum[k] : sum[k] * base_rest(big[k]));
  }
};

// {max (16-bit inputs: its base), factor of the exp, P's unit, label within the piece} of row j of x
template <bool F32>
GPA_DEV float4 row_of(const Args& a, int j, int n_rows) {
  if (j >= n_rows) return make_float4(0.f, 0.f, 0.f, __int_as_float(-2));  // no row
  const float2 l = a.lse[j];
  const float one = a.c.label[j] < 0 ? NAN : a.p_scale;
  const int64_t y = (int64_t)a.c.label[j] - a.v0;
  return make_float4(F32 ? l.x : scaled(l.x), F32 ? l.y * one : l.y * one * base_rest(l.x), one,
                     __int_as_float(y >= 0 && y < a.vn ? (int)y : -1));
}

template <Mode M, bool F32, int BN>
GPA_DEV void epilogue_t(const Args& a, const Tile& t, int n_rows, Row<F32, Cols<F32, BN>::kCw>& held, int rank,
                        const float4* table) {
  using C = Cols<F32, BN>;
  const int half = F32 ? (threadIdx.x - 128) >> 7 : 0;
  const int64_t at = (int64_t)t.m * kTile + rank * kHalf + (threadIdx.x & 127);
#pragma unroll
  for (int k = 0; k < C::kChunks; ++k) {
    float buffer[C::kCh];
    float (&v)[C::kCh] = held.take(k, buffer);
    const int j0 = half * C::kCw + k * C::kCh;
    if (M == kProbsT) {
      uint16_t* out = static_cast<uint16_t*>(a.p) + at;
      const int64_t plane = a.c.n_pad * a.p_pitch;
#pragma unroll
      for (int i = 0; i < C::kCh; ++i) {
        const float4 x = table[j0 + i];
        const int y = __float_as_int(x.w);
        float p = (F32 ? expf(v[i] - x.x) : ex2(fmaf(v[i], kLog2e, -x.x))) * x.y - (y == at ? x.z : 0.f);
        if (y == -2 || at >= a.vn) p = 0.f;
        uint16_t* o = out + (j0 + i) * a.p_pitch;
#pragma unroll
        for (int q = 0; q < (F32 ? 3 : 1); ++q) {
          const uint32_t b = pack2(p, 0.f, !F32 && a.f16) & 0xffffu;
          o[q * plane] = (uint16_t)b;
          if (F32) p -= __uint_as_float(b << 16);
        }
      }
      if (BN < kBK) {  // dW reduces over whole blocks of rows
#pragma unroll
        for (int i = 0; i < C::kCh; ++i)
#pragma unroll
          for (int q = 0; q < (F32 ? 3 : 1); ++q) out[(j0 + BN + i) * a.p_pitch + q * plane] = 0;
      }
    } else if (at < a.c.pitch) {
      float* out = a.dx + t.part * a.dx_part + at;
#pragma unroll
      for (int i = 0; i < C::kCh; ++i) {
        if (j0 + i >= n_rows) continue;
        float* o = out + (int64_t)(j0 + i) * a.c.pitch;
        *o = a.add ? *o + v[i] : v[i];
      }
    }
  }
}

// Planes of the products of a pair of operands, the smallest first.
GPA_DEV int plane_a(int q) { return q == 0 ? 2 : q == 1 || q == 3 ? 1 : 0; }
GPA_DEV int plane_b(int q) { return q == 2 ? 2 : q == 1 || q == 4 ? 1 : 0; }

// F32: segments added in registers; PRODUCTS: 6 for fp32 inputs (which also take the full exp), else 1
template <Mode M, bool F32, int BN, int PRODUCTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads_of(M, F32), 1)
    k_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Args a) {
  constexpr bool kT = M == kStatsT || M == kProbsT || M == kDxT;
  constexpr bool kAMn = M == kDw || M == kDxT, kBMn = M == kDx || M == kDw;
  constexpr bool kPlanes = PRODUCTS > 1, kShare = kPlanes && kT;
  constexpr int kSegment = kShare ? kSegmentShare : kPlanes ? kSegmentF32 : M == kDw ? kSegmentDw : kSegment16;
  constexpr int kPasses = kShare ? 3 : PRODUCTS;  // over a segment
  using S = Smem<BN, kShare>;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kStage = S::kStage;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::kBars);
  uint64_t *full = bars, *empty = bars + kStages, *acc_full = bars + 2 * kStages, *acc_empty = acc_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float4* table = reinterpret_cast<float4*>(sm + S::kTable);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cta_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc5::mbar_init(&full[i], 1);
      tc5::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&acc_full[i], 1);
      tc5::mbar_init(&acc_empty[i], 8 * groups_of(M, F32));  // the epilogue warps of both CTAs
    }
    tc5::mbar_fence_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc5::saddr(slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  let_next();
  after_previous();
  if (M == kProbsT)
    for (int j = threadIdx.x; j < BN; j += threads_of(M, F32)) table[j] = row_of<F32>(a, j, *a.c.n_rows);
  tc5::fence_before_sync();
  __syncthreads();
  pair_sync();
  tc5::fence_after_sync();
  const uint32_t tmem = *slot;
  const Walk<M> walk(a);
  bool ok = true;

  // The reduction of a tile goes by in segments, each into an accumulator of its own: all of it at
  // once (16-bit operands and results), or kSegment blocks times the products.
  auto segment_end = [](int k, int k1) { return F32 && k + kSegment < k1 ? k + kSegment : k1; };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      for (int t = pair; t < walk.total && ok; t += pairs) {
        const Tile x = walk.at(t);
        const int ra = x.m * kTile + rank * kHalf, rb = x.n * BN + rank * (BN / 2);
        // the piece's vocabulary entries are rows of W, whichever operand it is
        const int va = kT ? (int)a.v0 : 0, vb = M == kStats || M == kProbs || M == kDx ? (int)a.v0 : 0;
        for (int k0 = x.k0; k0 < x.k1 && ok; k0 = segment_end(k0, x.k1)) {
          const int blocks = segment_end(k0, x.k1) - k0;
          for (int j = 0; j < blocks * kPasses; ++j, ++it) {
            const int q = kPlanes ? j / blocks : 0, k = k0 + j - q * blocks;
            const uint32_t s = it % kStages, turn = it / kStages;
            if (turn && !(ok = tc5::mbar_wait(&empty[s], (turn - 1) & 1))) break;
            unsigned char* sa = sm + s * kStage;
            unsigned char* sb = sa + kOperand;
            const uint32_t bar = in_first(&full[s]);
            const int parts_b = kShare ? q + 1 : 1;  // part 2 of W meets part 0 of x, part 1 two, part 0 all
            if (rank == 0) tc5::mbar_expect_tx(&full[s], 2 * (kOperand + parts_b * S::kColumns));
            const int kk = k * kBK, pa = va + (kShare ? 2 - q : kPlanes ? plane_a(q) : 0) * a.a_plane;
            const int pb = vb + (kPlanes && !kShare ? plane_b(q) * a.b_plane : 0);
            if (kAMn) {
              tma_load(sa, &map_a, ra, pa + kk, bar);
              tma_load(sa + kOperand / 2, &map_a, ra + 64, pa + kk, bar);
            } else {
              tma_load(sa, &map_a, kk, pa + ra, bar);
            }
            if (kBMn) {
              tma_load(sb, &map_b, rb, pb + kk, bar);
              tma_load(sb + kOperand / 2, &map_b, rb + 64, pb + kk, bar);
            } else {
              for (int b = 0; b < parts_b; ++b)
                tma_load(sb + b * S::kColumns, &map_b, kk, pb + b * a.b_plane + rb, bar);
            }
          }
        }
      }
      // no copy is in flight when the pair leaves (after a wait that gave up, too)
      if (rank == 0)
        for (uint32_t j = it > kStages ? it - kStages : 0; j < it; ++j)
          ok = tc5::mbar_wait(&full[j % kStages], (j / kStages) & 1) && ok;
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t it = 0, count = 0;
      for (int t = pair; t < walk.total && ok; t += pairs) {
        const Tile x = walk.at(t);
        for (int k0 = x.k0; k0 < x.k1 && ok; k0 = segment_end(k0, x.k1), ++count) {
          const uint32_t buf = count & 1, use = count >> 1;
          if (use && !(ok = wait_cluster(&acc_empty[buf], (use - 1) & 1))) break;
          tc5::fence_after_sync();
          const int blocks = segment_end(k0, x.k1) - k0, steps = blocks * kPasses;
          for (int j = 0; j < steps; ++j, ++it) {
            const uint32_t s = it % kStages;
            if (!(ok = tc5::mbar_wait(&full[s], (it / kStages) & 1))) break;
            tc5::fence_after_sync();
            const uint32_t sa = tc5::saddr(sm + s * kStage), sb = sa + kOperand;
            const int last = kShare ? j / blocks : 0;  // parts of x in the stage, the smallest product first
            for (int b = last; b >= 0; --b)
#pragma unroll
              for (int ks = 0; ks < kBK / 16; ++ks)
                mma2(tmem + buf * kTile, operand<kAMn>(sa, ks), operand<kBMn>(sb + b * S::kColumns, ks), a.idesc,
                     j > 0 || b < last || ks > 0);
            commit2(&empty[s]);
          }
          if (ok) commit2(&acc_full[buf]);
        }
      }
    }
  } else if (warp >= 4) {
    using C = Cols<F32, BN>;
    static_assert(!kT || 128 % C::kLanes == 0, "a half's threads share the columns of a chunk evenly");
    constexpr int kCw = kT ? C::kCw : 64;  // columns that a thread adds up
    uint32_t count = 0;
    const int half = (warp - 4) >> 2;
    Stats<F32, BN, kPlanes> stats;
    float* square = reinterpret_cast<float*>(sm + S::kSquares) + half * 32 * kSquare;
    if constexpr (M == kStatsT) stats.start(a, walk.n_rows);
    constexpr bool kAhead = !F32 && (M == kStats || M == kProbs);
    RowIn next = {};
    if (kAhead && pair < walk.total) next = row_in<M>(a, walk.at(pair), walk.n_rows, rank);
    for (int t = pair; t < walk.total && ok; t += pairs) {
      const Tile x = walk.at(t);
      const RowIn in = next;
      if (kAhead && t + pairs < walk.total) next = row_in<M>(a, walk.at(t + pairs), walk.n_rows, rank);
      Row<F32, kCw> held;
      const bool none = x.k0 >= x.k1;  // no labelled row (kDw), or no entry of the piece (dx)
      if (none && M != kDw) continue;
      auto done = [&](bool empty) {
        if constexpr (M == kStatsT) stats.tile(a, x, held, rank, square);
        else if constexpr (kT) epilogue_t<M, F32, BN>(a, x, walk.n_rows, held, rank, table);
        else
          epilogue<M, F32, kPlanes>(a, x, walk.n_rows, held, kAhead ? in : row_in<M>(a, x, walk.n_rows, rank), rank,
                                    empty);
      };
      for (int k0 = x.k0; k0 < x.k1; k0 = segment_end(k0, x.k1), ++count) {
        const uint32_t buf = count & 1, use = count >> 1;
        ok = __all_sync(0xffffffffu, tc5::mbar_wait(&acc_full[buf], use & 1));
        if (M == kStatsT) ok = half_all(half, ok);
        if (!ok) break;
        tc5::fence_after_sync();
        if constexpr (F32) {
#pragma unroll
          for (int c = 0; c < kCw; c += 8) {
            float v[8];
            ld8(tc5::tmem_at(tmem, buf * kTile + half * kCw + c), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float& sum = held.acc[(c + i) / held.kCh][(c + i) % held.kCh];
              sum = k0 == x.k0 ? v[i] : sum + v[i];
            }
          }
        } else {
          held.tmem = tmem + buf * kTile + (kT ? 0 : half * (kTile / groups_of(M, F32)));
          done(false);
        }
        tc5::fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_first(in_first(&acc_empty[buf]));
      }
      if (ok && (F32 || none)) done(none);
    }
    if constexpr (M == kStatsT) stats.finish(a, walk.n_rows);
  }
  if (!ok) g_loss_status = GPA_B200_DEVICE_TIMEOUT;
  tc5::fence_before_sync();
  __syncthreads();
  pair_sync();
  tc5::fence_after_sync();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------------ host
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static std::atomic<EncodeFn> fn{nullptr};
  EncodeFn f = fn.load(std::memory_order_relaxed);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    f = reinterpret_cast<EncodeFn>(p);
    fn.store(f, std::memory_order_relaxed);
  }
  return f;
}

// [outer][inner] of 16-bit values, rows `pitch` elements apart, in boxes of 64 x `rows`
bool make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int64_t pitch, int rows, bool f16) {
  EncodeFn f = encoder();
  int dev = 0;
  // the encoder is a driver call and wants a current context, which a thread's first runtime call
  // on the device makes (a backward runs on a thread of its own)
  if (!f || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)rows}, one[2] = {1, 1};
  return f(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base),
           dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint32_t idesc_of(const Call& c, int columns, bool a_mn, bool b_mn) {
  uint32_t d = tc5::idesc_bf16(2 * kHalf, columns, a_mn, b_mn);
  if (c.dtype == GPA_B200_F16) d &= ~((1u << 7) | (1u << 10));  // both operands fp16
  return d;
}

int64_t w_rows(const Call& c) { return c.planes > 1 ? c.planes * up(c.vocab, kTile) : c.vocab; }

Args base_args(const Call& c) {
  Args a;
  std::memset(&a, 0, sizeof(a));
  a.c = c;
  a.f16 = c.dtype == GPA_B200_F16;
  a.p_scale = tc_p_scale(c.dtype);
  a.k_blocks = (c.pitch + kBK - 1) / kBK;
  a.a_plane = (int)c.n_pad;
  a.b_plane = (int)up(c.vocab, kTile);
  return a;
}

template <Mode M, bool F32, int BN, int PRODUCTS>
bool launch_as(const char* name, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int64_t tiles,
               cudaStream_t st) {
  constexpr int kSmem = (int)Smem<BN, (PRODUCTS > 1 && M >= kStatsT)>::kBytes;
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may take its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(k_product<M, F32, BN, PRODUCTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) !=
        cudaSuccess)
      return false;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int pairs = (int)std::min<int64_t>(tiles, tc_pairs());
  Launch scope(name, st);
  return launch_next(k_product<M, F32, BN, PRODUCTS>, 2 * pairs, threads_of(M, F32), kSmem, st, ma, mb, a);
}

bool exact_stats(const Call& c) { return c.dtype == GPA_B200_F32 || c.pitch > kSegment16 * kBK; }

template <Mode M, int BN>
bool launch(const char* name, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int64_t tiles,
            cudaStream_t st) {
  if (a.c.dtype == GPA_B200_F32) return launch_as<M, true, BN, 6>(name, ma, mb, a, tiles, st);
  if constexpr (M == kStats || M == kStatsT)
    if (exact_stats(a.c)) return launch_as<M, true, BN, 1>(name, ma, mb, a, tiles, st);
  if constexpr (M == kDw)
    if (long_dw(a.c)) return launch_as<M, true, BN, 1>(name, ma, mb, a, tiles, st);
  return launch_as<M, false, BN, 1>(name, ma, mb, a, tiles, st);
}

// z as W x^T for few rows: the map of W in boxes of 128 rows, of x in boxes of half the columns
template <Mode M>
bool launch_z_t(const char* name, Args a, cudaStream_t st) {
  const Call& c = a.c;
  const bool f16 = c.dtype == GPA_B200_F16;
  CUtensorMap ma, mb;
  if (!make_map(&ma, c.w, c.pitch, w_rows(c), c.w_pitch, kHalf, f16) ||
      !make_map(&mb, c.x, c.pitch, c.planes * c.n_pad, c.pitch, c.few / 2, f16))
    return false;
  std::swap(a.a_plane, a.b_plane);
  a.idesc = idesc_of(c, c.few, false, false);
  const int64_t tiles = (a.vn + kTile - 1) / kTile;
  return c.few == 32 ? launch<M, 32>(name, ma, mb, a, tiles, st) : launch<M, 128>(name, ma, mb, a, tiles, st);
}

}  // namespace

float tc_p_scale(int dtype) { return dtype == GPA_B200_F16 ? 16384.f : 1.f; }

int tc_pairs() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 74;
  int n = known[dev].load(std::memory_order_relaxed);
  if (!n) {
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (sms / 2));
    constexpr int kSmem = (int)Smem<256, false>::kBytes;
    cfg.blockDim = dim3(threads_of(kStats, false));
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    auto* kernel = k_product<kStats, false, 256, 1>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = std::max(1, sms / 2);
    }
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int tc_stats_parts(const Call& c) {
  const int64_t tiles = (c.vocab + kTile - 1) / kTile;
  const bool exact = exact_stats(c);
  if (!c.few) return (int)tiles * groups_of(kStats, exact);
  const int lanes = exact && c.few == 32 ? Cols<true, 32>::kLanes : Cols<false, 32>::kLanes;
  return (int)(2 * std::min<int64_t>(tiles, tc_pairs())) * lanes;
}

bool tc_stats(const Call& c, float2* part, float* z_label, cudaStream_t st) {
  const bool f16 = c.dtype == GPA_B200_F16;
  if (c.few) {
    Args a = base_args(c);
    a.part = part;
    a.z_label = z_label;
    a.vn = c.vocab;
    return launch_z_t<kStatsT>("loss_stats_tc5", a, st);
  }
  CUtensorMap ma, mb;
  if (!make_map(&ma, c.x, c.pitch, c.planes * c.n_pad, c.pitch, kHalf, f16) ||
      !make_map(&mb, c.w, c.pitch, w_rows(c), c.w_pitch, kHalf, f16))
    return false;
  Args a = base_args(c);
  a.part = part;
  a.z_label = z_label;
  a.tiles_n = (int)((c.vocab + kTile - 1) / kTile);
  a.idesc = idesc_of(c, kTile, false, false);
  return launch<kStats, 256>("loss_stats_tc5", ma, mb, a, (int64_t)a.tiles_n * (c.n_pad / kTile), st);
}

bool tc_probs(const Call& c, int64_t v0, int64_t vn, const float2* lse, void* p, int64_t p_pitch, cudaStream_t st) {
  const bool f16 = c.dtype == GPA_B200_F16;
  Args a = base_args(c);
  a.v0 = v0;
  a.vn = vn;
  a.lse = lse;
  a.p = p;
  a.p_pitch = p_pitch;
  if (c.few) return launch_z_t<kProbsT>("loss_probs_tc5", a, st);
  CUtensorMap ma, mb;
  if (!make_map(&ma, c.x, c.pitch, c.planes * c.n_pad, c.pitch, kHalf, f16) ||
      !make_map(&mb, c.w, c.pitch, w_rows(c), c.w_pitch, kHalf, f16))
    return false;
  a.tiles_n = (int)((vn + kTile - 1) / kTile);
  a.idesc = idesc_of(c, kTile, false, false);
  return launch<kProbs, 256>("loss_probs_tc5", ma, mb, a, (int64_t)a.tiles_n * (c.n_pad / kTile), st);
}

bool tc_dx(const Call& c, const void* p, int64_t p_pitch, int64_t v0, int64_t vn, int most_parts, bool add,
           float* dx, int64_t dx_part, cudaStream_t st) {
  const bool f16 = c.dtype == GPA_B200_F16;
  CUtensorMap ma, mb;
  if (!make_map(&ma, p, p_pitch, c.planes * c.n_pad, p_pitch, c.few ? c.few / 2 : kHalf, f16) ||
      !make_map(&mb, c.w, c.pitch, w_rows(c), c.w_pitch, kBK, f16))
    return false;
  Args a = base_args(c);
  a.v0 = v0;
  a.vn = vn;
  a.k_blocks = (int)((vn + kBK - 1) / kBK);
  a.dx = dx;
  a.dx_part = dx_part;
  a.add = add;
  a.tiles_n = (c.pitch + kTile - 1) / kTile;
  if (c.few) {  // dx^T = W^T P^T: the operands change places
    std::swap(a.a_plane, a.b_plane);
    a.idesc = idesc_of(c, c.few, true, false);
    const int64_t tiles = (int64_t)a.tiles_n * most_parts;
    return c.few == 32 ? launch<kDxT, 32>("loss_dx_tc5", mb, ma, a, tiles, st)
                       : launch<kDxT, 128>("loss_dx_tc5", mb, ma, a, tiles, st);
  }
  a.idesc = idesc_of(c, kTile, false, true);
  return launch<kDx, 256>("loss_dx_tc5", ma, mb, a, (int64_t)a.tiles_n * (c.n_pad / kTile) * most_parts, st);
}

bool tc_dw(const Call& c, const void* p, int64_t p_pitch, int64_t v0, int64_t vn, const void* x, const Upstream& up,
           void* dw, int64_t dw_pitch, cudaStream_t st) {
  const bool f16 = c.dtype == GPA_B200_F16;
  CUtensorMap ma, mb;
  // p may start inside the piece: no more columns than are read
  if (!make_map(&ma, p, vloss::up(vn, kTile), c.planes * c.n_pad, p_pitch, kBK, f16) ||
      !make_map(&mb, x, c.pitch, c.planes * c.n_pad, c.pitch, kBK, f16))
    return false;
  Args a = base_args(c);
  a.v0 = v0;
  a.vn = vn;
  a.up = up;
  a.dw = dw;
  a.b_plane = (int)c.n_pad;
  a.dw_pitch = dw_pitch;
  a.tiles_n = (c.pitch + kTile - 1) / kTile;
  a.idesc = idesc_of(c, kTile, true, true);
  return launch<kDw, 256>("loss_dw_tc5", ma, mb, a, (int64_t)a.tiles_n * ((vn + kTile - 1) / kTile), st);
}

}  // namespace vloss

int loss_device_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_loss_status, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_loss_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace gpa
