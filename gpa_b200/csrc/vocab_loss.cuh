// Softmax cross entropy over a vocabulary: shapes and buffers shared by its kernels
// (vocab_loss.cu: rows and joins; see there for the formulas).
#pragma once
#include "../../include/gpa_b200.h"
#include "common.cuh"

namespace gpa {
namespace vloss {

constexpr int kTile = 256;       // rows and vocabulary entries are padded to tiles of this

// One call, as its kernels see it.  Rows are the labelled rows only, packed to the front; their
// number is known on the device alone (n_rows).
struct Call {
  int64_t n;          // rows of the caller (an upper bound of the packed ones)
  int64_t vocab;
  int width, pitch;   // channels, and the element pitch of the packed rows
  int dtype;
  int planes;         // parts of each value: 1, or the 3 bf16 parts of fp32 (x, W and P in planes of n_pad rows,
                      // of vocab rounded up to tiles, and of n_pad rows)
  const int* n_rows;  // device: packed rows, counter of k_join, parts of dx, reduction blocks of a part
  const int* label;   // [n] label of a packed row, -1 when outside the vocabulary
  const int* row;     // [n] the caller's row of a packed row
  const void* x;      // packed rows [n_pad][pitch], zero behind the last one up to a multiple of 64
  const void* w;      // weight [vocab][w_pitch], 16-bit elements
  int64_t w_pitch;
  int64_t n_pad;      // n rounded up to tiles
  int few;            // 32 or 128: at least n, and z and dx are formed transposed; 0: more rows
};

// The gradient of a packed row's loss, s r:
//   r: 1 (each == NULL), each[row] (by_row) or each[packed row]
//   s: *s (1 if NULL), over the number of labelled rows for a mean
struct Upstream {
  const float* each;
  bool by_row;
  const float* s;
  bool mean;
  __device__ __forceinline__ float r(const Call& c, int64_t j) const {
    return !each ? 1.f : each[by_row ? c.row[j] : j];
  }
  __device__ __forceinline__ float scale(int n_rows) const {
    return (s ? *s : 1.f) / (mean ? (float)(n_rows > 0 ? n_rows : 1) : 1.f);
  }
};

__host__ __device__ inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// How the reduction of dx is cut: into the parts whose turns of the whole GPU, and passes over dx in
// fp32 to add them up, take least.  Decided on the device, where the number of packed rows is
// known; n_rows[2] holds the parts and n_rows[3] the reduction blocks (of 64) of each.
struct Split {
  int tiles_d, at_once;  // tiles across dx, tiles that run at a time
  int blocks;            // reduction blocks of 64 that the first piece has
  int most;              // parts that the buffer holds
  float turn, pass;      // seconds of a turn over a piece, and of writing and reading one part's tile row
  int parts, k_part;     // decided on the host where one row of tiles is all there can be (parts > 0)
};
__host__ __device__ inline int parts_of(const Split& s, int tiles_m, int* k_part) {
  int parts = 1;
  float cost = 3e38f;
  for (int n = 1; n <= s.most; ++n) {
    const int turns = (s.tiles_d * tiles_m * n + s.at_once - 1) / s.at_once;
    const float now = (float)turns / n * s.turn + n * tiles_m * s.pass;
    if (now < cost) cost = now, parts = n;
  }
  *k_part = (s.blocks + parts - 1) / parts;
  return (s.blocks + *k_part - 1) / *k_part;
}

// The kernels of a call follow one another closely: each lets the next one start its blocks
// (let_next) and does what needs no results first, then waits until everything before it on the
// stream is done (after_previous, by every thread, before its first access to global memory).
// 8 x 1024 x 151936 scores: 67.3 -> 63.9 us; 2457 x 1000 x 32003 step: 663 -> 643 us.
GPA_DEV void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
GPA_DEV void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that calls after_previous; any other kernel is launched the usual way.
template <typename... P, typename... A>
bool launch_next(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess;
}

// The products, on tensor cores (vocab_loss_tc5.cu); false when a launch failed.
// They tile by kTile x kTile and pair up the SMs: tc_pairs() tiles run at a time.
int tc_pairs();
int tc_stats_parts(const Call& c);  // (max, sum) pairs of a row that tc_stats leaves
float tc_p_scale(int dtype);  // P is stored times this
bool tc_stats(const Call& c, float2* part, float* z_label, cudaStream_t st);
bool tc_probs(const Call& c, int64_t v0, int64_t vn, const float2* lse, void* p, int64_t p_pitch, cudaStream_t st);
bool tc_dx(const Call& c, const void* p, int64_t p_pitch, int64_t v0, int64_t vn, int most_parts, bool add,
           float* dx, int64_t dx_part, cudaStream_t st);
// dW of a piece, from x or its rows times their r (the same planes); its rows are a multiple of 8 values long and start on 16 bytes (fp32: 32)
bool tc_dw(const Call& c, const void* p, int64_t p_pitch, int64_t v0, int64_t vn, const void* x, const Upstream& up,
           void* dw, int64_t dw_pitch, cudaStream_t st);

}  // namespace vloss

int loss_device_status(bool clear);
int loss_cut(const GpaLossArgs* a, int64_t labelled, int64_t* cut, const char** why);
int loss_forward(const GpaLossArgs* a, float* loss, void* saved, size_t saved_bytes, void* scratch,
                 size_t scratch_bytes, cudaStream_t st, const char** why);
int loss_backward(const GpaLossArgs* a, const void* saved, size_t saved_bytes, const float* dloss,
                  void* dhidden, void* dweight, void* scratch, size_t scratch_bytes, cudaStream_t st,
                  const char** why);
size_t loss_saved_bytes(const GpaLossArgs* a);
size_t loss_scratch_bytes(const GpaLossArgs* a, int backward);

}  // namespace gpa
