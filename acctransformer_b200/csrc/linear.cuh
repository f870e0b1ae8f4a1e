// Parameter blocks and launchers of linear attention and of rotary positions (internal to the library).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace acct {

constexpr int kLinMaxHeadDim = 128;
constexpr int kLinChunk = 128;      // rows that the products of one chunk take

// One operand of a pass: its map (column, row, head, batch entry), boxes of 64 columns and kLinChunk rows; head h of the pass reads head
// h / group.
struct LinOperand {
  CUtensorMap map;
  int group;
};

// y_t = scale * sum over i <= t (or i >= t, reverse) of exp(g |t - i|) (a_t . b_i) c_i.  The forward is (q, k, v); of the gradients dq is
// (dy, v, k), dk (v, dy, q) reversed and dv (k, q, dy) reversed: one computation serves all four.
struct LinPass {
  LinOperand a, b, c;
  CUtensorMap map_y;                // (unused where y is fp32)
  void* y;
  int64_t y_stride[3];              // of batch entry, head and row
  int y_f32;                        // y is fp32 (partial gradients of shared heads), rows at multiples of 32 bytes
  int y_wide;                       // 16-bit rows and heads begin at multiples of 32 bytes
  int reverse;
};

struct alignas(64) LinParams {
  LinPass pass[3];
  int passes;
  int B, N, S, D;                   // S: rows of an operand (all sequences' together, where they are packed)
  const float* log_decay;           // [N]
  const int* cu;                    // [B + 1]: sequence b has rows cu[b] .. cu[b + 1] - 1 of batch entry 0; or null ...
  const int* lens;                  // ... [B]: rows 0 .. lens[b] - 1 of batch entry b; or null: all S
  const float* state_in;            // [B, N, D, D] or null: zeros (one pass, not reversed)
  float* state_out;                 // may be state_in
  float scale;
  unsigned int* status;
  // Sequences cut into segments of so many chunks; 0: whole.  The slots hold a state for each pass, segment and head, [slots, passes, N, D, D]:
  // first what a segment alone leaves, then what is before it (the first one's is a copy of state_in).
  int seg_chunks, seg_slots;
  float* seg_states;
};

// exp(g n) as the sum of two numbers.  Where it is near 1 it multiplies the same state over and over, and an error of a rounding each time
// would add up: there expm1 has the distance to 1, of which the leading number takes what it can.
struct LinPower {
  float hi, lo;
};
__device__ __forceinline__ LinPower lin_power(float g, int n) {
  if (n == 0) return {1.f, 0.f};
  const float m = static_cast<float>(n), x = g * m;
  const float rest = x == -INFINITY ? 0.f : fmaf(g, m, -x);
  if (x < -0.5f) {
    const float e = expf(x);
    return {fmaf(e, rest, e), 0.f};
  }
  const float e = expm1f(x), d = fmaf(1.f + e, rest, e), hi = 1.f + d;
  return {hi, d - (hi - 1.f)};
}

// rows of sequence b: the first, and how many; whatever cu and lens hold, no row outside [0, S) is touched
__device__ __forceinline__ void lin_rows(const LinParams& p, int b, int& row0, int& n) {
  if (p.cu != nullptr) {
    row0 = min(max(p.cu[b], 0), p.S);
    n = min(max(p.cu[b + 1], row0), p.S) - row0;
  } else {
    row0 = 0;
    n = p.lens != nullptr ? min(max(p.lens[b], 0), p.S) : p.S;
  }
}

// How long sequences are cut (LinParams::seg_chunks and seg_slots; 0: not at all) where there are too few heads for the SMs.
void linear_segments(LinParams& p, int sm_count);
inline size_t linear_segment_bytes(const LinParams& p) {
  return static_cast<size_t>(p.seg_slots) * p.passes * p.N * p.D * p.D * 4;
}
cudaError_t launch_linear(const LinParams& p, bool bf16, cudaStream_t stream);

// out[b, h, s, :] = the sum over the `group` heads of parts[b, h * group + i, s, :] in their order, rounded once
struct LinReduce {
  const float* parts[2];            // fp32 [B, N_kv * group, S, D] packed
  void* out[2];
  int64_t out_stride[3];
  const int* lens;
  int B, N_kv, group, S, D;
};
cudaError_t launch_linear_reduce(const LinReduce& p, bool bf16, cudaStream_t stream);

struct LinStepParams {
  const void *q, *k, *v;
  void* y;
  float* state;
  const float* log_decay;
  int64_t q_stride[2], k_stride[2], v_stride[2];      // of sequence and head
  int B, N, D, group;
  float scale;
};
cudaError_t launch_linear_step(const LinStepParams& p, bool bf16, cudaStream_t stream);

// A pair (x1, x2) turned by position * frequency.  Rows are (batch entry, row); x[2]: the queries and the keys.
struct RotaryParams {
  struct {
    const void* x;
    void* y;
    int64_t x_stride[3], y_stride[3];      // of batch entry, head, row
    int heads;
  } t[2];
  const int* positions;             // [axes] x rows, with element strides
  int64_t pos_stride[3];            // of axis, batch entry, row
  const unsigned long long* turns;  // [rotated / 2]: turns per position, as a fraction of 2^64
  const int* axis;                  // [rotated / 2]
  int B, S, D, rotated;
  int adjacent, inverse;
  const long long* wide_positions;  // in the place of positions: of 64 bits
};
cudaError_t launch_rotary(const RotaryParams& p, bool bf16, cudaStream_t stream);

}  // namespace acct
