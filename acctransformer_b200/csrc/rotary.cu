// Rotary positions with several axes: every pair of a row is turned by (the row's position on the pair's axis) * (its frequency).
//
//   y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin;   the way back of a gradient is the turn by minus the angle
//
// The frequency is the nearest fraction of a turn in units of 2^-64, so position * frequency modulo a turn is one 64-bit product, exact
// to position * 2^-65 turns whatever the position; the sine and cosine of its leading 24 bits are good to 2^-23, also where position *
// frequency in fp32 would have lost the angle (from some 10^5 on).
//
// Bound by the rows' way in and out of memory.  A thread has the same few pairs of one row in several heads, for which it takes the
// sines and cosines once; queries and keys go in one launch.
// 2 x 8 192 rows of 32 + 8 heads of 128, there and back: 115 us, 89 % of the copy rate (a loop over eight heads, each loaded when the one before
// was done: 192 us).
#include <algorithm>

#include "fa_common.cuh"
#include "linear.cuh"

namespace acct {
namespace {

constexpr int kThreads = 256;

template <int VEC>
struct Raw;
template <> struct Raw<8> { using type = uint4; };
template <> struct Raw<4> { using type = uint2; };
template <> struct Raw<2> { using type = uint32_t; };
template <> struct Raw<1> { using type = uint16_t; };

template <bool BF16, int VEC>
__device__ __forceinline__ void unpack(const typename Raw<VEC>::type& r, float (&x)[VEC]) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(&r);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = BF16 ? __uint_as_float(static_cast<uint32_t>(h[i]) << 16) : __half2float(__ushort_as_half(h[i]));
}
template <bool BF16, int VEC>
__device__ __forceinline__ typename Raw<VEC>::type repack(const float (&x)[VEC]) {
  typename Raw<VEC>::type r;
  if constexpr (VEC == 1) {
    r = static_cast<uint16_t>(pack2<BF16>(x[0], 0.f));
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<BF16>(x[2 * i], x[2 * i + 1]);
  }
  return r;
}

// A unit: VEC neighbouring values of a row (adjacent: VEC / 2 pairs), or VEC values and their VEC partners half of the turned part on;
// behind those, VEC values that are copied.  A thread has a unit of one row in HEADS heads, all of which it loads before it turns any.
// Threads are counted in 32 bits, whose division is a fraction of that in 64: see launch_heads.  WIDE: positions of 64 bits (chosen for each pair at
// run time they cost 4 %).
template <bool BF16, int VEC, bool ADJACENT, int HEADS, bool WIDE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p, unsigned int units, unsigned int turned_units,
                                                          unsigned int q_blocks) {
  using R = typename Raw<VEC>::type;
  constexpr int kPairs = ADJACENT ? VEC / 2 : VEC;
  const bool is_k = blockIdx.x >= q_blocks;
  const auto& t = is_k ? p.t[1] : p.t[0];
  const unsigned int groups = (t.heads + HEADS - 1) / HEADS;
  const unsigned int i = (blockIdx.x - (is_k ? q_blocks : 0u)) * kThreads + threadIdx.x;
  const unsigned int unit = i % units, rest = i / units;
  // (neighbouring rows lie beside each other where rows are packed by head, neighbouring heads where they are packed by row)
  const bool by_head = t.x_stride[1] < t.x_stride[2];
  const unsigned int rows = static_cast<unsigned int>(p.B) * p.S;
  const unsigned int group = by_head ? rest % groups : rest / rows, row = by_head ? rest / groups : rest % rows;
  if (group >= groups || row >= rows) return;
  const unsigned int b = row / p.S, s = row % p.S;
  const bool copied = unit >= turned_units;
  const int pair0 = unit * kPairs, half = p.rotated / 2;
  const int d = copied ? p.rotated + (unit - turned_units) * VEC : ADJACENT ? unit * VEC : pair0;
  const int h0 = group * HEADS, heads = min(HEADS, t.heads - h0);
  const uint16_t* x = static_cast<const uint16_t*>(t.x) + b * t.x_stride[0] + h0 * t.x_stride[1] + s * t.x_stride[2] + d;
  uint16_t* y = static_cast<uint16_t*>(t.y) + b * t.y_stride[0] + h0 * t.y_stride[1] + s * t.y_stride[2] + d;
  R r1[HEADS], r2[ADJACENT ? 1 : HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
    if (h < heads) {
      r1[h] = *reinterpret_cast<const R*>(x + h * t.x_stride[1]);
      if constexpr (!ADJACENT)
        if (!copied) r2[h] = *reinterpret_cast<const R*>(x + h * t.x_stride[1] + half);
    }
  if (copied) {
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
      if (h < heads) *reinterpret_cast<R*>(y + h * t.y_stride[1]) = r1[h];
    return;
  }
  float c[kPairs], sn[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int64_t at = p.axis[pair0 + j] * p.pos_stride[0] + b * p.pos_stride[1] + s * p.pos_stride[2];
    const long long pos = WIDE ? p.wide_positions[at] : p.positions[at];
    const long long turn = static_cast<long long>(static_cast<unsigned long long>(pos) * p.turns[pair0 + j]);      // of 2^64; as signed: in [-1/2, 1/2)
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * (1.f / 2147483648.f), &sn[j], &c[j]);
    if (p.inverse) sn[j] = -sn[j];
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h >= heads) break;
    uint16_t* to = y + h * t.y_stride[1];
    if constexpr (ADJACENT) {
      float v[VEC], o[VEC];
      unpack<BF16, VEC>(r1[h], v);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        o[2 * j] = v[2 * j] * c[j] - v[2 * j + 1] * sn[j];
        o[2 * j + 1] = v[2 * j + 1] * c[j] + v[2 * j] * sn[j];
      }
      *reinterpret_cast<R*>(to) = repack<BF16, VEC>(o);
    } else {
      float v1[VEC], v2[VEC], o1[VEC], o2[VEC];
      unpack<BF16, VEC>(r1[h], v1);
      unpack<BF16, VEC>(r2[h], v2);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o1[j] = v1[j] * c[j] - v2[j] * sn[j];
        o2[j] = v2[j] * c[j] + v1[j] * sn[j];
      }
      *reinterpret_cast<R*>(to) = repack<BF16, VEC>(o1);
      *reinterpret_cast<R*>(to + half) = repack<BF16, VEC>(o2);
    }
  }
}

// Batch entries b0 .. b0 + B - 1, rows s0 .. s0 + S - 1 of each.
RotaryParams part_of(const RotaryParams& p, int b0, int B, int s0, int S) {
  RotaryParams part = p;
  part.B = B;
  part.S = S;
  for (auto& t : part.t) {
    if (t.x == nullptr) continue;
    t.x = static_cast<const uint16_t*>(t.x) + b0 * t.x_stride[0] + s0 * t.x_stride[2];
    t.y = static_cast<uint16_t*>(t.y) + b0 * t.y_stride[0] + s0 * t.y_stride[2];
  }
  const int64_t at = b0 * p.pos_stride[1] + s0 * p.pos_stride[2];
  if (p.positions != nullptr) part.positions += at;
  if (p.wide_positions != nullptr) part.wide_positions += at;
  return part;
}

template <bool BF16, int VEC, bool ADJACENT, int HEADS>
cudaError_t launch_heads(const RotaryParams& p, int units, int turned_units, cudaStream_t stream) {
  int64_t threads[2];      // of a row
  for (int w = 0; w < 2; ++w) threads[w] = static_cast<int64_t>(units) * ((p.t[w].heads + HEADS - 1) / HEADS);
  // A launch has as many rows as 32 bits count the threads of (small units of few heads pass that): whole batch entries, or part of one.
  const int64_t most = ((int64_t(1) << 32) - kThreads) / std::max(threads[0], threads[1]);
  const int S = static_cast<int>(std::min<int64_t>(p.S, most)), B = static_cast<int>(std::min<int64_t>(p.B, S < p.S ? 1 : most / S));
  const auto kernel = p.wide_positions != nullptr ? rotary_kernel<BF16, VEC, ADJACENT, HEADS, true> : rotary_kernel<BF16, VEC, ADJACENT, HEADS, false>;
  for (int64_t b0 = 0; b0 < p.B; b0 += B)
    for (int64_t s0 = 0; s0 < p.S; s0 += S) {
      const RotaryParams part = part_of(p, static_cast<int>(b0), static_cast<int>(std::min<int64_t>(B, p.B - b0)), static_cast<int>(s0),
                                        static_cast<int>(std::min<int64_t>(S, p.S - s0)));
      const int64_t rows = static_cast<int64_t>(part.B) * part.S;
      unsigned int blocks[2];
      for (int w = 0; w < 2; ++w) blocks[w] = static_cast<unsigned int>((rows * threads[w] + kThreads - 1) / kThreads);
      kernel<<<blocks[0] + blocks[1], kThreads, 0, stream>>>(part, units, turned_units, blocks[0]);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

template <bool BF16, int VEC, bool ADJACENT>
cudaError_t launch(const RotaryParams& p, cudaStream_t stream) {
  const int turned_units = ADJACENT ? p.rotated / VEC : p.rotated / 2 / VEC;
  const bool in_place = p.t[0].x == p.t[0].y && p.t[1].x == p.t[1].y;      // (both null where there are no heads)
  const int units = turned_units + (in_place ? 0 : (p.D - p.rotated) / VEC);
  // Sines and cosines for four heads at a time, unless there are so few rows that a head for each thread does not fill the SMs' 148 x 2 048.
  const int64_t threads = static_cast<int64_t>(p.B) * p.S * units * (p.t[0].heads + p.t[1].heads);
  return threads > 148 * 2048 ? launch_heads<BF16, VEC, ADJACENT, 4>(p, units, turned_units, stream)
                              : launch_heads<BF16, VEC, ADJACENT, 1>(p, units, turned_units, stream);
}

template <bool BF16>
cudaError_t by_width(const RotaryParams& p, cudaStream_t stream) {
  // the widest pieces that the turned part, or each half of it, divides into
  const int part = p.adjacent ? p.rotated : p.rotated / 2;
  if (p.adjacent) return part % 8 == 0 ? launch<BF16, 8, true>(p, stream) : part % 4 == 0 ? launch<BF16, 4, true>(p, stream) : launch<BF16, 2, true>(p, stream);
  return part % 8 == 0   ? launch<BF16, 8, false>(p, stream)
         : part % 4 == 0 ? launch<BF16, 4, false>(p, stream)
         : part % 2 == 0 ? launch<BF16, 2, false>(p, stream)
                         : launch<BF16, 1, false>(p, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, bool bf16, cudaStream_t stream) { return bf16 ? by_width<true>(p, stream) : by_width<false>(p, stream); }

}  // namespace acct
