// Rotary positions with several axes: every pair of a row is turned by (the row's position on the pair's axis) * (its frequency).
//
//   y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin;   the way back of a gradient is the turn by minus the angle
//
// The frequency is a fraction of a turn in units of 2^-64, so position * frequency modulo a turn is one 64-bit product, exact
// to position * 2^-65 turns whatever the position; the sine and cosine of its leading 24 bits are good to 2^-23, also where position *
// frequency in fp32 would have lost the angle (from some 10^5 on).
//
// Bound by the rows' way in and out of memory.  A thread has the same few pairs of one row in several heads, for which it takes the
// sines and cosines once; queries and keys go in one launch.
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
// behind those, VEC values that are copied.
template <bool BF16, int VEC, bool ADJACENT>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p, int units, int turned_units, int head_blocks) {
  using R = typename Raw<VEC>::type;
  constexpr int kPairs = ADJACENT ? VEC / 2 : VEC;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int unit = static_cast<int>(i % units);
  const int64_t rest = i / units;
  const int hb = static_cast<int>(rest % head_blocks);
  const int64_t row = rest / head_blocks;
  if (row >= static_cast<int64_t>(p.B) * p.S) return;
  const int b = static_cast<int>(row / p.S), s = static_cast<int>(row % p.S);
  const bool copied = unit >= turned_units;
  const int pair0 = unit * kPairs, half = p.rotated / 2;
  const int d = copied ? p.rotated + (unit - turned_units) * VEC : ADJACENT ? unit * VEC : pair0;
  float c[kPairs], sn[kPairs];
  if (!copied) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const long long pos = p.positions[p.axis[pair0 + j] * p.pos_stride[0] + b * p.pos_stride[1] + s * p.pos_stride[2]];
      const long long turn = static_cast<long long>(static_cast<unsigned long long>(pos) * p.turns[pair0 + j]);      // of 2^64; as signed: in [-1/2, 1/2)
      sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * (1.f / 2147483648.f), &sn[j], &c[j]);
      if (p.inverse) sn[j] = -sn[j];
    }
  }
  const int heads = p.t[0].heads + p.t[1].heads;
  for (int h = hb; h < heads; h += head_blocks) {
    const int which = h >= p.t[0].heads;
    const int hh = which ? h - p.t[0].heads : h;
    const uint16_t* x = static_cast<const uint16_t*>(p.t[which].x) + b * p.t[which].x_stride[0] + hh * p.t[which].x_stride[1] + s * p.t[which].x_stride[2] + d;
    uint16_t* y = static_cast<uint16_t*>(p.t[which].y) + b * p.t[which].y_stride[0] + hh * p.t[which].y_stride[1] + s * p.t[which].y_stride[2] + d;
    const R r1 = *reinterpret_cast<const R*>(x);
    if (copied) {
      *reinterpret_cast<R*>(y) = r1;
    } else if constexpr (ADJACENT) {
      float v[VEC], o[VEC];
      unpack<BF16, VEC>(r1, v);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        o[2 * j] = v[2 * j] * c[j] - v[2 * j + 1] * sn[j];
        o[2 * j + 1] = v[2 * j + 1] * c[j] + v[2 * j] * sn[j];
      }
      *reinterpret_cast<R*>(y) = repack<BF16, VEC>(o);
    } else {
      const R r2 = *reinterpret_cast<const R*>(x + half);
      float v1[VEC], v2[VEC], o1[VEC], o2[VEC];
      unpack<BF16, VEC>(r1, v1);
      unpack<BF16, VEC>(r2, v2);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o1[j] = v1[j] * c[j] - v2[j] * sn[j];
        o2[j] = v2[j] * c[j] + v1[j] * sn[j];
      }
      *reinterpret_cast<R*>(y) = repack<BF16, VEC>(o1);
      *reinterpret_cast<R*>(y + half) = repack<BF16, VEC>(o2);
    }
  }
}

template <bool BF16, int VEC, bool ADJACENT>
cudaError_t launch(const RotaryParams& p, cudaStream_t stream) {
  const int turned_units = ADJACENT ? p.rotated / VEC : p.rotated / 2 / VEC;
  const bool in_place = p.t[0].x == p.t[0].y && p.t[1].x == p.t[1].y;      // (both null where there are no heads)
  const int units = turned_units + (in_place ? 0 : (p.D - p.rotated) / VEC);
  const int heads = p.t[0].heads + p.t[1].heads;
  const int64_t per_head = static_cast<int64_t>(p.B) * p.S * units;
  const int head_blocks = per_head >= 148 * 2048 ? (heads + 7) / 8 : per_head * heads < 148 * 2048 ? heads : (heads + 1) / 2;
  const int64_t blocks = (per_head * head_blocks + kThreads - 1) / kThreads;
  rotary_kernel<BF16, VEC, ADJACENT><<<static_cast<unsigned int>(blocks), kThreads, 0, stream>>>(p, units, turned_units, head_blocks);
  return cudaGetLastError();
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
