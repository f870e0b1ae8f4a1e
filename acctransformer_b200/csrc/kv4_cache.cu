// Rows into the 4-bit cache, and back out of it (kv4_common.cuh has the layout).
//
// Both are bound by memory: 16 bits in and 5 out a value, or the other way round.  A warp takes one record of one head, so that
// the minimum and maximum of a group are a few shuffles, and every lane ends up with the very words that it writes.  Where only
// some of a record's rows are meant (a single token, the ends of a prompt) it loads and stores those and leaves the others alone.
#include "fa_common.cuh"
#include "fa_kernels.cuh"
#include "kv4_common.cuh"

namespace acct {
namespace {

constexpr int kRowsWarps = 8;       // per block

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t x) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  else return __half2float(__ushort_as_half(x));
}
// two-wide minimum and maximum that keep a NaN
template <bool BF16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Smallest (low half) and largest (high half) of the two halves of `lo` and of `hi`.
template <bool BF16>
__device__ __forceinline__ uint32_t fold(uint32_t lo, uint32_t hi) {
  return __byte_perm(min2<BF16>(lo, lo >> 16), max2<BF16>(hi, hi >> 16), 0x5410);
}
// ... and of two lanes'
template <bool BF16>
__device__ __forceinline__ uint32_t fold_lanes(uint32_t mm, int bit) {
  const uint32_t other = __shfl_xor_sync(0xffffffffu, mm, bit);
  return __byte_perm(min2<BF16>(mm, other), max2<BF16>(mm, other), 0x7610);
}

struct Group {
  uint16_t step, low;
  float low_f, inv;
};
// Step and minimum of a group from its extremes.  The step is rounded down, so that no value of the group (15 steps above the
// minimum at most) can leave the 16-bit type.  A group with a value that is not finite gets a NaN for its step.
template <bool BF16>
__device__ __forceinline__ Group make_group(uint32_t mm) {
  Group g;
  g.low = static_cast<uint16_t>(mm & 0xffffu);
  g.low_f = to_float<BF16>(g.low);
  const float range = __fsub_rn(to_float<BF16>(static_cast<uint16_t>(mm >> 16)), g.low_f);
  const float want = __fdiv_rn(range, 15.0f);
  if constexpr (BF16) g.step = __bfloat16_as_ushort(__float2bfloat16_rz(want));
  else g.step = __half_as_ushort(__float2half_rz(want));
  if (!(range < INFINITY)) g.step = 0x7fff;
  const float s = to_float<BF16>(g.step);
  g.inv = s > 0.f ? fminf(__fdiv_rn(1.0f, s), 3.4028235e38f) : 0.f;
  return g;
}
// Code of x: round((x - minimum) / step), half to even, at most 15.  Adding 1.5 * 2^23 leaves the integer in the low bits.
__device__ __forceinline__ uint32_t code_of(float x, const Group& g) {
  const float v = fminf(__fmul_rn(__fsub_rn(x, g.low_f), g.inv), 15.0f);
  return __float_as_uint(__fadd_rn(v, 12582912.0f)) & 15u;
}

// NG neighbouring words
template <int NG>
__device__ __forceinline__ void store_words(uint8_t* rec, int w, int place, const uint32_t (&x)[NG]) {
  using R = Kv4Record<NG>;
  if constexpr (NG == 4) *reinterpret_cast<uint4*>(rec + R::word(w, place)) = make_uint4(x[0], x[1], x[2], x[3]);
  else if constexpr (NG == 2) *reinterpret_cast<uint2*>(rec + R::word(w, place)) = make_uint2(x[0], x[1]);
  else {
#pragma unroll
    for (int i = 0; i < NG; ++i) *reinterpret_cast<uint32_t*>(rec + R::word(w + i, place)) = x[i];
  }
}
template <int NG>
__device__ __forceinline__ void load_words(const uint8_t* rec, int w, int place, uint32_t (&x)[NG]) {
  using R = Kv4Record<NG>;
  if constexpr (NG == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(rec + R::word(w, place));
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else if constexpr (NG == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(rec + R::word(w, place));
    x[0] = v.x; x[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < NG; ++i) x[i] = *reinterpret_cast<const uint32_t*>(rec + R::word(w + i, place));
  }
}

// Which record of which sequence the `item`-th one is that holds any of the rows, and what of it: slots [lo, hi) of the sequence
// are meant, and slot s is row s + shift.  Lane by lane over the sequences, 32 at a time; the same in all lanes.
struct Piece {
  int b, rec, lo, hi, shift;
};
__device__ __forceinline__ bool find_piece(const Kv4Rows& r, int B, int S_max, int item, Piece& out) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < B; b0 += 32) {
    if (r.cu == nullptr) b0 = item & ~31;      // a row per sequence: item b is sequence b
    if (b0 >= B) return false;
    const int b = b0 + lane;
    int lo = 0, hi = 0, shift = 0, n = 0;
    if (b < B) {
      int row0 = b, row1 = b + 1;
      if (r.cu != nullptr) {                   // (whatever they hold, no row outside [0, T) is touched)
        row0 = min(max(r.cu[b], 0), r.T);
        row1 = min(max(r.cu[b + 1], row0), r.T);
      }
      const int start = r.start[b];
      shift = row0 - start;
      lo = max(start, 0);
      hi = static_cast<int>(min(static_cast<int64_t>(start) + (row1 - row0), static_cast<int64_t>(S_max)));
      if (hi > lo) n = (hi - 1) / kKv4Rows - lo / kKv4Rows + 1;
    }
    int from = lane;
    if (r.cu != nullptr) {
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      const unsigned int past = __ballot_sync(0xffffffffu, upto > item);
      if (past == 0u) {
        item -= __shfl_sync(0xffffffffu, upto, 31);
        continue;
      }
      from = __ffs(past) - 1;
      item -= __shfl_sync(0xffffffffu, upto - n, from);
    } else {
      from = item & 31;
      if (__shfl_sync(0xffffffffu, n, from) == 0) return false;
      item = 0;
    }
    out.b = b0 + from;
    out.lo = __shfl_sync(0xffffffffu, lo, from);
    out.hi = __shfl_sync(0xffffffffu, hi, from);
    out.shift = __shfl_sync(0xffffffffu, shift, from);
    out.rec = out.lo / kKv4Rows + item;
    return true;
  }
  return false;
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_append_kernel(const Kv4Cache c, const Kv4Rows r) {
  using R = Kv4Record<NG>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
  const int h = static_cast<int>(unit % c.N_kv);
  Piece piece;
  if (!find_piece(r, c.B, c.S_max, static_cast<int>(unit / c.N_kv), piece)) return;
  const int slot0 = piece.rec * kKv4Rows;
  auto meant = [&](int row) { return slot0 + row >= piece.lo && slot0 + row < piece.hi; };
  const uint16_t* src_k = static_cast<const uint16_t*>(r.k) + h * r.k_stride[1];
  const uint16_t* src_v = static_cast<const uint16_t*>(r.v) + h * r.v_stride[1];

  // all loads first: eight columns of rows g and 8 + g of K, four columns of rows 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t of V
  uint4 kx[2][NG];
  uint2 vx[4][NG];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half * 8 + g;
    const int64_t at = (static_cast<int64_t>(slot0) + row + piece.shift) * r.k_stride[0] + 8 * t;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      kx[half][grp] = make_uint4(0u, 0u, 0u, 0u);
      if (meant(row) && 32 * grp + 8 * t < c.D) kx[half][grp] = *reinterpret_cast<const uint4*>(src_k + at + 32 * grp);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (i >> 1) * 8 + 2 * t + (i & 1);
    const int64_t at = (static_cast<int64_t>(slot0) + row + piece.shift) * r.v_stride[0] + 4 * g;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      vx[i][grp] = make_uint2(0u, 0u);
      if (meant(row) && 32 * grp + 4 * g < c.D) vx[i][grp] = *reinterpret_cast<const uint2*>(src_v + at + 32 * grp);
    }
  }
  uint8_t* rec = kv4_record(c, piece.b, h, piece.rec, R::kBytes);
  constexpr uint32_t kNothing = BF16 ? 0xff807f80u : 0xfc007c00u;      // minimum +inf, maximum -inf: columns past head_dim

#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half * 8 + g;
    uint32_t words[NG];
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const uint32_t x[4] = {kx[half][grp].x, kx[half][grp].y, kx[half][grp].z, kx[half][grp].w};
      uint32_t mm = fold<BF16>(min2<BF16>(min2<BF16>(x[0], x[1]), min2<BF16>(x[2], x[3])), max2<BF16>(max2<BF16>(x[0], x[1]), max2<BF16>(x[2], x[3])));
      if (32 * grp + 8 * t >= c.D) mm = kNothing;
      mm = fold_lanes<BF16>(fold_lanes<BF16>(mm, 1), 2);
      const Group q = make_group<BF16>(mm);
      uint32_t w = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w |= code_of(to_float<BF16>(static_cast<uint16_t>(x[e >> 1] >> (16 * (e & 1)))), q) << (4 * e);
      words[grp] = w;
      if (meant(row) && t == grp) {
        *reinterpret_cast<uint16_t*>(rec + R::k_step(row, grp)) = q.step;
        *reinterpret_cast<uint16_t*>(rec + R::k_min(row, grp)) = q.low;
      }
    }
    if (meant(row)) store_words<NG>(rec, half * NG, lane, words);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = p * 8 + 2 * t;             // and row + 1
    const bool m0 = meant(row), m1 = meant(row + 1);
    uint32_t words[NG];
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      Group q[2];
      uint32_t w = 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 x = vx[2 * p + i][grp];
        uint32_t mm = fold<BF16>(min2<BF16>(x.x, x.y), max2<BF16>(x.x, x.y));
        if (32 * grp + 4 * g >= c.D) mm = kNothing;
        mm = fold_lanes<BF16>(fold_lanes<BF16>(fold_lanes<BF16>(mm, 4), 8), 16);
        q[i] = make_group<BF16>(mm);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w |= code_of(to_float<BF16>(static_cast<uint16_t>((e < 2 ? x.x : x.y) >> (16 * (e & 1)))), q[i]) << (16 * i + 4 * e);
      }
      words[grp] = w;
      if (g == grp) {
        if (m0 && m1) {
          *reinterpret_cast<uint2*>(rec + R::v_step(row, grp)) =
              make_uint2(q[0].step | (static_cast<uint32_t>(q[1].step) << 16), q[0].low | (static_cast<uint32_t>(q[1].low) << 16));
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i == 0 ? m0 : m1) {
              *reinterpret_cast<uint16_t*>(rec + R::v_step(row + i, grp)) = q[i].step;
              *reinterpret_cast<uint16_t*>(rec + R::v_min(row + i, grp)) = q[i].low;
            }
        }
      }
    }
    const int place = R::v_place(g, t);
    if (m0 && m1) {
      store_words<NG>(rec + R::kV, p * NG, place, words);
    } else if (m0 || m1) {                     // the other half of each word is another row's
#pragma unroll
      for (int grp = 0; grp < NG; ++grp)
        *reinterpret_cast<uint16_t*>(rec + R::kV + R::word(p * NG + grp, place) + (m0 ? 0 : 2)) = static_cast<uint16_t>(m0 ? words[grp] : words[grp] >> 16);
    }
  }
}

// What code `c` (a few bits of a word) stands for, in 16 bits: one rounding.
template <bool BF16>
__device__ __forceinline__ uint32_t value_of(uint32_t code, float step, float low) {
  const float c = __uint_as_float(code | 0x4b000000u) - 8388608.0f;
  const float v = fmaf(c, step, low);
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_read_kernel(const Kv4Cache c, const Kv4Rows r) {
  using R = Kv4Record<NG>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
  const int h = static_cast<int>(unit % c.N_kv);
  Piece piece;
  if (!find_piece(r, c.B, c.S_max, static_cast<int>(unit / c.N_kv), piece)) return;
  const int slot0 = piece.rec * kKv4Rows;
  auto meant = [&](int row) { return slot0 + row >= piece.lo && slot0 + row < piece.hi; };
  uint16_t* dst_k = static_cast<uint16_t*>(r.k) + h * r.k_stride[1];
  uint16_t* dst_v = static_cast<uint16_t*>(r.v) + h * r.v_stride[1];
  const uint8_t* rec = kv4_record(c, piece.b, h, piece.rec, R::kBytes);

  uint32_t kw[2][NG], vw[2][NG], ks[2][NG], km[2][NG];
  uint2 vsm[2][NG];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half * 8 + g;
    load_words<NG>(rec, half * NG, lane, kw[half]);
    load_words<NG>(rec + R::kV, half * NG, R::v_place(g, t), vw[half]);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      ks[half][grp] = *reinterpret_cast<const uint16_t*>(rec + R::k_step(row, grp));
      km[half][grp] = *reinterpret_cast<const uint16_t*>(rec + R::k_min(row, grp));
      vsm[half][grp] = *reinterpret_cast<const uint2*>(rec + R::v_step(half * 8 + 2 * t, grp));
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half * 8 + g;
    if (!meant(row)) continue;
    uint16_t* at = dst_k + (static_cast<int64_t>(slot0) + row + piece.shift) * r.k_stride[0] + 8 * t;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      if (32 * grp + 8 * t >= c.D) continue;
      const float s = to_float<BF16>(static_cast<uint16_t>(ks[half][grp])), m = to_float<BF16>(static_cast<uint16_t>(km[half][grp]));
      uint32_t x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = value_of<BF16>((kw[half][grp] >> (8 * e)) & 15u, s, m) | (value_of<BF16>((kw[half][grp] >> (8 * e + 4)) & 15u, s, m) << 16);
      *reinterpret_cast<uint4*>(at + 32 * grp) = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = p * 8 + 2 * t + i;
      if (!meant(row)) continue;
      uint16_t* at = dst_v + (static_cast<int64_t>(slot0) + row + piece.shift) * r.v_stride[0] + 4 * g;
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        if (32 * grp + 4 * g >= c.D) continue;
        const float s = to_float<BF16>(static_cast<uint16_t>(vsm[p][grp].x >> (16 * i))), m = to_float<BF16>(static_cast<uint16_t>(vsm[p][grp].y >> (16 * i)));
        const uint32_t w = vw[p][grp] >> (16 * i);
        *reinterpret_cast<uint2*>(at + 32 * grp) =
            make_uint2(value_of<BF16>(w & 15u, s, m) | (value_of<BF16>((w >> 4) & 15u, s, m) << 16),
                       value_of<BF16>((w >> 8) & 15u, s, m) | (value_of<BF16>((w >> 12) & 15u, s, m) << 16));
      }
    }
}

// Records that T rows of B sequences can touch: n rows lie in at most (n + 30) / 16.
unsigned int row_blocks(const Kv4Cache& c, const Kv4Rows& r) {
  const int64_t items = r.cu == nullptr ? c.B : (static_cast<int64_t>(r.T) + 30ll * c.B) / kKv4Rows;
  return static_cast<unsigned int>((items * c.N_kv + kRowsWarps - 1) / kRowsWarps);
}

}  // namespace

#define KV4_ROWS_KERNEL(name)                                                                                                       \
  ((c.D + 31) / 32 == 1 ? (bf16 ? name<1, true> : name<1, false>) : (c.D + 31) / 32 == 2 ? (bf16 ? name<2, true> : name<2, false>) \
   : (c.D + 31) / 32 == 3 ? (bf16 ? name<3, true> : name<3, false>) : (bf16 ? name<4, true> : name<4, false>))

cudaError_t launch_kv4_append(const Kv4Cache& c, const Kv4Rows& r, bool bf16, cudaStream_t stream) {
  KV4_ROWS_KERNEL(kv4_append_kernel)<<<row_blocks(c, r), kRowsWarps * 32, 0, stream>>>(c, r);
  return cudaGetLastError();
}

cudaError_t launch_kv4_read(const Kv4Cache& c, const Kv4Rows& r, bool bf16, cudaStream_t stream) {
  KV4_ROWS_KERNEL(kv4_read_kernel)<<<row_blocks(c, r), kRowsWarps * 32, 0, stream>>>(c, r);
  return cudaGetLastError();
}
#undef KV4_ROWS_KERNEL

}  // namespace acct
