// Rows into the 4-bit cache, and back out of it (kv4_common.cuh has the layout).
//
// Both would be bound by memory: 16 bits in and 5 out a value, or the other way round.  A warp takes K or V of one record of one head, so
// that the minimum and maximum of a group are a few shuffles, every lane ends up with the very words that it writes, and
// enough warps are resident to keep loads in flight.  Where only some of a record's rows are meant (a single token, the ends of a
// prompt) it loads and stores those and leaves the others alone.
//
// 16 prompts of up to 4 096 tokens, 8 heads of 128, in and out again: 110 us for 497 MB in all, 76 at the rate of a copy.
// Reading issues in 55 % of the clocks; writing, with extremes, steps and rounding for each value, in 69 %: nothing is at its limit,
// the arithmetic is what comes closest.
// A single token per sequence is latency: 6.6 us on the device for one write and one read.
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
template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t x, float& a, float& b) {
  if constexpr (BF16) {
    a = __uint_as_float(x << 16);
    b = __uint_as_float(x & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    a = f.x;
    b = f.y;
  }
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

// Step and 1 / step of a group from its extremes.  The step is rounded down, so that no value of the group (15 steps above the
// minimum at most) can leave the 16-bit type.  A group with a value that is not finite gets a NaN for its step.
template <bool BF16>
__device__ __forceinline__ uint32_t make_step(uint32_t mm, float& inv) {
  const float low = to_float<BF16>(static_cast<uint16_t>(mm)), high = to_float<BF16>(static_cast<uint16_t>(mm >> 16));
  const float range = __fsub_rn(high, low), want = __fdiv_rn(range, 15.0f);
  uint16_t step;
  if constexpr (BF16) step = __bfloat16_as_ushort(__float2bfloat16_rz(want));
  else step = __half_as_ushort(__float2half_rz(want));
  if (!(range < INFINITY)) step = 0x7fff;
  const float s = to_float<BF16>(step);
  inv = s > 0.f ? fminf(__frcp_rn(s), 3.4028235e38f) : 0.f;
  return step;
}
// Codes of four pairs (x[i], y[i]), each round((x - minimum) / step), half to even, at most 15: nibble i of the low half for x, of
// the high half for y.  Two-wide arithmetic; adding 1.5 * 2^23 rounds to an integer, and four codes of 4 bits are summed up
// exactly as floats.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], const float (&y)[4], float low_x, float low_y, float inv_x, float inv_y) {
  const uint64_t low = f2_pack(-low_x, -low_y), inv = f2_pack(inv_x, inv_y);
  const uint64_t magic = f2_pack(12582912.0f, 12582912.0f), minus = f2_pack(-12582912.0f, -12582912.0f);
  uint64_t sum = f2_pack(0.f, 0.f);
  constexpr float kWeight[4] = {1.f, 16.f, 256.f, 4096.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(f2_mul(f2_add(f2_pack(x[i], y[i]), low), inv), a, b);
    const uint64_t c = f2_add(f2_add(f2_pack(fminf(a, 15.f), fminf(b, 15.f)), magic), minus);
    sum = f2_fma(c, f2_pack(kWeight[i], kWeight[i]), sum);
  }
  float a, b;
  f2_unpack(f2_add(sum, f2_pack(8388608.f, 8388608.f)), a, b);      // the integer in the low bits
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
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

// Which piece of work this warp has: K or V (`value`) of head h of the piece.
struct RowsUnit {
  int h;
  bool value;
  Piece piece;
};
__device__ __forceinline__ bool find_unit(const Kv4Cache& c, const Kv4Rows& r, RowsUnit& out) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
  const int within = static_cast<int>(unit % (2 * c.N_kv));
  out.h = within >> 1;
  out.value = (within & 1) != 0;
  return find_piece(r, c.B, c.S_max, static_cast<int>(unit / (2 * c.N_kv)), out.piece);
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_append_kernel(const Kv4Cache c, const Kv4Rows r) {
  using R = Kv4Record<NG>;
  constexpr uint32_t kNothing = BF16 ? 0xff807f80u : 0xfc007c00u;      // minimum +inf, maximum -inf: columns past head_dim
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  RowsUnit unit;
  if (!find_unit(c, r, unit)) return;
  const Piece& piece = unit.piece;
  const int slot0 = piece.rec * kKv4Rows;
  auto meant = [&](int row) { return slot0 + row >= piece.lo && slot0 + row < piece.hi; };
  uint8_t* rec = kv4_record(c, piece.b, unit.h, piece.rec, R::kBytes);

  // Extremes of every group, in all lanes that have a part of it: the four of a row of K, the eight of a row of V.  Then each of
  // them forms the steps of a few groups only, a division and a reciprocal that cost more than all codes of a group.
  if (!unit.value) {
    // eight columns of rows g and 8 + g
    const uint16_t* src = static_cast<const uint16_t*>(r.k) + unit.h * r.k_stride[1];
    uint4 x[2][NG];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = half * 8 + g;
      const int64_t at = (static_cast<int64_t>(slot0) + row + piece.shift) * r.k_stride[0] + 8 * t;
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        x[half][grp] = make_uint4(0u, 0u, 0u, 0u);
        if (meant(row) && 32 * grp + 8 * t < c.D) x[half][grp] = *reinterpret_cast<const uint4*>(src + at + 32 * grp);
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = half * 8 + g;
      uint32_t mm[NG], mine = 0u;      // lane t has group t
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        const uint4 v = x[half][grp];
        mm[grp] = fold<BF16>(min2<BF16>(min2<BF16>(v.x, v.y), min2<BF16>(v.z, v.w)), max2<BF16>(max2<BF16>(v.x, v.y), max2<BF16>(v.z, v.w)));
        if (32 * grp + 8 * t >= c.D) mm[grp] = kNothing;
        mm[grp] = fold_lanes<BF16>(fold_lanes<BF16>(mm[grp], 1), 2);
        if (t == grp) mine = mm[grp];
      }
      float my_inv;
      const uint32_t my_step = make_step<BF16>(mine, my_inv);
      if (meant(row) && t < NG) {
        *reinterpret_cast<uint16_t*>(rec + R::k_step(row, 0) + 2 * t) = static_cast<uint16_t>(my_step);
        *reinterpret_cast<uint16_t*>(rec + R::k_min(row, 0) + 2 * t) = static_cast<uint16_t>(mine);
      }
      uint32_t words[NG];
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        const float inv = __shfl_sync(0xffffffffu, my_inv, (lane & ~3) | grp), low = to_float<BF16>(static_cast<uint16_t>(mm[grp]));
        float a[4], b[4];
        unpack2<BF16>(x[half][grp].x, a[0], a[1]);
        unpack2<BF16>(x[half][grp].y, a[2], a[3]);
        unpack2<BF16>(x[half][grp].z, b[0], b[1]);
        unpack2<BF16>(x[half][grp].w, b[2], b[3]);
        words[grp] = codes_of(a, b, low, low, inv, inv);
      }
      if (meant(row)) kv4_store_words<NG>(rec, half * NG, lane, words);
    }
    return;
  }
  // four columns of rows 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t
  const uint16_t* src = static_cast<const uint16_t*>(r.v) + unit.h * r.v_stride[1];
  uint2 x[4][NG];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (i >> 1) * 8 + 2 * t + (i & 1);
    const int64_t at = (static_cast<int64_t>(slot0) + row + piece.shift) * r.v_stride[0] + 4 * g;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      x[i][grp] = make_uint2(0u, 0u);
      if (meant(row) && 32 * grp + 4 * g < c.D) x[i][grp] = *reinterpret_cast<const uint2*>(src + at + 32 * grp);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = p * 8 + 2 * t;             // and row + 1
    const bool m0 = meant(row), m1 = meant(row + 1);
    uint32_t mm[2][NG], mine = 0u;             // lane g has row g & 1, group g >> 1
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        const uint2 v = x[2 * p + i][grp];
        mm[i][grp] = fold<BF16>(min2<BF16>(v.x, v.y), max2<BF16>(v.x, v.y));
        if (32 * grp + 4 * g >= c.D) mm[i][grp] = kNothing;
        mm[i][grp] = fold_lanes<BF16>(fold_lanes<BF16>(fold_lanes<BF16>(mm[i][grp], 4), 8), 16);
        if (g == 2 * grp + i) mine = mm[i][grp];
      }
    float my_inv;
    const uint32_t my_step = make_step<BF16>(mine, my_inv);
    if (meant(row + (g & 1)) && g < 2 * NG) {
      *reinterpret_cast<uint16_t*>(rec + R::v_step(row, 0) + (g >> 1) * 8 + (g & 1) * 2) = static_cast<uint16_t>(my_step);
      *reinterpret_cast<uint16_t*>(rec + R::v_min(row, 0) + (g >> 1) * 8 + (g & 1) * 2) = static_cast<uint16_t>(mine);
    }
    uint32_t words[NG];
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const float inv0 = __shfl_sync(0xffffffffu, my_inv, (2 * grp) * 4 + t), inv1 = __shfl_sync(0xffffffffu, my_inv, (2 * grp + 1) * 4 + t);
      float a[4], b[4];
      unpack2<BF16>(x[2 * p][grp].x, a[0], a[1]);
      unpack2<BF16>(x[2 * p][grp].y, a[2], a[3]);
      unpack2<BF16>(x[2 * p + 1][grp].x, b[0], b[1]);
      unpack2<BF16>(x[2 * p + 1][grp].y, b[2], b[3]);
      words[grp] = codes_of(a, b, to_float<BF16>(static_cast<uint16_t>(mm[0][grp])), to_float<BF16>(static_cast<uint16_t>(mm[1][grp])), inv0, inv1);
    }
    const int place = R::v_place(g, t);
    if (m0 && m1) {
      kv4_store_words<NG>(rec + R::kV, p * NG, place, words);
    } else if (m0 || m1) {                     // the other half of each word is another row's
#pragma unroll
      for (int grp = 0; grp < NG; ++grp)
        *reinterpret_cast<uint16_t*>(rec + R::kV + R::word(p * NG + grp, place) + (m0 ? 0 : 2)) = static_cast<uint16_t>(m0 ? words[grp] : words[grp] >> 16);
    }
  }
}

// Values two at a time, code * step + minimum rounded once to 16 bits; then neighbours of a row side by side.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_read_kernel(const Kv4Cache c, const Kv4Rows r) {
  using R = Kv4Record<NG>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  RowsUnit unit;
  if (!find_unit(c, r, unit)) return;
  const Piece& piece = unit.piece;
  const int slot0 = piece.rec * kKv4Rows;
  auto meant = [&](int row) { return slot0 + row >= piece.lo && slot0 + row < piece.hi; };
  const uint8_t* rec = kv4_record(c, piece.b, unit.h, piece.rec, R::kBytes);
  uint32_t w[2][NG];
  if (!unit.value) {
    uint16_t* dst = static_cast<uint16_t*>(r.k) + unit.h * r.k_stride[1];
    uint32_t step[2][NG], low[2][NG];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      kv4_load_words<NG>(rec, half * NG, lane, w[half]);
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        step[half][grp] = *reinterpret_cast<const uint16_t*>(rec + R::k_step(half * 8 + g, grp));
        low[half][grp] = *reinterpret_cast<const uint16_t*>(rec + R::k_min(half * 8 + g, grp));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = half * 8 + g;
      uint16_t* at = dst + (static_cast<int64_t>(slot0) + row + piece.shift) * r.k_stride[0] + 8 * t;
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        uint32_t x[4];
        kv4_value_pairs<BF16>(w[half][grp], __byte_perm(step[half][grp], 0u, 0x1010), __byte_perm(low[half][grp], 0u, 0x1010), x);
        if (meant(row) && 32 * grp + 8 * t < c.D)
          *reinterpret_cast<uint4*>(at + 32 * grp) = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                                                                __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
      }
    }
    return;
  }
  uint16_t* dst = static_cast<uint16_t*>(r.v) + unit.h * r.v_stride[1];
  uint2 both[2][NG];      // steps and minima of rows 2 t, 2 t + 1 of the half
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    kv4_load_words<NG>(rec + R::kV, p * NG, R::v_place(g, t), w[p]);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) both[p][grp] = *reinterpret_cast<const uint2*>(rec + R::v_step(p * 8 + 2 * t, grp));
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = p * 8 + 2 * t;
    uint16_t* at = dst + (static_cast<int64_t>(slot0) + row + piece.shift) * r.v_stride[0] + 4 * g;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      uint32_t x[4];
      kv4_value_pairs<BF16>(w[p][grp], both[p][grp].x, both[p][grp].y, x);
      if (32 * grp + 4 * g < c.D) {
        if (meant(row)) *reinterpret_cast<uint2*>(at + 32 * grp) = make_uint2(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410));
        if (meant(row + 1))
          *reinterpret_cast<uint2*>(at + r.v_stride[0] + 32 * grp) = make_uint2(__byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
      }
    }
  }
}

// Records that T rows of B sequences can touch: n rows lie in at most (n + 30) / 16.
unsigned int row_blocks(const Kv4Cache& c, const Kv4Rows& r) {
  const int64_t items = r.cu == nullptr ? c.B : (static_cast<int64_t>(r.T) + 30ll * c.B) / kKv4Rows;
  return static_cast<unsigned int>((items * 2 * c.N_kv + kRowsWarps - 1) / kRowsWarps);
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
