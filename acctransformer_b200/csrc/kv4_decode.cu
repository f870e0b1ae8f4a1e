// Decode over the 4-bit cache: one query token per sequence, 1..16 query heads per cache head.
//
// The step is bound by reading the cache once (160 bytes per key and head at head_dim 128), but at 5 bits a value there is little
// time per value: an SM gets 23 bytes per clock, a 16-row record in 110, in which its four schedulers issue 440 instructions
// for 4 096 codes.  So a code takes no arithmetic of its own that can be avoided:
//   S = Q K^T    k = s c + m splits into s (Q c) + m (sum of Q): the codes go to mma.m16n8k16 as they are, one group of 32 columns
//                at a time, and s and m meet 16 x 16 sums instead of 16 x 128 values.  In fp16 a code in the low bits of a half is
//                the subnormal number c * 2^-24, exact to multiply (and c * 2^-20 four bits up: those columns of Q are divided by
//                16), so a mask is all it takes; in bf16 it goes into the low bits of 128 and 128 is subtracted.  m times the sum
//                of Q is one more product, whose operand holds the sums in three parts so that nothing of them is lost.
//   O += P V     here the steps belong to the contraction: v = s c + m is formed in 16 bits (one rounding, as if the cache were
//                in 16 bits), two rows of a column at a time, with the code subtracted out of 1024 + c, 64 + c or 128 + c.
// Records come in by one bulk copy each through a ring per warp; nothing is shared between the warps of a block before the end.
//
// The parts of a slice leave (acc[D], max, sum) per query head; kv4_finish_kernel joins them and, where the probabilities are
// wanted, takes the scores that were left in scratch (4 bytes per key and query head) to exp2(x - max) / sum, added up over the
// group.  Where few slices leave room on the GPU, the parts of one are a cluster and join without a second kernel.
#include "fa_common.cuh"
#include "fa_kernels.cuh"
#include "kv4_common.cuh"
#include "ptx.cuh"

namespace acct {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kSlots = 4;             // records in a warp's ring

// D (16x8, fp32) += A (16x16, row) * B (16x8, col); 16-bit operands
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// The four pairs of codes of a word (nibble j of either half), for Q K^T: what they multiply to is the code times
// 2^-24, 2^-20, 2^-24, 2^-20 in fp16, the code itself in bf16.
constexpr float kCodeScaleF16 = 16777216.0f;
template <bool BF16>
__device__ __forceinline__ void key_codes(uint32_t w, uint32_t (&x)[4]) {
  if constexpr (BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = sub2<true>(((w >> (4 * j)) & 0x000f000fu) | 0x43004300u, 0x43004300u);
  } else {
    const uint32_t u = w >> 8;
    x[0] = w & 0x000f000fu; x[1] = w & 0x00f000f0u; x[2] = u & 0x000f000fu; x[3] = u & 0x00f000f0u;
  }
}
// The same for P V: the values, code * step + minimum, of two rows.
template <bool BF16>
__device__ __forceinline__ void value_pairs(uint32_t w, uint32_t step, uint32_t low, uint32_t (&x)[4]) {
  if constexpr (BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = sub2<true>(((w >> (4 * j)) & 0x000f000fu) | 0x43004300u, 0x43004300u);
  } else {
    const uint32_t u = w >> 8;
    x[0] = sub2<false>((w & 0x000f000fu) | 0x64006400u, 0x64006400u);      // 1024 + c
    x[1] = sub2<false>((w & 0x00f000f0u) | 0x54005400u, 0x54005400u);      // 64 + c
    x[2] = sub2<false>((u & 0x000f000fu) | 0x64006400u, 0x64006400u);
    x[3] = sub2<false>((u & 0x00f000f0u) | 0x54005400u, 0x54005400u);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = fma2<BF16>(x[j], step, low);
}

template <int N>
__device__ __forceinline__ void shared_words(uint32_t addr, uint32_t* x) {      // N words, in as few loads as their alignment allows
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]) : "r"(addr + 4 * i));
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[i]), "=r"(x[i + 1]) : "r"(addr + 4 * i));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[i]) : "r"(addr + 4 * i));
  }
}
// the words of a lane's place: units of kUnit words, 32 units apart
template <int NG>
__device__ __forceinline__ void lane_words(uint32_t base, int place, uint32_t (&x)[2 * NG]) {
  using R = Kv4Record<NG>;
#pragma unroll
  for (int u = 0; u < R::kWords; u += R::kUnit) shared_words<R::kUnit>(base + R::word(u, place), x + u);
}

// UPPER: the group has more than 8 query heads, i.e. rows 8..15 of the MMAs carry heads too.
template <int NG, bool BF16, bool UPPER>
__global__ void __launch_bounds__(kThreads) kv4_decode_kernel(const Kv4DecodeParams p) {
  using R = Kv4Record<NG>;
  constexpr int kHi = UPPER ? 2 : 1;
  constexpr int DPAD = 32 * NG;

  extern __shared__ __align__(128) uint8_t ksm[];
  __shared__ uint64_t full[kWarps][kSlots];
  __shared__ volatile uint32_t abort_flag;

  const int G = p.kv_group;
  const int split = blockIdx.x, unit_kv = blockIdx.y;
  const int b = unit_kv / p.cache.N_kv, h_kv = unit_kv % p.cache.N_kv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kSlots; ++i) mbar_init(&full[0][0] + i, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();

  int len = p.cache.S_max;
  if (p.seq_lens != nullptr) len = min(len, max(0, p.seq_lens[b]));
  const int n_rec = (len + kKv4Rows - 1) / kKv4Rows;
  const int per = ((n_rec + p.splits - 1) / p.splits + kWarps - 1) / kWarps * kWarps;
  const int r0 = split * per, r1 = min(n_rec, r0 + per);
  const int mine = r1 - r0 > warp ? (r1 - r0 - warp + kWarps - 1) / kWarps : 0;      // records r0 + warp, r0 + warp + 4, ..

  uint8_t* ring = ksm + warp * (kSlots * R::kBytes);
  const bool paged = p.cache.table != nullptr;
  int pages = 0;                       // lane i: the page of this warp's record (i of the last 32 asked for)
  auto issue = [&](int i) {            // the i-th record of this warp into ring slot i % kSlots; the whole warp calls it
    const int rec = r0 + warp + i * kWarps;
    const uint8_t* src;
    if (paged) {
      if ((i & 31) == 0) {
        const int r = rec + lane * kWarps;
        pages = r < r1 ? p.cache.table[static_cast<int64_t>(b) * p.cache.max_pages + (r >> p.cache.page_shift)] : 0;
        pages = min(max(pages, 0), p.cache.num_pages - 1);
      }
      const int64_t page = __shfl_sync(0xffffffffu, pages, i & 31);
      src = p.cache.records + (((page * p.cache.N_kv + h_kv) << p.cache.page_shift) + (rec & ((1 << p.cache.page_shift) - 1))) * R::kBytes;
    } else {
      src = p.cache.records + ((static_cast<int64_t>(b) * p.cache.N_kv + h_kv) * p.cache.recs + rec) * R::kBytes;
    }
    if (elect_one()) {
      uint64_t* bar = &full[warp][i % kSlots];
      mbar_expect_tx(bar, R::kBytes);
      bulk_load(ring + (i % kSlots) * R::kBytes, src, R::kBytes, bar);
    }
  };
#pragma unroll
  for (int i = 0; i < kSlots - 1; ++i)
    if (i < mine) issue(i);

  // ---- the query heads as A fragments, columns in the order of the codes: of a thread's eight columns 32 grp + 8 t + .. of a
  // group the pairs (0, 4), (1, 5), (2, 6), (3, 7); in fp16 the second and fourth pair divided by 16
  uint32_t qa[2 * NG][2 * kHi], qm[2 * kHi];
#pragma unroll
  for (int hi = 0; hi < kHi; ++hi) {
    const int head = g + 8 * hi;
    float mean_t = 0.f;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const int d = 32 * grp + 8 * t;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (head < G && d < p.D)
        u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(b) * p.N + h_kv * G + head) * p.D + d);
      const uint32_t pairs[4] = {__byte_perm(u.x, u.z, 0x5410), __byte_perm(u.x, u.z, 0x7632), __byte_perm(u.y, u.w, 0x5410), __byte_perm(u.y, u.w, 0x7632)};
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<BF16>(pairs[j]);
        sum += f.x + f.y;
        uint32_t w = pairs[j];
        if (!BF16 && (j & 1) != 0) w = pack2<BF16>(f.x * 0.0625f, f.y * 0.0625f);
        qa[2 * grp + (j >> 1)][(j & 1) * kHi + hi] = w;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == grp) mean_t = sum * 0.03125f;          // of the group's 32 columns: in the range of Q whatever that is
    }
    // the mean as a sum of three 16-bit numbers
    uint32_t w0 = pack2<BF16>(mean_t, 0.f);
    const float rest1 = mean_t - unpack2<BF16>(w0).x;
    const uint32_t w1 = pack2<BF16>(rest1, 0.f);
    const float rest2 = rest1 - unpack2<BF16>(w1).x;
    qm[hi] = (w0 & 0xffffu) | (w1 << 16);
    qm[kHi + hi] = pack2<BF16>(rest2, 0.f);
  }

  float o[4 * NG][2 * kHi];
#pragma unroll
  for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
    for (int e = 0; e < 2 * kHi; ++e) o[i][e] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};      // rows g and g + 8; l is this thread's share
  const float f_code = BF16 ? p.scale_log2 : p.scale_log2 * kCodeScaleF16, f_mean = p.scale_log2 * 32.0f;

  for (int it = 0; it < mine; ++it) {
    if (it + kSlots - 1 < mine) issue(it + kSlots - 1);
    mbar_wait(&full[warp][it % kSlots], (it / kSlots) & 1, &abort_flag, p.status, DEV_TIMEOUT_TMA);
    const uint32_t rec = smem_u32(ring + (it % kSlots) * R::kBytes);
    const int row0 = (r0 + warp + it * kWarps) * kKv4Rows;
    const bool partial = row0 + kKv4Rows > len;

    // ---- S = Q K^T, in log2 units: x[half][row half of the MMA][column]
    float x[2][kHi][2];
    {
      uint32_t kw[2 * NG];
      lane_words<NG>(rec, lane, kw);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t low = 0u, steps[NG];
        if (t < NG) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(low) : "r"(rec + R::kKm + ((half * 8 + g) * NG + t) * 2));
        low = __byte_perm(low, 0u, 0x1010);
        shared_words<NG>(rec + R::kKs + (half * 4 + t) * NG * 4, steps);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816<BF16>(c, qm[0], UPPER ? qm[kHi - 1] : 0u, qm[kHi], UPPER ? qm[2 * kHi - 1] : 0u, low, low);
#pragma unroll
        for (int hi = 0; hi < kHi; ++hi) x[half][hi][0] = x[half][hi][1] = 0.f;
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          uint32_t kb[4];
          key_codes<BF16>(kw[half * NG + grp], kb);
          float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t(&q)[2 * kHi] = qa[2 * grp + j];
            mma16816<BF16>(a, q[0], UPPER ? q[kHi - 1] : 0u, q[kHi], UPPER ? q[2 * kHi - 1] : 0u, kb[2 * j], kb[2 * j + 1]);
          }
          const float2 s = unpack2<BF16>(steps[grp]);
#pragma unroll
          for (int hi = 0; hi < kHi; ++hi) {
            x[half][hi][0] = fmaf(a[2 * hi], s.x, x[half][hi][0]);
            x[half][hi][1] = fmaf(a[2 * hi + 1], s.y, x[half][hi][1]);
          }
        }
#pragma unroll
        for (int hi = 0; hi < kHi; ++hi)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[half][hi][e] = fmaf(x[half][hi][e], f_code, c[2 * hi + e] * f_mean);
      }
    }
    if (partial) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int hi = 0; hi < kHi; ++hi)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (row0 + half * 8 + 2 * t + e >= len) x[half][hi][e] = -INFINITY;
    }
    if (p.scores != nullptr) {
#pragma unroll
      for (int hi = 0; hi < kHi; ++hi)
        if (g + 8 * hi < G) {
          float* at = p.scores + (static_cast<int64_t>(b) * p.N + h_kv * G + g + 8 * hi) * p.S_pad + row0 + 2 * t;
          *reinterpret_cast<float2*>(at) = make_float2(x[0][hi][0], x[0][hi][1]);
          *reinterpret_cast<float2*>(at + 8) = make_float2(x[1][hi][0], x[1][hi][1]);
        }
    }
    // ---- online softmax; this thread holds, per row, keys 2t, 2t+1 of each half
    uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int hi = 0; hi < kHi; ++hi) {
      float mx = fmaxf(fmaxf(x[0][hi][0], x[0][hi][1]), fmaxf(x[1][hi][0], x[1][hi][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_run[hi], mx);           // row0 < len, so the record's first key exists
      const float alpha = ex2(m_run[hi] - m_new);         // 0 on the first record (m_run = -inf)
      const float p0 = ex2(x[0][hi][0] - m_new), p1 = ex2(x[0][hi][1] - m_new), p2 = ex2(x[1][hi][0] - m_new), p3 = ex2(x[1][hi][1] - m_new);
      l_run[hi] = fmaf(l_run[hi], alpha, (p0 + p1) + (p2 + p3));
      m_run[hi] = m_new;
      pa[hi] = pack2<BF16>(p0, p1);                       // P in 16 bits is the operand of P V; the sum is of what it was before
      pa[2 + hi] = pack2<BF16>(p2, p3);
      if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
          o[i][2 * hi] *= alpha;
          o[i][2 * hi + 1] *= alpha;
        }
      }
    }
    // ---- O += P V
    {
      uint32_t vw[2 * NG], vsm[2][2 * NG];
      lane_words<NG>(rec + R::kV, R::v_place(g, t), vw);
      shared_words<2 * NG>(rec + R::kVsm + t * NG * 8, vsm[0]);
      shared_words<2 * NG>(rec + R::kVsm + (4 + t) * NG * 8, vsm[1]);
      if (partial) {      // rows that do not exist: whatever their steps and minima are, 0 times them has to be 0
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int row = row0 + q * 8 + 2 * t;
          const uint32_t there = (row < len ? 0xffffu : 0u) | (row + 1 < len ? 0xffff0000u : 0u);
#pragma unroll
          for (int i = 0; i < 2 * NG; ++i) vsm[q][i] &= there;
        }
      }
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        uint32_t v0[4], v1[4];
        value_pairs<BF16>(vw[grp], vsm[0][2 * grp], vsm[0][2 * grp + 1], v0);
        value_pairs<BF16>(vw[NG + grp], vsm[1][2 * grp], vsm[1][2 * grp + 1], v1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float(&acc)[2 * kHi] = o[4 * grp + j];
          float c[4] = {acc[0], acc[1], UPPER ? acc[2 * kHi - 2] : 0.f, UPPER ? acc[2 * kHi - 1] : 0.f};
          mma16816<BF16>(c, pa[0], pa[1], pa[2], pa[3], v0[j], v1[j]);
#pragma unroll
          for (int e = 0; e < 2 * kHi; ++e) acc[e] = c[e];
        }
      }
    }
    __syncwarp();      // every lane has read this slot before a later copy may land in it
  }

  // ---- merge the four warps per query head, then write the part's result (the rings are dead by now: their memory holds the
  // warps' accumulators)
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    l_run[hi] += __shfl_xor_sync(0xffffffffu, l_run[hi], 1);
    l_run[hi] += __shfl_xor_sync(0xffffffffu, l_run[hi], 2);
  }
  linger_after_abort(&abort_flag);
  __syncthreads();
  constexpr int kHeads = 8 * kHi;
  float* s_acc = reinterpret_cast<float*>(ksm);                       // [warp][kHeads][DPAD]
  float* s_m = s_acc + kWarps * kHeads * DPAD;                        // [warp][kHeads]
  float* s_l = s_m + kWarps * kHeads;
#pragma unroll
  for (int hi = 0; hi < kHi; ++hi) {
    const int head = g + 8 * hi;
    if (t == 0) { s_m[warp * kHeads + head] = m_run[hi]; s_l[warp * kHeads + head] = l_run[hi]; }
#pragma unroll
    for (int grp = 0; grp < NG; ++grp)
#pragma unroll
      for (int e = 0; e < 2; ++e)      // columns 2t and 2t+1 of the MMA: 4 (2t) + j and 4 (2t+1) + j of the group
        *reinterpret_cast<float4*>(s_acc + (warp * kHeads + head) * DPAD + 32 * grp + 8 * t + 4 * e) =
            make_float4(o[4 * grp][2 * hi + e], o[4 * grp + 1][2 * hi + e], o[4 * grp + 2][2 * hi + e], o[4 * grp + 3][2 * hi + e]);
  }
  __syncthreads();
  for (int head = 0; head < G; ++head) {
    const int64_t slot = (static_cast<int64_t>(b) * p.N + h_kv * G + head) * p.splits + split;
    float big = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) big = fmaxf(big, s_m[w * kHeads + head]);
    float weight[kWarps], lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = s_m[w * kHeads + head];
      weight[w] = mw == -INFINITY ? 0.f : ex2(mw - big);
      lsum = fmaf(s_l[w * kHeads + head], weight[w], lsum);
    }
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) a = fmaf(s_acc[(w * kHeads + head) * DPAD + d], weight[w], a);
      p.part_acc[slot * p.D + d] = a;
    }
    if (threadIdx.x == 0) {
      p.part_ml[slot * 2] = big;
      p.part_ml[slot * 2 + 1] = lsum;
    }
  }
}

// Joins the parts: block (x, unit) has head x of the group for the output, and keys from x * kFinishKeys on for the weights.
constexpr int kFinishThreads = 128, kFinishKeys = 1024;
template <bool BF16>
__global__ void __launch_bounds__(kFinishThreads) kv4_finish_kernel(const Kv4DecodeParams p) {
  __shared__ float s_m[16], s_inv[16];
  const int unit_kv = blockIdx.y, b = unit_kv / p.cache.N_kv, h_kv = unit_kv % p.cache.N_kv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.kv_group, n = p.splits;
  const int64_t unit0 = static_cast<int64_t>(b) * p.N + h_kv * G;      // the group's first query head
  auto of_part = [&](int head, int s) {
    const float2 none = make_float2(-INFINITY, 0.f);
    return s < n ? reinterpret_cast<const float2*>(p.part_ml)[(unit0 + head) * n + s] : none;
  };
  for (int head = warp; head < G; head += kFinishThreads / 32) {
    const float2 e0 = of_part(head, lane), e1 = of_part(head, 32 + lane);
    float big = fmaxf(e0.x, e1.x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
    float l = (e0.x == -INFINITY ? 0.f : e0.y * ex2(e0.x - big)) + (e1.x == -INFINITY ? 0.f : e1.y * ex2(e1.x - big));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (lane == 0) {
      s_m[head] = big;
      s_inv[head] = l != 0.f ? 1.0f / l : 0.f;
    }
  }
  __syncthreads();
  if (blockIdx.x < G) {
    const int head = blockIdx.x;
    for (int d = threadIdx.x; d < p.D; d += kFinishThreads) {
      const float* part = p.part_acc + (unit0 + head) * n * p.D + d;
      float a = 0.f;
#pragma unroll 8
      for (int s = 0; s < n; ++s) {
        const float ms = reinterpret_cast<const float2*>(p.part_ml)[(unit0 + head) * n + s].x;
        a = fmaf(part[static_cast<int64_t>(s) * p.D], ms == -INFINITY ? 0.f : ex2(ms - s_m[head]), a);
      }
      a *= s_inv[head];
      const int64_t at = (unit0 + head) * p.D + d;
      if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16(a);
      else reinterpret_cast<__half*>(p.y)[at] = __float2half(a);
    }
  }
  if (p.weights == nullptr) return;
  int len = p.cache.S_max;
  if (p.seq_lens != nullptr) len = min(len, max(0, p.seq_lens[b]));
  const int end = min(len, (static_cast<int>(blockIdx.x) + 1) * kFinishKeys);
  for (int key = blockIdx.x * kFinishKeys + threadIdx.x; key < end; key += kFinishThreads) {
    float w = 0.f;
    for (int head = 0; head < G; ++head) w = fmaf(ex2(p.scores[(unit0 + head) * p.S_pad + key] - s_m[head]), s_inv[head], w);
    p.weights[static_cast<int64_t>(unit_kv) * p.cache.S_max + key] += w;
  }
}

template <int NG>
cudaError_t launch_ng(const Kv4DecodeParams& p, bool bf16, cudaStream_t stream) {
  const bool upper = p.kv_group > 8;
  const size_t ring = static_cast<size_t>(kWarps) * kSlots * Kv4Record<NG>::kBytes;
  const size_t merge = static_cast<size_t>(kWarps) * (upper ? 16 : 8) * (32 * NG + 2) * sizeof(float);
  const size_t smem = ring > merge ? ring : merge;
  void (*kern)(const Kv4DecodeParams) = bf16 ? (upper ? kv4_decode_kernel<NG, true, true> : kv4_decode_kernel<NG, true, false>)
                                             : (upper ? kv4_decode_kernel<NG, false, true> : kv4_decode_kernel<NG, false, false>);
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  kern<<<dim3(p.splits, p.B * p.cache.N_kv), kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, bool bf16, cudaStream_t stream, int*) {
  const int groups = (p.D + 31) / 32;
  cudaError_t e = groups == 1 ? launch_ng<1>(p, bf16, stream) : groups == 2 ? launch_ng<2>(p, bf16, stream)
                  : groups == 3 ? launch_ng<3>(p, bf16, stream) : launch_ng<4>(p, bf16, stream);
  if (e != cudaSuccess) return e;
  const int chunks = p.weights != nullptr ? (p.cache.S_max + kFinishKeys - 1) / kFinishKeys : 1;
  const dim3 grid(chunks > p.kv_group ? chunks : p.kv_group, p.B * p.cache.N_kv);
  if (bf16) kv4_finish_kernel<true><<<grid, kFinishThreads, 0, stream>>>(p);
  else kv4_finish_kernel<false><<<grid, kFinishThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace acct
