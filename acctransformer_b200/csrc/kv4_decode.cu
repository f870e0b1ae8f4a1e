// Decode over the 4-bit cache: one query token per sequence, 1..16 query heads per cache head.
//
// The step is bound by reading the cache once (160 bytes per key and head at head_dim 128), but at 5 bits a value there is little
// time per value: an SM gets 23 bytes per clock, a 16-row record in 110, in which its four schedulers issue 440 instructions
// for 4 096 codes.  So rows and columns of the cache are the 16-row operand of mma.m16n8k16 and the query heads the 8 columns of
// the other (17 products a record for up to 4 heads), and a code takes no arithmetic of its own that can be avoided:
//   S^T = K Q^T   k = s c + m splits into s (c Q) + m (sum of Q): the codes go into the product as they are, one group of 32 columns
//                 at a time, and s and m meet 16 x 8 sums instead of 16 x 128 values.  In fp16 a code in the low bits of a half is
//                 the subnormal number c * 2^-24, exact to multiply (and c * 2^-20 four bits up: those columns of Q are divided by
//                 16), so a mask is all it takes; in bf16 it goes into the low bits of 128 and 128 is subtracted.  m times the sum
//                 of Q is one more product, whose operand holds the sums in three parts so that nothing of them is lost.  In fp16
//                 a head of Q whose largest value is below 2^10 is multiplied by a power of two that brings it there, and its
//                 scores are divided by it: a sixteenth of Q, and the parts of its sums, then lose 2^-34 of that value at most.
//   O^T += V^T P  here the steps belong to the contraction: v = s c + m is formed in 16 bits (one rounding, as if the cache were
//                 in 16 bits), two rows of a column at a time, with the code subtracted out of 1024 + c, 64 + c or 128 + c.
//                 P is rounded to 16 bits too, which would cost as much again (in fp16, over 2 048 keys, 3.4e-4 of the result from
//                 the exact one; its own last rounding makes 2.1e-4).  What the rounding leaves is an operand as well: with up to 4
//                 heads in the 4 columns that they leave free, where it costs 12 instructions a record (32 x 8 slices of up to
//                 16 384 keys, fp16: 97 -> 101 us, 115 -> 119 with probabilities), up to 8 in products of its own (102 -> 111,
//                 134 -> 143): 2.8e-4.  With more it is left out: 145 us would be 170, 220 be 242, and the 4 bits are coarser
//                 by two orders.
// The running maximum is only refreshed where a score exceeds it by more than 8 (in log2 units), so that most records need no
// exchange between lanes.  Records come in by one bulk copy each through a ring per warp; nothing is shared between the warps of
// a block before the end.
//
// The parts of a slice leave (acc[D], max, sum) per query head; kv4_finish_kernel joins them and, where the probabilities are
// wanted, takes the scores that were left in scratch (4 bytes per key and query head) to exp2(x - max) / sum, added up over the
// group.
#include <algorithm>

#include "fa_common.cuh"
#include "fa_kernels.cuh"
#include "kv4_common.cuh"
#include "ptx.cuh"

namespace acct {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kStepRecs = 2;          // records that a warp takes at a time: waits, addresses and softmax checks for both at once
constexpr int kSlots = 3;             // steps in a warp's ring

// D (16x8, fp32) += A (16x16, row) * B (16x8, col); 16-bit operands
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same with nothing to add to
template <bool BF16>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// A bulk copy whose lines are the first to leave L2: the cache is read once a step, what should stay are the scores.
__device__ __forceinline__ uint64_t read_once_policy() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
               : "memory");
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
    for (int j = 0; j < 4; ++j) x[j] = kv4_sub2<true>(kv4_mask_or(w >> (4 * j), 0x000f000fu, 0x43004300u), 0x43004300u);
  } else {
    const uint32_t u = w >> 8;
    x[0] = w & 0x000f000fu; x[1] = w & 0x00f000f0u; x[2] = u & 0x000f000fu; x[3] = u & 0x00f000f0u;
  }
}
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t* x) {      // N words, in as few loads as their alignment allows
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(at + 4 * i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(at + 4 * i);
      x[i] = v.x; x[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const uint32_t*>(at + 4 * i);
  }
}
// the words of a lane's place: units of kUnit words, 32 units apart
template <int NG>
__device__ __forceinline__ void lane_words(const uint8_t* base, int place, uint32_t (&x)[2 * NG]) {
  using R = Kv4Record<NG>;
#pragma unroll
  for (int u = 0; u < R::kWords; u += R::kUnit) load_words<R::kUnit>(base + R::word(u, place), x + u);
}
// NG 16-bit numbers of a row, as floats
template <int NG, bool BF16>
__device__ __forceinline__ void row_steps(const uint8_t* at, float (&s)[NG]) {
  if constexpr (NG % 2 == 0) {
    uint32_t w[NG / 2];
    load_words<NG / 2>(at, w);
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) {
      const float2 f = unpack2<BF16>(w[i]);
      s[2 * i] = f.x; s[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NG; ++i) s[i] = unpack2<BF16>(*reinterpret_cast<const uint16_t*>(at + 2 * i)).x;
  }
}
// the transpose of an 8 x 8 matrix of 16-bit numbers, lane (g, t) having row g, columns 2 t and 2 t + 1
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// How the batch is cut.  Every sequence into `splits` parts, where the caller says so.  Otherwise into parts of about equal length,
// `p.parts` for the heads of the batch together, so that thread blocks finish together whatever the lengths are: the length of
// a part follows from the sum of all lengths, which every block forms for itself (one load and a reduction, at the latency of
// the length that it needs anyway).  Never shorter than kMinSteps.
constexpr int kMinSteps = 16;
__device__ __forceinline__ int steps_of(const Kv4DecodeParams& p, int b) {
  int len = p.cache.S_max;
  if (p.seq_lens != nullptr) len = min(len, max(0, p.seq_lens[b]));
  return (len + kStepRecs * kKv4Rows - 1) / (kStepRecs * kKv4Rows);
}
// steps of a part, the same in all lanes
__device__ __forceinline__ int part_steps(const Kv4DecodeParams& p) {
  int total = 0;
  for (int b = threadIdx.x & 31; b < p.B; b += 32) total += steps_of(p, b);
  total = __reduce_add_sync(0xffffffffu, total);
  return max(kMinSteps, (total + p.parts - 1) / p.parts);
}
__device__ __forceinline__ int parts_of(const Kv4DecodeParams& p, int steps, int part) {
  return p.parts == 0 ? p.splits : min(p.splits, max(1, (steps + part - 1) / part));
}

constexpr float kRefresh = 8.0f;      // log2 units by which a score may exceed the running maximum
// The running maximum before there is one.  A finite number: a key that does not exist, or whose score is below fp32's range, then
// counts for exp2(-inf - kLowest) = 0 also where a warp has met no other key yet; and as the lowest of fp32 it is no higher than
// any score that is in range.
constexpr float kLowest = -3.402823466e38f;

// Resident thread blocks per SM, which the registers decide (152 to 168 and 228 to 234 a thread at head_dim 128).  With four, at 128
// registers, or five, at 96 and a record at a time, the step is no faster (32 x 8 slices of up to 16 384 keys 95 and 103 us against
// 90, all before what P's rounding leaves was multiplied).
constexpr int blocks_per_sm(int heads) { return heads <= 8 ? 3 : 2; }

// the float at `p` of this block's shared memory, in that of block `rank` of the cluster
__device__ __forceinline__ float cluster_read(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map(p, rank)) : "memory");
  return v;
}

constexpr int kMaxCluster = 8;

// HEADS: 4, 8 or 16, query heads per cache head at most.  CL: the parts of a slice are one cluster, and finish together.
template <int NG, bool BF16, int HEADS, bool CL>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(HEADS)) kv4_decode_kernel(const Kv4DecodeParams p) {
  using R = Kv4Record<NG>;
  constexpr int DPAD = 32 * NG, HI = HEADS > 8 ? 2 : 1, kHeads = 8 * HI;      // HI: times 8 columns
  constexpr bool kSpare = HEADS == 4;      // columns 4..7 are heads 0..3 once more, with what is left of P
  constexpr bool kRest = HEADS == 8;       // a product of its own for what is left

  extern __shared__ __align__(128) uint8_t ksm[];
  __shared__ uint64_t full[kWarps][kSlots];
  __shared__ volatile uint32_t abort_flag;

  if constexpr (!CL) release_dependents();
  const int G = p.kv_group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  // block -> head, and the `item`-th of all parts: sequence b, part `split` of n_parts
  int h_kv = blockIdx.x % p.cache.N_kv;
  int item = blockIdx.x / p.cache.N_kv, b = 0, split = 0, n_parts = p.splits, n_steps = 0;
  if constexpr (CL) {
    split = blockIdx.x % p.splits;
    item = blockIdx.x / p.splits;
    b = item / p.cache.N_kv;
    h_kv = item % p.cache.N_kv;
    n_steps = steps_of(p, b);
  } else if (p.parts == 0) {
    b = item / p.splits;
    split = item % p.splits;
    n_steps = steps_of(p, b);
  } else {
    const int part = part_steps(p);
    bool found = false;
    for (int b0 = 0; b0 < p.B && !found; b0 += 32) {
      const int steps = b0 + lane < p.B ? steps_of(p, b0 + lane) : 0, n = b0 + lane < p.B ? parts_of(p, steps, part) : 0;
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      const unsigned int past = __ballot_sync(0xffffffffu, upto > item);
      found = past != 0u;
      const int from = found ? __ffs(past) - 1 : 31;
      const int before = __shfl_sync(0xffffffffu, found ? upto - n : upto, from);
      item -= before;
      b = b0 + from;
      split = item;
      n_parts = __shfl_sync(0xffffffffu, n, from);
      n_steps = __shfl_sync(0xffffffffu, steps, from);
    }
    if (!found) return;
  }
  const int unit_kv = b * p.cache.N_kv + h_kv;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kSlots; ++i) mbar_init(&full[0][0] + i, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();

  int len = p.cache.S_max;
  if (p.seq_lens != nullptr) len = min(len, max(0, p.seq_lens[b]));
  const int n_rec = (len + kKv4Rows - 1) / kKv4Rows;
  const int per = ((n_steps + n_parts - 1) / n_parts + kWarps - 1) / kWarps * kWarps;
  const int s0 = split * per + warp, s1 = min(n_steps, (split + 1) * per);      // this warp: steps s0, s0 + 4, .. before s1

  constexpr int kStepBytes = kStepRecs * R::kBytes;
  uint8_t* ring = ksm + warp * (kSlots * kStepBytes);
  const bool paged = p.cache.table != nullptr;
  const uint8_t* records = p.cache.records;
  if (!paged) records += (static_cast<int64_t>(b) * p.cache.N_kv + h_kv) * p.cache.recs * R::kBytes;
  const uint64_t policy = read_once_policy();
  int pages = 0;                       // lane i: the page of the i-th of the last 32 records asked for, two for each step
  auto issue = [&](int step, int slot, int turn) {      // a step's records into a ring slot; the whole warp calls it
    const int rec = step * kStepRecs;
    const bool both = rec + 1 < n_rec;
    const uint8_t *src, *src1;
    if (paged) {
      if (turn % 16 == 0) {
        const int r = (step + (lane >> 1) * kWarps) * kStepRecs + (lane & 1);
        pages = r < n_rec ? p.cache.table[static_cast<int64_t>(b) * p.cache.max_pages + (r >> p.cache.page_shift)] : 0;
        pages = min(max(pages, 0), p.cache.num_pages - 1);
      }
      const int64_t page = __shfl_sync(0xffffffffu, pages, turn % 16 * 2), page1 = __shfl_sync(0xffffffffu, pages, turn % 16 * 2 + 1);
      const int mask = (1 << p.cache.page_shift) - 1;
      src = records + (((page * p.cache.N_kv + h_kv) << p.cache.page_shift) + (rec & mask)) * R::kBytes;
      src1 = records + (((page1 * p.cache.N_kv + h_kv) << p.cache.page_shift) + ((rec + 1) & mask)) * R::kBytes;
    } else {
      src = records + static_cast<int64_t>(rec) * R::kBytes;
      src1 = src + R::kBytes;
    }
    if (elect_one()) {
      uint64_t* bar = &full[warp][slot];
      uint8_t* dst = ring + slot * kStepBytes;
      mbar_expect_tx(bar, both ? kStepBytes : R::kBytes);
      if (both && src1 == src + R::kBytes) {
        bulk_load(dst, src, kStepBytes, bar, policy);
      } else {
        bulk_load(dst, src, R::kBytes, bar, policy);
        if (both) bulk_load(dst + R::kBytes, src1, R::kBytes, bar, policy);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kSlots - 1; ++i)
    if (s0 + i * kWarps < s1) issue(s0 + i * kWarps, i, i);

  // ---- the query heads as B fragments (column g = head g), columns of Q in the order of the codes: of a thread's eight 32 grp +
  // 8 t + .. of a group the pairs (0, 4), (1, 5), (2, 6), (3, 7); in fp16 the second and fourth pair divided by 16
  // f_head: what takes the products of heads 2 t and 2 t + 1 to scores in log2 units
  uint32_t qb[HI][2 * NG][2], qm[HI][2];
  float f_head[HI][2];
#pragma unroll
  for (int hi = 0; hi < HI; ++hi) {
    const int head = kSpare ? g & 3 : g + 8 * hi;
    uint4 u[NG];
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const int d = 32 * grp + 8 * t;
      u[grp] = make_uint4(0u, 0u, 0u, 0u);
      if (head < G && d < p.D)
        u[grp] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(b) * p.N + h_kv * G + head) * p.D + d);
    }
    float lift = 1.0f;
    f_head[hi][0] = f_head[hi][1] = p.scale_log2;
    if constexpr (!BF16) {      // the largest value of the head to 2^10 or more; an infinity or a NaN is larger than that
      constexpr uint32_t kAbs = 0x7fff7fffu;
      uint32_t most = 0u;
#pragma unroll
      for (int grp = 0; grp < NG; ++grp)
        most = __vmaxu2(most, __vmaxu2(__vmaxu2(u[grp].x & kAbs, u[grp].y & kAbs), __vmaxu2(u[grp].z & kAbs, u[grp].w & kAbs)));
      most = max(most & 0xffffu, most >> 16);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int up = max(0, 25 - max(1, static_cast<int>(most >> 10)));      // (2^10 has 25 in its exponent's bits)
      lift = __int_as_float((127 + up) << 23);
      const float back = __int_as_float((127 - up) << 23);
#pragma unroll
      for (int e = 0; e < 2; ++e) f_head[hi][e] *= kCodeScaleF16 * __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
    }
    float mean_t = 0.f;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const uint32_t pairs[4] = {__byte_perm(u[grp].x, u[grp].z, 0x5410), __byte_perm(u[grp].x, u[grp].z, 0x7632),
                                 __byte_perm(u[grp].y, u[grp].w, 0x5410), __byte_perm(u[grp].y, u[grp].w, 0x7632)};
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<BF16>(pairs[j]);
        sum += f.x + f.y;
        const float times = (j & 1) != 0 ? 0.0625f * lift : lift;
        qb[hi][2 * grp + (j >> 1)][j & 1] = BF16 ? pairs[j] : pack2<BF16>(f.x * times, f.y * times);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == grp) mean_t = sum * (lift * 0.03125f);          // of the group's 32 columns: in the range of Q whatever that is
    }
    // the mean as a sum of three 16-bit numbers
    const uint32_t w0 = pack2<BF16>(mean_t, 0.f);
    const float rest1 = mean_t - unpack2<BF16>(w0).x;
    const uint32_t w1 = pack2<BF16>(rest1, 0.f);
    const float rest2 = rest1 - unpack2<BF16>(w1).x;
    qm[hi][0] = (w0 & 0xffffu) | (w1 << 16);
    qm[hi][1] = pack2<BF16>(rest2, 0.f);
  }

  // O^T: rows g and g + 8 of tile (grp, j) are columns 32 grp + 4 g + 2 j and the next; columns heads 2 t and 2 t + 1
  float o[HI][2 * NG][4];
  float m_run[HI][2], l_run[HI][2];      // heads 2 t and 2 t + 1; l is this thread's share
#pragma unroll
  for (int hi = 0; hi < HI; ++hi) {
    m_run[hi][0] = m_run[hi][1] = kLowest;
    l_run[hi][0] = l_run[hi][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[hi][i][e] = 0.f;
  }
  constexpr float kMean = BF16 ? 32.0f : 32.0f / kCodeScaleF16;      // a mean's product in the units of the codes' products

  float* scores = p.scores == nullptr ? nullptr : p.scores + (static_cast<int64_t>(unit_kv) * p.S_pad + g) * p.G_pad + 2 * t;

  int turn = 0, slot = 0;
  uint32_t parity = 0;
  for (int step = s0; step < s1; step += kWarps, ++turn) {
    if (step + (kSlots - 1) * kWarps < s1) issue(step + (kSlots - 1) * kWarps, slot == 0 ? kSlots - 1 : slot - 1, turn + kSlots - 1);
    mbar_wait(&full[warp][slot], parity, &abort_flag, p.status, DEV_TIMEOUT_TMA);
    const uint8_t* rec0 = ring + slot * kStepBytes;
    const int row0 = step * (kStepRecs * kKv4Rows);
    const bool partial = row0 + kStepRecs * kKv4Rows > len;      // (then what is there of the second record may be an earlier one)

    // ---- S^T = K Q^T, in log2 units: x[record][hi] = rows g (0, 1) and g + 8 (2, 3), heads 2 t and 2 t + 1
    float x[kStepRecs][HI][4];
#pragma unroll
    for (int r = 0; r < kStepRecs; ++r) {
      const uint8_t* rec = rec0 + r * R::kBytes;
      uint32_t kw[2 * NG], low[2] = {0u, 0u};
      float step_of[2][NG];
      lane_words<NG>(rec, lane, kw);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (t < NG) low[half] = *reinterpret_cast<const uint16_t*>(rec + R::k_min(half * 8, 0) + (g * NG + t) * 2);
        low[half] = __byte_perm(low[half], 0u, 0x1010);
        row_steps<NG, BF16>(rec + R::k_step(half * 8, 0) + g * NG * 2, step_of[half]);
      }
#pragma unroll
      for (int hi = 0; hi < HI; ++hi)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[r][hi][e] = 0.f;
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        uint32_t ka[2][4];
        key_codes<BF16>(kw[grp], ka[0]);
        key_codes<BF16>(kw[NG + grp], ka[1]);
#pragma unroll
        for (int hi = 0; hi < HI; ++hi) {
          float c[4];
          mma16816_zero<BF16>(c, ka[0][0], ka[1][0], ka[0][1], ka[1][1], qb[hi][2 * grp][0], qb[hi][2 * grp][1]);
          mma16816<BF16>(c, ka[0][2], ka[1][2], ka[0][3], ka[1][3], qb[hi][2 * grp + 1][0], qb[hi][2 * grp + 1][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][hi][e] = fmaf(c[e], step_of[e >> 1][grp], x[r][hi][e]);
        }
      }
#pragma unroll
      for (int hi = 0; hi < HI; ++hi) {
        float c[4];
        mma16816_zero<BF16>(c, low[0], low[1], low[0], low[1], qm[hi][0], qm[hi][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[r][hi][e] = fmaf(c[e], kMean, x[r][hi][e]) * f_head[hi][e & 1];
      }
    }
    if (partial) {
#pragma unroll
      for (int r = 0; r < kStepRecs; ++r)
#pragma unroll
        for (int hi = 0; hi < HI; ++hi)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (row0 + r * kKv4Rows + g + 8 * (e >> 1) >= len) x[r][hi][e] = -INFINITY;
    }
    if (scores != nullptr) {
      float* at = scores + static_cast<int64_t>(row0) * p.G_pad;
#pragma unroll
      for (int r = 0; r < kStepRecs; ++r) {
        if (r > 0 && row0 + r * kKv4Rows >= len) break;
#pragma unroll
        for (int hi = 0; hi < HI; ++hi)
          if (8 * hi + 2 * t < G) {
            *reinterpret_cast<float2*>(at + 8 * hi) = make_float2(x[r][hi][0], x[r][hi][1]);
            *reinterpret_cast<float2*>(at + 8 * p.G_pad + 8 * hi) = make_float2(x[r][hi][2], x[r][hi][3]);
          }
        at += kKv4Rows * p.G_pad;
      }
    }
    // ---- online softmax
    bool exceeds = false;
    float most[HI][2];
#pragma unroll
    for (int hi = 0; hi < HI; ++hi)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        most[hi][e] = fmaxf(x[0][hi][e], x[0][hi][e + 2]);
#pragma unroll
        for (int r = 1; r < kStepRecs; ++r) most[hi][e] = fmax3(most[hi][e], x[r][hi][e], x[r][hi][e + 2]);
        exceeds |= most[hi][e] > m_run[hi][e] + kRefresh;
      }
    if (__any_sync(0xffffffffu, exceeds)) {
#pragma unroll
      for (int hi = 0; hi < HI; ++hi)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = most[hi][e];
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_new = fmaxf(m_run[hi][e], mx);
          const float alpha = ex2(m_run[hi][e] - m_new);
          m_run[hi][e] = m_new;
          l_run[hi][e] *= alpha;
#pragma unroll
          for (int i = 0; i < 2 * NG; ++i) {
            o[hi][i][e] *= alpha;
            o[hi][i][e + 2] *= alpha;
          }
        }
    }
    // ---- P, and O^T += V^T P
#pragma unroll
    for (int r = 0; r < kStepRecs; ++r) {
      // P in 16 bits is the operand of P V, and what that leaves of it another one; the sum of P is of what it was before
      uint32_t pb[HI][2], rest[HI][2];
#pragma unroll
      for (int hi = 0; hi < HI; ++hi) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = ex2(x[r][hi][e] - m_run[hi][e & 1]);
        l_run[hi][0] += pr[0] + pr[2];
        l_run[hi][1] += pr[1] + pr[3];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w = pack2<BF16>(pr[2 * e], pr[2 * e + 1]);
          const float2 f = unpack2<BF16>(w);
          const uint32_t left = pack2<BF16>(pr[2 * e] - f.x, pr[2 * e + 1] - f.y);
          if (kSpare && t >= 2) w = left;
          pb[hi][e] = transpose8(w);
          if (kRest) rest[hi][e] = transpose8(left);
        }
      }
      const uint8_t* rec = rec0 + r * R::kBytes;
      uint32_t vw[2 * NG], vsm[2][2 * NG];
      lane_words<NG>(rec + R::kV, R::v_place(g, t), vw);
      load_words<2 * NG>(rec + R::kVsm + t * NG * 8, vsm[0]);
      load_words<2 * NG>(rec + R::kVsm + (4 + t) * NG * 8, vsm[1]);
      if (partial) {      // rows that do not exist: whatever their steps and minima are, 0 times them has to be 0
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int row = row0 + r * kKv4Rows + q * 8 + 2 * t;
          const uint32_t there = (row < len ? 0xffffu : 0u) | (row + 1 < len ? 0xffff0000u : 0u);
#pragma unroll
          for (int i = 0; i < 2 * NG; ++i) vsm[q][i] &= there;
        }
      }
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        uint32_t v0[4], v1[4];
        kv4_value_pairs<BF16>(vw[grp], vsm[0][2 * grp], vsm[0][2 * grp + 1], v0);
        kv4_value_pairs<BF16>(vw[NG + grp], vsm[1][2 * grp], vsm[1][2 * grp + 1], v1);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int hi = 0; hi < HI; ++hi) {
            mma16816<BF16>(o[hi][2 * grp + j], v0[2 * j], v0[2 * j + 1], v1[2 * j], v1[2 * j + 1], pb[hi][0], pb[hi][1]);
            if (kRest) mma16816<BF16>(o[hi][2 * grp + j], v0[2 * j], v0[2 * j + 1], v1[2 * j], v1[2 * j + 1], rest[hi][0], rest[hi][1]);
          }
      }
    }
    if (++slot == kSlots) { slot = 0; parity ^= 1u; }
    __syncwarp();      // every lane has read this slot before a later copy may land in it
  }

  // ---- merge the four warps per query head, then write the part's result (the rings are dead by now: their memory holds the
  // warps' accumulators)
#pragma unroll
  for (int hi = 0; hi < HI; ++hi)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int bit = 4; bit < 32; bit <<= 1) l_run[hi][e] += __shfl_xor_sync(0xffffffffu, l_run[hi][e], bit);
  if (kSpare) {      // (their maxima are those of the heads, of which they are copies)
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[0][i][e] += __shfl_xor_sync(0xffffffffu, o[0][i][e], 2);
  }
  linger_after_abort(&abort_flag);
  __syncthreads();
  float* s_acc = reinterpret_cast<float*>(ksm);                       // [warp][kHeads][DPAD]
  float* s_m = s_acc + kWarps * kHeads * DPAD;                        // [warp][kHeads]
  float* s_l = s_m + kWarps * kHeads;
#pragma unroll
  for (int hi = 0; hi < HI; ++hi)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = warp * kHeads + 8 * hi + 2 * t + e;
      if (g == 0) { s_m[head] = m_run[hi][e]; s_l[head] = l_run[hi][e]; }
#pragma unroll
      for (int grp = 0; grp < NG; ++grp)
        *reinterpret_cast<float4*>(s_acc + head * DPAD + 32 * grp + 4 * g) =
            make_float4(o[hi][2 * grp][e], o[hi][2 * grp][e + 2], o[hi][2 * grp + 1][e], o[hi][2 * grp + 1][e + 2]);
    }
  __syncthreads();
  // the block's result of a head: acc[d], maximum, sum
  auto of_head = [&](int head, float& big, float& lsum, float (&weight)[kWarps]) {
    big = -INFINITY;
    lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) big = fmaxf(big, s_m[w * kHeads + head]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = s_m[w * kHeads + head];
      weight[w] = mw == -INFINITY ? 0.f : ex2(mw - big);
      lsum = fmaf(s_l[w * kHeads + head], weight[w], lsum);
    }
  };
  if constexpr (!CL) {
    for (int head = 0; head < G; ++head) {
      const int64_t slot = (static_cast<int64_t>(b) * p.N + h_kv * G + head) * p.splits + split;
      float big, lsum, weight[kWarps];
      of_head(head, big, lsum, weight);
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
  } else {
    __shared__ float s_part[kHeads][DPAD], s_pm[kHeads], s_pl[kHeads];      // this block's, which the others of the cluster read
    __shared__ float s_max[kHeads], s_inv[kHeads], s_share[kMaxCluster][kHeads];
    for (int head = 0; head < G; ++head) {
      float big, lsum, weight[kWarps];
      of_head(head, big, lsum, weight);
      for (int d = threadIdx.x; d < p.D; d += kThreads) {
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) a = fmaf(s_acc[(w * kHeads + head) * DPAD + d], weight[w], a);
        s_part[head][d] = a;
      }
      if (threadIdx.x == 0) { s_pm[head] = big; s_pl[head] = lsum; }
    }
    cluster_sync();
    if (threadIdx.x < G) {
      const int head = threadIdx.x;
      float m[kMaxCluster], l[kMaxCluster], big = -INFINITY, sum = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        m[s] = s < p.splits ? cluster_read(&s_pm[head], s) : -INFINITY;
        l[s] = s < p.splits ? cluster_read(&s_pl[head], s) : 0.f;
      }
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) big = fmaxf(big, m[s]);
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        const float w = m[s] == -INFINITY ? 0.f : ex2(m[s] - big);
        s_share[s][head] = w;
        sum = fmaf(l[s], w, sum);
      }
      s_max[head] = big;
      s_inv[head] = sum != 0.f ? 1.0f / sum : 0.f;
    }
    __syncthreads();
    // every splits-th 128 of the group's G x D results
    for (int i = split * kThreads + threadIdx.x; i < G * p.D; i += kThreads * p.splits) {
      const int head = i / p.D, d = i % p.D;
      float v[kMaxCluster], a = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) v[s] = s < p.splits ? cluster_read(&s_part[head][d], s) : 0.f;
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) a = fmaf(v[s], s_share[s][head], a);
      a *= s_inv[head];
      const int64_t at = (static_cast<int64_t>(b) * p.N + h_kv * G + head) * p.D + d;
      if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16(a);
      else reinterpret_cast<__half*>(p.y)[at] = __float2half(a);
    }
    if (p.weights != nullptr) {
      // the keys of this block, whose scores it has written itself; four at a time, whose loads do not wait for one another
      const int first = split * per * kStepRecs * kKv4Rows, end = min(len, first + per * kStepRecs * kKv4Rows);
      const float* row = p.scores + static_cast<int64_t>(unit_kv) * p.S_pad * p.G_pad;
      float* weights = p.weights + static_cast<int64_t>(unit_kv) * p.cache.S_max;
      for (int key0 = first + threadIdx.x; key0 < end; key0 += 4 * kThreads) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = key0 + i * kThreads < end ? weights[key0 + i * kThreads] : 0.f;
        for (int head = 0; head < G; head += 2) {
          const bool two = head + 1 < G;
          const float m0 = s_max[head], i0 = s_inv[head], m1 = two ? s_max[head + 1] : 0.f, i1 = two ? s_inv[head + 1] : 0.f;
          float2 sc[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[i] = key0 + i * kThreads < end ? *reinterpret_cast<const float2*>(row + static_cast<int64_t>(key0 + i * kThreads) * p.G_pad + head)
                                              : make_float2(-INFINITY, -INFINITY);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float sum = ex2(sc[i].x - m0) * i0;
            if (two) sum = fmaf(ex2(sc[i].y - m1), i1, sum);
            w[i] += sum;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + i * kThreads < end) weights[key0 + i * kThreads] = w[i];
      }
    }
    cluster_sync();      // nobody's shared memory goes away while another block still reads it
  }
}

// Joins the parts.  Block (x, unit) has head x of the group for the output, and the keys from x * kFinishKeys on for the weights,
// of which a thread takes four.  What bounds it is latency, so nothing waits for a load before all of them are out: those of the
// parts' maxima and sums, of the first 16 parts of the output, of the weights and of two heads' scores.
constexpr int kFinishThreads = 128, kFinishKeys = 4 * kFinishThreads, kFinishBatch = 16;
template <bool BF16>
__global__ void __launch_bounds__(kFinishThreads) kv4_finish_kernel(const Kv4DecodeParams p) {
  __shared__ float s_share[16][64];      // what a part counts for: exp2(its maximum - the largest)
  __shared__ float s_m[16], s_inv[16];
  const int unit_kv = blockIdx.y, b = unit_kv / p.cache.N_kv, h_kv = unit_kv % p.cache.N_kv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.kv_group, d = threadIdx.x;
  const int64_t unit0 = static_cast<int64_t>(b) * p.N + h_kv * G;      // the group's first query head
  wait_for_primary();
  int len = p.cache.S_max;
  if (p.seq_lens != nullptr) len = min(len, max(0, p.seq_lens[b]));
  const int first = blockIdx.x * kFinishKeys;
  const bool output = blockIdx.x < G, weigh = p.weights != nullptr && first < len;
  if (!output && !weigh) return;
  const int n = parts_of(p, (len + kStepRecs * kKv4Rows - 1) / (kStepRecs * kKv4Rows), p.parts == 0 ? 1 : part_steps(p));

  const float* part = p.part_acc + (unit0 + blockIdx.x) * p.splits * p.D + d;
  float v[kFinishBatch], old[4];
  float2 x[4];
  if (output) {
#pragma unroll
    for (int i = 0; i < kFinishBatch; ++i) v[i] = i < n && d < p.D ? part[static_cast<int64_t>(i) * p.D] : 0.f;
  }
  float* weights = p.weights + static_cast<int64_t>(unit_kv) * p.cache.S_max;
  const float* scores = p.scores + static_cast<int64_t>(unit_kv) * p.S_pad * p.G_pad;
  auto load_scores = [&](int head) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = first + i * kFinishThreads + threadIdx.x;
      x[i] = key < len ? *reinterpret_cast<const float2*>(scores + static_cast<int64_t>(key) * p.G_pad + head) : make_float2(-INFINITY, -INFINITY);
    }
  };
  if (weigh) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = first + i * kFinishThreads + threadIdx.x;
      old[i] = key < len ? weights[key] : 0.f;
    }
    load_scores(0);
  }
  for (int head = weigh ? warp : blockIdx.x + warp * 16; head < (weigh ? G : blockIdx.x + 1); head += kFinishThreads / 32) {
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + (unit0 + head) * p.splits;
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 e0 = lane < n ? ml[lane] : none, e1 = 32 + lane < n ? ml[32 + lane] : none;
    float big = fmaxf(e0.x, e1.x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
    const float w0 = e0.x == -INFINITY ? 0.f : ex2(e0.x - big), w1 = e1.x == -INFINITY ? 0.f : ex2(e1.x - big);
    float l = e0.y * w0 + e1.y * w1;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    s_share[head][lane] = w0;
    s_share[head][32 + lane] = w1;
    if (lane == 0) { s_m[head] = big; s_inv[head] = inv; }
  }
  __syncthreads();
  if (output && d < p.D) {
    float a = 0.f;
    for (int i0 = 0; i0 < n; i0 += kFinishBatch) {
      if (i0 > 0) {
#pragma unroll
        for (int i = 0; i < kFinishBatch; ++i) v[i] = i0 + i < n ? part[static_cast<int64_t>(i0 + i) * p.D] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kFinishBatch; ++i) a = fmaf(v[i], s_share[blockIdx.x][i0 + i], a);
    }
    a *= s_inv[blockIdx.x];
    const int64_t at = (unit0 + blockIdx.x) * p.D + d;
    if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16(a);
    else reinterpret_cast<__half*>(p.y)[at] = __float2half(a);
  }
  if (!weigh) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int head = 0; head < G; head += 2) {
    if (head > 0) load_scores(head);
    const bool two = head + 1 < G;
    const float m0 = s_m[head], i0 = s_inv[head], m1 = two ? s_m[head + 1] : 0.f, i1 = two ? s_inv[head + 1] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = fmaf(ex2(x[i].x - m0), i0, w[i]);
      if (two) w[i] = fmaf(ex2(x[i].y - m1), i1, w[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = first + i * kFinishThreads + threadIdx.x;
    if (key < len) weights[key] = old[i] + w[i];
  }
}

template <int NG>
cudaError_t launch_ng(const Kv4DecodeParams& p, bool bf16, cudaStream_t stream, int* resident) {
  const int heads = p.kv_group > 8 ? 16 : p.kv_group > 4 ? 8 : 4;
  const size_t ring = static_cast<size_t>(kWarps) * kSlots * kStepRecs * Kv4Record<NG>::kBytes;
  const size_t merge = static_cast<size_t>(kWarps) * (heads > 8 ? 16 : 8) * (32 * NG + 2) * sizeof(float);
  // No more blocks to an SM than the grid counts on, also where fewer groups need less: with room for more, some SMs are given more
  // and others fewer, and everybody waits for the former.
  const size_t least = (227 << 10) / (blocks_per_sm(heads) + 1) + 1;
  const size_t smem = std::max({ring, merge, least});
#define KV4_DECODE(BF, HEADS) (p.clustered ? kv4_decode_kernel<NG, BF, HEADS, true> : kv4_decode_kernel<NG, BF, HEADS, false>)
#define KV4_DECODE_HEADS(BF) (heads == 4 ? KV4_DECODE(BF, 4) : heads == 8 ? KV4_DECODE(BF, 8) : KV4_DECODE(BF, 16))
  void (*kern)(const Kv4DecodeParams) = bf16 ? KV4_DECODE_HEADS(true) : KV4_DECODE_HEADS(false);
#undef KV4_DECODE_HEADS
#undef KV4_DECODE
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.parts == 0 ? p.B * p.splits : p.parts + p.B) * p.cache.N_kv);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.clustered ? 1 : 0;
  if (resident != nullptr) return resident_clusters(reinterpret_cast<const void*>(kern), cfg, p.splits, resident);
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

int kv4_decode_blocks_per_sm(int kv_group) { return blocks_per_sm(kv_group); }

cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, bool bf16, cudaStream_t stream, int* resident) {
  const int groups = (p.D + 31) / 32;
  const cudaError_t e = groups == 1   ? launch_ng<1>(p, bf16, stream, resident)
                        : groups == 2 ? launch_ng<2>(p, bf16, stream, resident)
                        : groups == 3 ? launch_ng<3>(p, bf16, stream, resident)
                                      : launch_ng<4>(p, bf16, stream, resident);
  if (e != cudaSuccess || p.clustered) return e;
  const int chunks = p.weights != nullptr ? (p.cache.S_max + kFinishKeys - 1) / kFinishKeys : 1;
  const dim3 grid(chunks > p.kv_group ? chunks : p.kv_group, p.B * p.cache.N_kv);
  return launch_behind(bf16 ? kv4_finish_kernel<true> : kv4_finish_kernel<false>, p, grid, kFinishThreads, stream);
}

}  // namespace acct
