// The cache in 4 bits: how a record of 16 rows is laid out, and where it is.
//
// Every 32 neighbouring values of a row (one token, one head; the last group may be short) share a minimum m and a step s, both
// in the cache's 16-bit type, and are codes 0..15; code c stands for c * s + m.  A row of head_dim 128 takes 160 bytes for K and
// V instead of 512.
//
// 16 rows of K and of V of one head are one record, 640 bytes per group of 32 columns (2 560 at head_dim 128), laid out for the
// lanes that multiply it (lane = 4 g + t, as in the operands of mma.m16n8k16), so that one bulk copy brings a record in, a lane
// finds its words side by side, and no word has to be moved between lanes:
//   K codes    lane (g, t), word 8-row half * NG + group: row g of the half, columns 32 group + 8 t .. + 7, nibble = column
//   V codes    lane (g, t), word p * NG + group: rows 8 p + 2 t (low 16 bits) and 8 p + 2 t + 1 (high), columns
//              32 group + 4 g .. + 3, nibble = column: two rows of one column are where an operand of P V has them
//   K steps, K minima   [row][group] each
//   V both     [p][t][group][steps of the two rows, minima of the two rows]
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace acct {

constexpr int kKv4Rows = 16;        // rows of a record
constexpr int kKv4MaxGroups = 4;    // head_dim up to 128

// byte offsets inside a record
template <int NG>
struct Kv4Record {
  static constexpr int kWords = 2 * NG;                 // words of K, and of V, per lane
  static constexpr int kUnit = NG % 2 == 0 ? 4 : 2;     // of which so many are neighbours: [kWords / kUnit][32 lanes][kUnit]
  static constexpr int kV = 256 * NG, kKs = 512 * NG, kKm = 544 * NG, kVsm = 576 * NG, kBytes = 640 * NG;

  // byte offset of word w of the unit at `place` (0..31)
  __host__ __device__ static constexpr int word(int w, int place) { return (((w / kUnit) * 32 + place) * kUnit + w % kUnit) * 4; }
  // Where lane (g, t) has its V words: the eight lanes that hold a pair of rows side by side (a row is read and written alone,
  // too), turned by 2 t so that any eight consecutive lanes still cover all banks.
  __host__ __device__ static constexpr int v_place(int g, int t) { return t * 8 + ((g + 2 * t) & 7); }
  __host__ __device__ static constexpr int k_step(int row, int grp) { return kKs + (row * NG + grp) * 2; }
  __host__ __device__ static constexpr int k_min(int row, int grp) { return kKm + (row * NG + grp) * 2; }
  __host__ __device__ static constexpr int v_step(int row, int grp) { return kVsm + ((((row >> 3) * 4 + ((row & 7) >> 1)) * NG + grp) * 4 + (row & 1)) * 2; }
  __host__ __device__ static constexpr int v_min(int row, int grp) { return v_step(row, grp) + 4; }
};

struct Kv4Cache {
  uint8_t* records;                 // [B, N_kv, recs][record], or pages [num_pages, N_kv, 1 << page_shift][record]
  const int* table;                 // [B, max_pages], or null: contiguous
  int B, N_kv, D, S_max;
  int recs;                         // records per head of a contiguous cache
  int page_shift;                   // records per page = 1 << page_shift
  int max_pages, num_pages;
};

// Record `rec` of a head.  A page number that is none reads and writes page 0 or the last one, never memory outside.
__device__ __forceinline__ uint8_t* kv4_record(const Kv4Cache& c, int b, int h, int rec, int bytes) {
  if (c.table == nullptr) return c.records + ((static_cast<int64_t>(b) * c.N_kv + h) * c.recs + rec) * bytes;
  const int page = min(max(c.table[static_cast<int64_t>(b) * c.max_pages + (rec >> c.page_shift)], 0), c.num_pages - 1);
  return c.records + (((static_cast<int64_t>(page) * c.N_kv + h) << c.page_shift) + (rec & ((1 << c.page_shift) - 1))) * bytes;
}

template <bool BF16>
__device__ __forceinline__ uint32_t kv4_sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t kv4_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (w & mask) | bits
__device__ __forceinline__ uint32_t kv4_mask_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(w), "r"(mask), "r"(bits));
  return d;
}

// The values of the four pairs of codes of a word (nibble j of either half): code * step + minimum, rounded once.  The code is
// subtracted out of 1024 + c, 64 + c or 128 + c.
template <bool BF16>
__device__ __forceinline__ void kv4_value_pairs(uint32_t w, uint32_t step, uint32_t low, uint32_t (&x)[4]) {
  if constexpr (BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = kv4_sub2<true>(kv4_mask_or(w >> (4 * j), 0x000f000fu, 0x43004300u), 0x43004300u);
  } else {
    const uint32_t u = w >> 8;
    x[0] = kv4_sub2<false>(kv4_mask_or(w, 0x000f000fu, 0x64006400u), 0x64006400u);      // 1024 + c
    x[1] = kv4_sub2<false>(kv4_mask_or(w, 0x00f000f0u, 0x54005400u), 0x54005400u);      // 64 + c
    x[2] = kv4_sub2<false>(kv4_mask_or(u, 0x000f000fu, 0x64006400u), 0x64006400u);
    x[3] = kv4_sub2<false>(kv4_mask_or(u, 0x00f000f0u, 0x54005400u), 0x54005400u);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = kv4_fma2<BF16>(x[j], step, low);
}

// the NG neighbouring words from word w of the unit at `place` on
template <int NG>
__device__ __forceinline__ void kv4_store_words(uint8_t* rec, int w, int place, const uint32_t (&x)[NG]) {
  using R = Kv4Record<NG>;
  if constexpr (NG == 4) *reinterpret_cast<uint4*>(rec + R::word(w, place)) = make_uint4(x[0], x[1], x[2], x[3]);
  else if constexpr (NG == 2) *reinterpret_cast<uint2*>(rec + R::word(w, place)) = make_uint2(x[0], x[1]);
  else {
#pragma unroll
    for (int i = 0; i < NG; ++i) *reinterpret_cast<uint32_t*>(rec + R::word(w + i, place)) = x[i];
  }
}
template <int NG>
__device__ __forceinline__ void kv4_load_words(const uint8_t* rec, int w, int place, uint32_t (&x)[NG]) {
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

struct Kv4Rows {                    // rows of tokens outside the cache: [T, N_kv, D]
  void *k, *v;
  int64_t k_stride[2], v_stride[2]; // elements, of a token and of a head
  const int* cu;                    // [B + 1]: sequence b has rows cu[b] .. cu[b + 1] - 1; null: row b, T = B
  const int* start;                 // [B]: the first of them is slot start[b] of its sequence
  int T;
};

struct Kv4DecodeParams {
  Kv4Cache cache;
  const void* q;
  void* y;
  const int* seq_lens;
  float* weights;                   // [B, N_kv, S_max] or null: every key's probability is added, over the group's heads
  float* scores;                    // with weights: [B, N_kv, S_pad, G_pad] scratch
  float* part_acc;                  // [B * N, splits, D]
  float* part_ml;                   // [B * N, splits, 2]
  unsigned int* status;
  int B, N, D, kv_group;
  int splits;                       // most parts of a sequence, and room for so many in part_acc and part_ml
  int parts;                        // 0: every sequence has `splits` parts; else the parts that the whole batch is cut into, about
  int S_pad, G_pad;                 // slots in whole records, query heads per cache head rounded up to an even number
  int clustered;
  float scale_log2;
};

struct Kv4EvictParams {
  Kv4Cache src, dst;
  const float* weights;             // [B, N_kv, src.S_max]
  float* weights_out;               // [B, N_kv, dst.S_max]
  int* kept;                        // [B, N_kv, keep]
  const int* seq_lens;
  int* seq_lens_out;
  int keep, recent;
};

// A kernel that is launched behind another one of the same call starts while that one still runs (programmatic dependent launch):
// its launch and its prologue are off the path.  The first says when (every block, or by ending), the second waits, before it
// touches anything that the first has written, until the whole of the first is done and its writes are visible.
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class P>
cudaError_t launch_behind(void (*kern)(const P), const P& p, dim3 grid, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

cudaError_t launch_kv4_append(const Kv4Cache& c, const Kv4Rows& r, bool bf16, cudaStream_t stream);
cudaError_t launch_kv4_read(const Kv4Cache& c, const Kv4Rows& r, bool bf16, cudaStream_t stream);
int kv4_decode_blocks_per_sm(int kv_group);      // that are resident at once
// (with `resident` nothing is launched: it receives how many clusters of p.splits blocks the device holds at once)
cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, bool bf16, cudaStream_t stream, int* resident = nullptr);
cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream);

}  // namespace acct
