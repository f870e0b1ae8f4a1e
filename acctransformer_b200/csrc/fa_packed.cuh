// Packed sequences: which tile of which sequence a thread block works on.
#pragma once
#include "fa_kernels.cuh"

namespace acct {

// On the host: the rows of a tile, and what follows from them.  With 2^(s - 1) < d <= 2^s m = ceil(2^(31 + s) / d) has m d = 2^(31 + s) + r
// with r < d <= 2^s, so n * m >> (31 + s) is n / d rounded down while n r < 2^(31 + s), as for any n < 2^31 + 2^20.
inline void set_tile_tokens(FwdParams& p, int tokens) {
  int shift = 0;
  while ((1 << shift) < tokens) ++shift;
  p.tile_tokens = tokens;
  p.tile_shift = 31 + shift;
  p.tile_magic = static_cast<unsigned int>(((uint64_t(1) << p.tile_shift) + static_cast<unsigned int>(tokens) - 1) / static_cast<unsigned int>(tokens));
  p.tile_bound = static_cast<int>((static_cast<int64_t>(p.T_q) + static_cast<int64_t>(tokens - 1) * p.B) / tokens);
}

// What a thread block of the packed form works on: tile `tile` of the sequence whose rows begin at q0 and k0.
struct PackedItem {
  int tile, q0, len_q, k0, len_k;
};

// Finds tiles by their number: all sequences' tiles of `rows` rows, those with the most K/V tiles first (a late start of a long one
// is what the SMs would wait for at the end).  One warp; a lane has sequences lane, lane + 32, ...  Up to 128 sequences their rows
// are read once and the order comes from a search over the number of K/V tiles; with more, long ones matter less, and they
// come one after the other.
class PackedFinder {
 public:
  __device__ __forceinline__ explicit PackedFinder(const FwdParams& params) : p(params), most(0) {}

  // Before the first find(), by the same warp; apart from it so that the loads can be under way while the block sets itself up.
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s[i] = {0, 0, 0, 0, 0};
      if (p.B <= 32 * kPer && lane() + 32 * i < p.B) read(lane() + 32 * i, s[i]);
      most = max(most, (s[i].len_k + kTile - 1) / kTile);
    }
  }

  // The `item`-th tile, the same in all lanes; len_q = 0 where there are not so many.
  __device__ __forceinline__ PackedItem find(int item) const {
    PackedItem found = {0, 0, 0, 0, 0};
    if (p.B <= 32 * kPer) {
      int lo = 0, hi = __reduce_max_sync(0xffffffffu, most) + 1, before = 0;       // count(lo) > item >= count(hi) = before
      if (count(0) <= item) return found;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2, n = count(mid);
        if (n > item) lo = mid;
        else { hi = mid; before = n; }
      }
      int left = item - before;                  // among the tiles with exactly `lo` K/V tiles
      bool done = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (!done && 32 * i < p.B) {
          const int least = with(s[i], lo), n = least - with(s[i], lo + 1);
          done = settle(s[i], n, tiles(s[i]) - least, left, found);
        }
    } else {
      int left = item;
      bool done = false;
      for (int b0 = 0; b0 < p.B && !done; b0 += 32 * kPer) {
        PackedItem x[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          x[i] = {0, 0, 0, 0, 0};
          if (b0 + 32 * i + lane() < p.B) read(b0 + 32 * i + lane(), x[i]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (!done) done = settle(x[i], tiles(x[i]), 0, left, found);
      }
      if (done) found.tile = tiles(found) - 1 - found.tile;
    }
    return found;
  }

 private:
  static constexpr int kPer = 4;
  const FwdParams& p;
  int most;
  PackedItem s[kPer];

  __device__ __forceinline__ static int lane() { return threadIdx.x & 31; }
  __device__ __forceinline__ void read(int b, PackedItem& x) const {      // (whatever cu holds, no row outside [0, T) is touched)
    x.q0 = min(max(p.cu_q[b], 0), p.T_q);
    x.len_q = min(max(p.cu_q[b + 1], x.q0), p.T_q) - x.q0;
    x.k0 = min(max(p.cu_k[b], 0), p.T_k);
    x.len_k = min(max(p.cu_k[b + 1], x.k0), p.T_k) - x.k0;
  }
  // ceil(n / rows of a tile), n >= 0
  __device__ __forceinline__ int in_tiles(int n) const {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n) + static_cast<uint32_t>(p.tile_tokens - 1)) * p.tile_magic >> p.tile_shift);
  }
  __device__ __forceinline__ int tiles(const PackedItem& x) const { return in_tiles(x.len_q); }
  // tiles of the sequence with `many` or more K/V tiles: from a certain one on, with a causal mask
  __device__ __forceinline__ int with(const PackedItem& x, int many) const {
    const int n = tiles(x);
    if (many <= 0) return n;
    const int keys = (many - 1) * kTile + 1;                   // a tile that sees this many
    if (x.len_k < keys) return 0;
    if (!p.mods.causal) return n;
    const int last = keys - (x.len_k - x.len_q);               // ... has its last row here or later
    return n - min(n, in_tiles(max(1, last)) - 1);
  }
  __device__ __forceinline__ int count(int many) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (32 * i < p.B) n += with(s[i], many);
    return __reduce_add_sync(0xffffffffu, n);
  }
  // Among n tiles of this lane's sequence, the first of which is `first`; true where the `left`-th of all lanes' is one.
  __device__ __forceinline__ bool settle(const PackedItem& x, int n, int first, int& left, PackedItem& found) const {
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane() >= d) upto += y;
    }
    const unsigned int past = __ballot_sync(0xffffffffu, upto > left);
    if (past == 0u) {
      left -= __shfl_sync(0xffffffffu, upto, 31);
      return false;
    }
    const int from = __ffs(past) - 1;
    found.tile = __shfl_sync(0xffffffffu, first, from) + left - __shfl_sync(0xffffffffu, upto - n, from);
    found.q0 = __shfl_sync(0xffffffffu, x.q0, from);
    found.len_q = __shfl_sync(0xffffffffu, x.len_q, from);
    found.k0 = __shfl_sync(0xffffffffu, x.k0, from);
    found.len_k = __shfl_sync(0xffffffffu, x.len_k, from);
    return true;
  }
};

}  // namespace acct
