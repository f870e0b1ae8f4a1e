// What stays of a cache: of every head the last `recent` slots, and of those before them the ones with the largest weights, up to
// `keep` in all, in their order, into another cache.
//
// Selection (one block per head): the weights as integers that order alike, and the need-th largest of them, T, by counting into
// 2 048 bins between the smallest and the largest and comparing the few in its bin; then all above T and the first of those
// equal to it, placed by one prefix sum.  The result depends on no order of execution.  The copy (a warp for two records of the smaller
// cache) takes codes as they are: nothing is decoded and rounded again.
//
// 32 sequences of up to 8 192 slots, 8 heads of 128, half of them stay: 197 us with the read that follows, 145 at the rate of a copy.  The
// copy is bound by its reads: two rows of V share their words, and four rows of K a sector of steps, so neighbours that go are read
// with those that stay (16 x 8 heads of 8 192 slots: 135 MB for 84 that stay, at 55 % of the DRAM rate).  Selection there is latency, 17 us.
#include "fa_kernels.cuh"
#include "kv4_common.cuh"

namespace acct {
namespace {

constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBinBits = 11, kBins = 1 << kBinBits, kPerThread = kBins / kSelectThreads;
constexpr uint32_t kListed = 512;           // members of a bin that are compared with one another
constexpr int kCopyWarps = 8, kCopyRecs = 2;      // records that a warp copies at a time, for the loads in flight
constexpr int kSharedKeys = 48 * 1024;      // weights that the long form keeps in shared memory (192 KB)

// A weight as an integer that orders like it; a NaN is the largest.  Never 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);      // (-0 is 0)
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

// E > 0: a thread holds E neighbouring weights in registers.  E = 0: any number, in shared memory up to kSharedKeys, else read
// again for every count.
template <int E>
__global__ void __launch_bounds__(kSelectThreads, E == 16 ? 2 : 1) kv4_select_kernel(const Kv4EvictParams p) {
  extern __shared__ uint32_t shared_keys[];
  __shared__ uint32_t bins[kBins], list[kListed], s_most[kSelectWarps], s_least[kSelectWarps];
  __shared__ uint32_t s_bin, s_above, s_members, s_value;
  __shared__ int s_listed;
  __shared__ unsigned long long warp_total[kSelectWarps];
  release_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int unit = blockIdx.x, b = unit / p.src.N_kv;
  const int len = min(max(p.seq_lens[b], 0), p.src.S_max);
  const int total = min(len, p.keep);
  const int old = max(0, len - p.recent);
  const int need = total - (len - old);            // of the old ones
  const float* w = p.weights + static_cast<int64_t>(unit) * p.src.S_max;
  int* kept = p.kept + static_cast<int64_t>(unit) * p.keep;
  float* out = p.weights_out + static_cast<int64_t>(unit) * p.dst.S_max;

  if (unit % p.src.N_kv == 0 && tid == 0) p.seq_lens_out[b] = total;
  // the recent ones, and nothing behind them
  for (int i = tid; i < len - old; i += kSelectThreads) {
    kept[need + i] = old + i;
    out[need + i] = w[old + i];
  }
  for (int i = total + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
  for (int i = total + tid; i < p.dst.S_max; i += kSelectThreads) out[i] = 0.f;
  if (need <= 0) return;

  // this thread's share: neighbours, so that a prefix sum over threads is one over slots
  const int per = E > 0 ? E : ((old + kSelectThreads - 1) / kSelectThreads) | 1;      // (odd: lanes on distinct banks)
  const int first = min(tid * per, old), last = min(first + per, old);
  uint32_t key[E > 0 ? E : 1];
  const bool shared = E == 0 && old <= kSharedKeys;
  if constexpr (E > 0) {
#pragma unroll
    for (int i = 0; i < E; ++i) key[i] = first + i < last ? order_key(w[first + i]) : 0u;
  } else if (shared) {
    for (int i = tid; i < old; i += kSelectThreads) shared_keys[i] = order_key(w[i]);
    __syncthreads();
  }
  auto each = [&](auto&& f) {      // f(slot, key) for this thread's share, in order; key 0 where there is none: all lanes keep step
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) f(first + i, key[i]);
    } else {
      for (int i = first; i < first + per; ++i) f(i, i >= last ? 0u : shared ? shared_keys[i] : order_key(w[i]));
    }
  };

  uint32_t T = 0u;
  if (need < old) {
    uint32_t most = 0u, least = 0xffffffffu;
    each([&](int, uint32_t k) {
      if (k != 0u) { most = max(most, k); least = min(least, k); }
    });
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) { s_most[warp] = most; s_least[warp] = least; }
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, s_most[lane % kSelectWarps]);
    least = __reduce_min_sync(0xffffffffu, s_least[lane % kSelectWarps]);
    // Rounds: the keys from `least` to `most` into kBins bins of equal width, and on with the bin in which the need-th largest
    // lies, until it is one value wide or its members are few.
    uint32_t wanted = static_cast<uint32_t>(need);
    for (;;) {
      const int shift = max(0, 32 - __clz(most - least) - kBinBits);
      each([&](int, uint32_t k) {
        const bool in = k >= least && k <= most && k != 0u;
        const uint32_t bin = (k - least) >> shift;
        // weights that are alike, zeros above all, would queue for one word: those of the first lane's bin are counted by the warp
        const uint32_t first_bin = __shfl_sync(0xffffffffu, bin, 0);
        const unsigned int same = __ballot_sync(0xffffffffu, in && bin == first_bin);
        if (lane == 0 && same != 0u) atomicAdd(&bins[first_bin], __popc(same));
        if (in && bin != first_bin) atomicAdd(&bins[bin], 1u);
      });
      __syncthreads();
      // from the top: thread t has bins kBins - 1 - t * kPerThread and the next lower ones
      uint32_t n = 0u;
      uint32_t own[kPerThread];
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) n += own[i] = bins[kBins - 1 - (tid * kPerThread + i)];
      uint32_t upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      if (lane == 31) s_most[warp] = upto;
      __syncthreads();
      uint32_t before = upto - n;
#pragma unroll
      for (int i = 0; i < kSelectWarps; ++i)
        if (i < warp) before += s_most[i];
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        if (before < wanted && before + own[i] >= wanted) {      // exactly one bin of one thread
          s_bin = kBins - 1 - (tid * kPerThread + i);
          s_above = before;
          s_members = own[i];
        }
        before += own[i];
      }
      if (tid == 0) s_listed = 0;
      __syncthreads();
      const uint32_t bin = s_bin, members = s_members;
      wanted -= s_above;
      least += bin << shift;
      const uint32_t width = (1u << shift) - 1u;
      most = most - least > width ? least + width : most;
      T = least;
      if (shift == 0) break;
      if (members <= kListed) {
        each([&](int, uint32_t k) {
          if (k >= least && k <= most && k != 0u) list[atomicAdd(&s_listed, 1)] = k;
        });
        __syncthreads();
        for (uint32_t i = tid; i < members; i += kSelectThreads) {
          const uint32_t k = list[i];
          uint32_t larger = 0u, not_smaller = 0u;
          for (uint32_t j = 0; j < members; ++j) {
            larger += list[j] > k;
            not_smaller += list[j] >= k;
          }
          if (larger < wanted && not_smaller >= wanted) s_value = k;      // (threads with equal keys write the same)
        }
        __syncthreads();
        T = s_value;
        break;
      }
      for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
      __syncthreads();
    }
  }
  // counts above T and equal to T, and what the threads before this one have of them
  uint32_t above = 0u, equal = 0u;
  each([&](int, uint32_t k) {
    above += k > T; equal += k == T && k != 0u;
  });
  unsigned long long mine = (static_cast<unsigned long long>(above) << 32) | equal, upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) warp_total[warp] = upto;
  __syncthreads();
  unsigned long long before = upto - mine, all = 0ull;
#pragma unroll
  for (int i = 0; i < kSelectWarps; ++i) {
    const unsigned long long x = warp_total[i];
    all += x;
    if (i < warp) before += x;
  }
  uint32_t n_above = static_cast<uint32_t>(before >> 32), n_equal = static_cast<uint32_t>(before);
  const uint32_t take_equal = static_cast<uint32_t>(need) - static_cast<uint32_t>(all >> 32);
  each([&](int slot, uint32_t k) {
    const bool is_above = k > T, is_equal = k == T && k != 0u;
    if (is_above || (is_equal && n_equal < take_equal)) {
      const uint32_t at = n_above + min(n_equal, take_equal);
      kept[at] = slot;
      out[at] = w[slot];
    }
    n_above += is_above;
    n_equal += is_equal;
  });
}

// One warp for two records of the smaller cache: lane (g, t) collects the words that it has there, from wherever its rows were.
template <int NG>
__global__ void __launch_bounds__(kCopyWarps * 32) kv4_gather_kernel(const Kv4EvictParams p) {
  using R = Kv4Record<NG>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int items = (p.keep + kCopyRecs * kKv4Rows - 1) / (kCopyRecs * kKv4Rows);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kCopyWarps + (threadIdx.x >> 5);
  const int unit = static_cast<int>(item / items), rec0 = static_cast<int>(item % items) * kCopyRecs;
  if (unit >= p.src.B * p.src.N_kv) return;
  wait_for_primary();
  const int b = unit / p.src.N_kv, h = unit % p.src.N_kv;
  const int at = rec0 * kKv4Rows + lane;          // lane l: row l % 16 of record l / 16
  const int slot = at < p.keep ? p.kept[static_cast<int64_t>(unit) * p.keep + at] : -1;
  const unsigned int there = __ballot_sync(0xffffffffu, slot >= 0);      // (kept slots come first)
  if (there == 0u) return;
  const uint8_t* mine = slot >= 0 ? kv4_record(p.src, b, h, slot / kKv4Rows, R::kBytes) : nullptr;
  const int mine_row = slot & (kKv4Rows - 1);

  uint32_t kw[kCopyRecs][2][NG], va[kCopyRecs][2][NG], vb[kCopyRecs][2][NG], sel[kCopyRecs][2];
#pragma unroll
  for (int r = 0; r < kCopyRecs; ++r)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      auto row_of = [&](int i, int& row) {
        row = __shfl_sync(0xffffffffu, mine_row, r * kKv4Rows + i);
        return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r * kKv4Rows + i));
      };
      int row, ra, rb;
      const uint8_t *src = row_of(half * 8 + g, row), *sa = row_of(half * 8 + 2 * t, ra), *sb = row_of(half * 8 + 2 * t + 1, rb);
#pragma unroll
      for (int i = 0; i < NG; ++i) kw[r][half][i] = va[r][half][i] = vb[r][half][i] = 0u;
      if (src != nullptr) kv4_load_words<NG>(src, (row >> 3) * NG, (row & 7) * 4 + t, kw[r][half]);
      if (sa != nullptr) kv4_load_words<NG>(sa + R::kV, (ra >> 3) * NG, R::v_place(g, (ra & 7) >> 1), va[r][half]);
      if (sb != nullptr) kv4_load_words<NG>(sb + R::kV, (rb >> 3) * NG, R::v_place(g, (rb & 7) >> 1), vb[r][half]);
      sel[r][half] = ((ra & 1) != 0 ? 0x32u : 0x10u) | ((rb & 1) != 0 ? 0x7600u : 0x5400u);
    }
  // steps and minima of this lane's row
  uint16_t ks[NG], km[NG], vs[NG], vm[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    ks[i] = km[i] = vs[i] = vm[i] = 0;
    if (mine != nullptr) {
      ks[i] = *reinterpret_cast<const uint16_t*>(mine + R::k_step(mine_row, i));
      km[i] = *reinterpret_cast<const uint16_t*>(mine + R::k_min(mine_row, i));
      vs[i] = *reinterpret_cast<const uint16_t*>(mine + R::v_step(mine_row, i));
      vm[i] = *reinterpret_cast<const uint16_t*>(mine + R::v_min(mine_row, i));
    }
  }
  uint8_t* dst[kCopyRecs];
#pragma unroll
  for (int r = 0; r < kCopyRecs; ++r) {
    dst[r] = nullptr;
    if ((there >> (r * kKv4Rows)) == 0u) continue;
    dst[r] = kv4_record(p.dst, b, h, rec0 + r, R::kBytes);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      kv4_store_words<NG>(dst[r], half * NG, lane, kw[r][half]);
      uint32_t w[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) w[i] = __byte_perm(va[r][half][i], vb[r][half][i], sel[r][half]);
      kv4_store_words<NG>(dst[r] + R::kV, half * NG, R::v_place(g, t), w);
    }
  }
  uint8_t* to = lane < kKv4Rows ? dst[0] : dst[1];
  const int row = lane & (kKv4Rows - 1);
  if (to == nullptr) return;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    *reinterpret_cast<uint16_t*>(to + R::k_step(row, i)) = ks[i];
    *reinterpret_cast<uint16_t*>(to + R::k_min(row, i)) = km[i];
    *reinterpret_cast<uint16_t*>(to + R::v_step(row, i)) = vs[i];
    *reinterpret_cast<uint16_t*>(to + R::v_min(row, i)) = vm[i];
  }
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream) {
  const int units = p.src.B * p.src.N_kv;
  const int slots = p.src.S_max;
  if (slots <= 4 * kSelectThreads) kv4_select_kernel<4><<<units, kSelectThreads, 0, stream>>>(p);
  else if (slots <= 16 * kSelectThreads) kv4_select_kernel<16><<<units, kSelectThreads, 0, stream>>>(p);
  else if (slots <= 32 * kSelectThreads) kv4_select_kernel<32><<<units, kSelectThreads, 0, stream>>>(p);
  else {
    const size_t smem = sizeof(uint32_t) * (slots < kSharedKeys ? slots : kSharedKeys);
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv4_select_kernel<0>), sizeof(uint32_t) * kSharedKeys);
    if (e != cudaSuccess) return e;
    kv4_select_kernel<0><<<units, kSelectThreads, smem, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t items = static_cast<int64_t>((p.keep + kCopyRecs * kKv4Rows - 1) / (kCopyRecs * kKv4Rows)) * units;
  const unsigned int blocks = static_cast<unsigned int>((items + kCopyWarps - 1) / kCopyWarps);
  const int groups = (p.src.D + 31) / 32;
  return launch_behind(groups == 1   ? kv4_gather_kernel<1>
                       : groups == 2 ? kv4_gather_kernel<2>
                       : groups == 3 ? kv4_gather_kernel<3>
                                     : kv4_gather_kernel<4>,
                       p, dim3(blocks), kCopyWarps * 32, stream);
}

}  // namespace acct
