// What stays of a cache: of every head the last `recent` slots, and of those before them the ones with the largest weights, up to
// `keep` in all, in their order, into another cache.
//
// Selection (one block per head): the weights as integers that order alike, and the largest T with at least `need` of them at or
// above it, two bits at a time by counting; then all above T and the first of those equal to it, placed by one prefix sum.  The
// result depends on no order of execution.  The copy (one warp per record of the smaller cache) takes codes as they are: nothing
// is decoded and rounded again.
#include "fa_kernels.cuh"
#include "kv4_common.cuh"

namespace acct {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kCopyWarps = 8;
constexpr int kSharedKeys = 50 * 1024;      // weights that the long form keeps in shared memory (200 KB)

// A weight as an integer that orders like it; a NaN is the largest.  Never 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);      // (-0 is 0)
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

// Sum over the block of three counts, the same in all threads.  `buf` alternates from call to call, so one barrier is enough.
__device__ __forceinline__ void block_sum3(uint32_t (&x)[3], uint32_t (*buf)[kSelectWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t s = __reduce_add_sync(0xffffffffu, x[i]);
    if (lane == 0) buf[i][warp] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) x[i] = __reduce_add_sync(0xffffffffu, buf[i][lane]);
}

// E > 0: a thread holds E neighbouring weights in registers.  E = 0: any number, in shared memory up to kSharedKeys, else read
// again for every count.
template <int E>
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const Kv4EvictParams p) {
  extern __shared__ uint32_t shared_keys[];
  __shared__ uint32_t sums[2][3][kSelectWarps];
  __shared__ unsigned long long warp_total[kSelectWarps];
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
  auto each = [&](auto&& f) {                      // f(slot, key) for this thread's share, in order
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) f(first + i, key[i]);
    } else {
      for (int i = first; i < last; ++i) f(i, shared ? shared_keys[i] : order_key(w[i]));
    }
  };

  uint32_t T = 0u;
  if (need < old) {
    int turn = 0;
    for (int bit = 30; bit >= 0; bit -= 2) {
      uint32_t n[3] = {0u, 0u, 0u};
      const uint32_t c1 = T | (1u << bit), c2 = T | (2u << bit), c3 = T | (3u << bit);
      each([&](int, uint32_t k) {
        n[0] += k >= c1; n[1] += k >= c2; n[2] += k >= c3;
      });
      block_sum3(n, sums[turn]);
      turn ^= 1;
      const uint32_t least = static_cast<uint32_t>(need);
      T = n[2] >= least ? c3 : n[1] >= least ? c2 : n[0] >= least ? c1 : T;
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

// One warp per record of the smaller cache: lane (g, t) collects the words that it has there, from wherever its rows were.
template <int NG>
__global__ void __launch_bounds__(kCopyWarps * 32) kv4_gather_kernel(const Kv4EvictParams p) {
  using R = Kv4Record<NG>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int recs = (p.keep + kKv4Rows - 1) / kKv4Rows;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kCopyWarps + (threadIdx.x >> 5);
  const int unit = static_cast<int>(item / recs), rec = static_cast<int>(item % recs);
  if (unit >= p.src.B * p.src.N_kv) return;
  const int b = unit / p.src.N_kv, h = unit % p.src.N_kv;
  const int* kept = p.kept + static_cast<int64_t>(unit) * p.keep;
  const int at = rec * kKv4Rows + (lane & 15);
  const int slot = at < p.keep ? kept[at] : -1;
  if (__ballot_sync(0xffffffffu, slot >= 0) == 0u) return;       // (kept slots come first)
  const uint8_t* mine = slot >= 0 ? kv4_record(p.src, b, h, slot / kKv4Rows, R::kBytes) : nullptr;
  const int mine_row = slot & (kKv4Rows - 1);
  auto record_of = [&](int row) {
    return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), row));
  };
  uint8_t* dst = kv4_record(p.dst, b, h, rec, R::kBytes);

  uint32_t kw[2][NG], va[2][NG], vb[2][NG];
  uint32_t sel[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint8_t* src = record_of(half * 8 + g);
    const int row = __shfl_sync(0xffffffffu, mine_row, half * 8 + g);
#pragma unroll
    for (int i = 0; i < NG; ++i)
      kw[half][i] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + R::word((row >> 3) * NG + i, (row & 7) * 4 + t)) : 0u;
    const int ra = half * 8 + 2 * t, rb = ra + 1;
    const uint8_t *sa = record_of(ra), *sb = record_of(rb);
    const int wa = __shfl_sync(0xffffffffu, mine_row, ra), wb = __shfl_sync(0xffffffffu, mine_row, rb);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      va[half][i] = sa != nullptr ? *reinterpret_cast<const uint32_t*>(sa + R::kV + R::word((wa >> 3) * NG + i, R::v_place(g, (wa & 7) >> 1))) : 0u;
      vb[half][i] = sb != nullptr ? *reinterpret_cast<const uint32_t*>(sb + R::kV + R::word((wb >> 3) * NG + i, R::v_place(g, (wb & 7) >> 1))) : 0u;
    }
    sel[half] = ((wa & 1) != 0 ? 0x32u : 0x10u) | ((wb & 1) != 0 ? 0x7600u : 0x5400u);
  }
  // steps and minima: lanes 0-15 those of K, 16-31 those of V
  uint16_t step[NG], low[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    step[i] = low[i] = 0;
    if (mine != nullptr) {
      step[i] = *reinterpret_cast<const uint16_t*>(mine + (lane < 16 ? R::k_step(mine_row, i) : R::v_step(mine_row, i)));
      low[i] = *reinterpret_cast<const uint16_t*>(mine + (lane < 16 ? R::k_min(mine_row, i) : R::v_min(mine_row, i)));
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      *reinterpret_cast<uint32_t*>(dst + R::word(half * NG + i, lane)) = kw[half][i];
      *reinterpret_cast<uint32_t*>(dst + R::kV + R::word(half * NG + i, R::v_place(g, t))) = __byte_perm(va[half][i], vb[half][i], sel[half]);
    }
  const int row = lane & 15;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    *reinterpret_cast<uint16_t*>(dst + (lane < 16 ? R::k_step(row, i) : R::v_step(row, i))) = step[i];
    *reinterpret_cast<uint16_t*>(dst + (lane < 16 ? R::k_min(row, i) : R::v_min(row, i))) = low[i];
  }
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream) {
  const int units = p.src.B * p.src.N_kv;
  const int slots = p.src.S_max;
  if (slots <= 2 * kSelectThreads) kv4_select_kernel<2><<<units, kSelectThreads, 0, stream>>>(p);
  else if (slots <= 8 * kSelectThreads) kv4_select_kernel<8><<<units, kSelectThreads, 0, stream>>>(p);
  else if (slots <= 16 * kSelectThreads) kv4_select_kernel<16><<<units, kSelectThreads, 0, stream>>>(p);
  else {
    const size_t smem = sizeof(uint32_t) * (slots < kSharedKeys ? slots : kSharedKeys);
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv4_select_kernel<0>), sizeof(uint32_t) * kSharedKeys);
    if (e != cudaSuccess) return e;
    kv4_select_kernel<0><<<units, kSelectThreads, smem, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t items = static_cast<int64_t>((p.keep + kKv4Rows - 1) / kKv4Rows) * units;
  const unsigned int blocks = static_cast<unsigned int>((items + kCopyWarps - 1) / kCopyWarps);
  const int groups = (p.src.D + 31) / 32;
  if (groups == 1) kv4_gather_kernel<1><<<blocks, kCopyWarps * 32, 0, stream>>>(p);
  else if (groups == 2) kv4_gather_kernel<2><<<blocks, kCopyWarps * 32, 0, stream>>>(p);
  else if (groups == 3) kv4_gather_kernel<3><<<blocks, kCopyWarps * 32, 0, stream>>>(p);
  else kv4_gather_kernel<4><<<blocks, kCopyWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace acct
