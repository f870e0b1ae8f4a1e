// Attention of packed sequences at head_dim up to 128: the forward of fa_fwd.cu, cut for many sequences of few tiles.
//
// A tile of 128 score rows per block, two blocks per SM (256 columns of tensor memory, half of the registers and of shared memory
// each), every block with a list of tiles, whose next one is looked up while one is worked on.  What a tile needs before its first
// scores and after its last product, a third of its time where a sequence has five tiles of keys, falls under the other block's
// work; the two tiles per block of fa_fwd.cu are at the same point of theirs at the same time.  24 chunks of up to 1 500 tokens, 16
// heads of 64: 226 us, 266 there.  8 prompts of up to 4 096 tokens, 32 heads of 128 on 8: 555 us, 569 there.  (A block for each
// tile instead of lists: 253 and 580, when this took 229 and 550; one block with both tiles as independent streams: 262 and
// 588.)  Long sequences go there (the rule is at acct_infer_packed): two tiles share each load of K and V.
//
// The rows of a tile are `tile_heads` query heads that read one head of K and V, times 128 / tile_heads tokens (row = token *
// heads + head: a box of the tensor map as it is).  K and V are then read once per group instead of once per head, and a tile's
// causal edge is 128 / heads tokens wide, so fewer scores are computed only to be left out.
//
// Warps: 0-3 softmax (thread = score row), 4 loads, 5 MMA, 6 looks up tiles, 7 stores.  Per K/V tile: S = Q K^T -> scores in
// registers, running maximum refreshed only where it grows by more than 2^8, P to tensor memory in two halves -> O += P V.  P is
// rounded to the 16 bits that the product takes, its sum is of the values before that, in 32 bits.  At head_dim up to 64 the next
// scores are formed under this tile's softmax (chunks 220 -> 210 us in a row of calls); above, there is no room for them.
//
// What bounds it: 128 x 128 exponentials take the SM 1 024 clk, and with maxima, sums and 16-bit packing a tile takes it 1 780 clk at
// 8 192 keys of 64 and 1 960 of 128; at 1 024 keys 2 380 and 2 960, as half of every diagonal tile is masked and the tile lists end
// unevenly.  4 prompts of up to 200 tokens, 12.3 us, are latency: 1 000 to 1 500 clk until the block is set up, 2 000 to 2 900 to the
// first tile's number, 2 100 to its scores, 2 000 to 3 500 per K/V tile, 500 to 2 000 for the last P V and 1 100 for the way out.
#include "fa_common.cuh"
#include "fa_kernels.cuh"
#include "fa_packed.cuh"
#include "ptx.cuh"

namespace acct {
namespace {

constexpr int kThreads = 256;
constexpr int kRegsSoftmax = 208, kRegsControl = 48;      // of 128 a thread at launch: 4 x 32 x (208 + 48) = 256 x 128
constexpr float kRescaleThreshold = 8.0f;                 // log2 units

// What the roles have to know of an item.
struct Work {
  int head0, h_kv;
  int q_row, tokens;            // first row of q and o, and how many; 0 rows: the end
  int k_row, kv_len, tiles;     // first row of k and v, rows of the sequence, K/V tiles that the item's last token needs
  int sees;                     // keys that the first token sees (all of them without a causal mask); may be negative
};

struct Shared {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full, s_free, p_half, p_ready, o_done, o_free, o_staged;
  uint64_t work_full[2], work_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
  Work work[2], softmax_work[2];
};

template <int DPAD, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) fa_fwd_packed_kernel(const __grid_constant__ FwdParams p) {
  constexpr int NB = DPAD / 64;                 // 64-column (128-byte) blocks per row
  constexpr uint32_t kTileBytes = NB * 16384u;  // one 128-row tile
  // At head_dim up to 64 there is room for P beside the scores, and for a second K and V: the next scores are formed under this
  // tile's softmax.  Above, P lies over the scores and they follow P V.
  constexpr bool kAhead = DPAD == 64;
  constexpr int kSt = kAhead ? 2 : 1;           // K and V buffers
  constexpr uint32_t kColP = kAhead ? 128 : 0, kColO = kAhead ? 192 : 128;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = sQ + kTileBytes;                // tile n is in buffer n % kSt
  uint8_t* sV = sK + kSt * kTileBytes;          // the last one of an item is also the way out for O, between its P V and the next V
  __shared__ Shared sh;

  const int tid = threadIdx.x;
  const int warp = static_cast<int>(warp_uniform(tid >> 5));
  const bool causal = p.mods.causal != 0;

  PackedFinder finder(p);
  if (warp == 6) finder.load();
  if (tid == 32) {
    mbar_init(&sh.q_full, 1);
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&sh.k_full[i], 1); mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1); mbar_init(&sh.v_empty[i], 1);
    }
    mbar_init(&sh.s_full, 1); mbar_init(&sh.s_free, 128); mbar_init(&sh.p_half, 128); mbar_init(&sh.p_ready, 128);
    mbar_init(&sh.o_done, 1); mbar_init(&sh.o_free, 128); mbar_init(&sh.o_staged, 128);
    for (int i = 0; i < 2; ++i) { mbar_init(&sh.work_full[i], 1); mbar_init(&sh.work_empty[i], 4); }
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 4) { tmem_alloc(&sh.tmem_base, 256); tmem_relinquish(); }
  if (tid == 5 * 32) { prefetch_tmap(&p.map_q); prefetch_tmap(&p.map_k); prefetch_tmap(&p.map_v); prefetch_tmap(&p.map_o); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = warp_uniform(sh.tmem_base);
  volatile uint32_t* abort_flag = &sh.abort_flag;

  // The next item of a role, for a converged warp; `n`: how many it has had.  After a wait that ran out there is no next one.
  auto next_work = [&](uint32_t n) {
    Work w;
    const bool got = mbar_wait(&sh.work_full[n & 1], (n >> 1) & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
    w = sh.work[n & 1];
    if (__any_sync(0xffffffffu, !got)) w.tokens = 0;
    __syncwarp();
    if (elect_one()) mbar_arrive(&sh.work_empty[n & 1]);
    return w;
  };

  if (warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    reg_dealloc<kRegsControl>();
    uint32_t n = 0;      // K/V tiles asked for
    for (uint32_t i = 0;; ++i) {
      const Work w = next_work(i);
      if (w.tokens == 0) break;
      if (elect_one()) {
        if (w.tiles > 0) {      // the scores before were the last to read Q
          if (n > 0) mbar_wait(&sh.k_empty[(n - 1) % kSt], ((n - 1) / kSt) & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
          mbar_expect_tx(&sh.q_full, NB * static_cast<uint32_t>(p.tile_heads * p.tile_tokens) * 128u);
          for (int nb = 0; nb < NB; ++nb) tma_load_4d(sQ + nb * 16384, &p.map_q, &sh.q_full, nb * 64, w.head0, w.q_row, 0);
        }
        for (int it = 0; it < w.tiles; ++it) {
          const uint32_t s = (n + it) % kSt, before = ((n + it) / kSt - 1) & 1;
          const bool used = n + it >= kSt;
          if (used) mbar_wait(&sh.k_empty[s], before, abort_flag, p.status, DEV_TIMEOUT_SYNC);
          mbar_expect_tx(&sh.k_full[s], kTileBytes);
          for (int nb = 0; nb < NB; ++nb)
            tma_load_4d(sK + s * kTileBytes + nb * 16384, &p.map_k, &sh.k_full[s], nb * 64, w.k_row + it * kTile, w.h_kv, 0);
          if (used) mbar_wait(&sh.v_empty[s], before, abort_flag, p.status, DEV_TIMEOUT_SYNC);
          mbar_expect_tx(&sh.v_full[s], kTileBytes);
          for (int nb = 0; nb < NB; ++nb)
            tma_load_4d(sV + s * kTileBytes + nb * 16384, &p.map_v, &sh.v_full[s], nb * 64, w.k_row + it * kTile, w.h_kv, 0);
        }
      }
      __syncwarp();
      n += w.tiles;
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer
    reg_dealloc<kRegsControl>();
    const uint32_t idesc_s = make_idesc(BF16, 128, 128, false, false), idesc_o = make_idesc(BF16, 128, DPAD, false, true);
    const uint64_t kmajor = make_sdesc_base(16, 1024), mnmajor = make_sdesc_base(16384, 1024);
    const uint32_t k_hi = static_cast<uint32_t>(kmajor >> 32), mn_hi = static_cast<uint32_t>(mnmajor >> 32);
    const uint32_t q_lo = static_cast<uint32_t>(kmajor) | ((smem_u32(sQ) >> 4) & 0x3fffu);
    const uint32_t kt_lo = static_cast<uint32_t>(kmajor) | ((smem_u32(sK) >> 4) & 0x3fffu);
    const uint32_t vt_lo = static_cast<uint32_t>(mnmajor) | ((smem_u32(sV) >> 4) & 0x3fffu);
    const uint32_t t_o = tmem + kColO;
    uint32_t had = 0, items = 0, n = 0;      // items of the mailbox, items with tiles before the current one, tiles before it
    auto next_item = [&]() {                 // the next one that has tiles
      Work w;
      do {
        w = next_work(had++);
      } while (w.tokens != 0 && w.tiles == 0);
      return w.tokens == 0 ? 0 : w.tiles;
    };
    // scores of tile m, the first of its item or not: what they wait for, and the products
    auto wait_s = [&](uint32_t m, bool first) {
      if (first) mbar_wait(&sh.q_full, (items + (m > 0)) & 1, abort_flag, p.status, DEV_TIMEOUT_TMA);
      mbar_wait(&sh.k_full[m % kSt], (m / kSt) & 1, abort_flag, p.status, DEV_TIMEOUT_TMA);
      if (kAhead && m > 0) {
        mbar_wait(&sh.s_free, (m - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
        tc_fence_after_sync();
      }
    };
    auto issue_s = [&](uint32_t m) {
      const uint32_t s = m % kSt;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DPAD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * 1024u + (kk & 3) * 2u;   // 16-byte units
          umma_ss_lohi(tmem, q_lo + off, k_hi, kt_lo + s * (kTileBytes >> 4) + off, k_hi, idesc_s, kk > 0);
        }
        umma_commit(&sh.s_full);
        umma_commit(&sh.k_empty[s]);
      }
    };
    int tiles = next_item();
    if (tiles > 0) {
      wait_s(0, true);
      issue_s(0);
    }
    while (tiles > 0) {
      int next = 0;
      for (int it = 0; it < tiles; ++it, ++n) {
        const bool last = it + 1 == tiles;
        const uint32_t s = n % kSt, v_lo = vt_lo + s * (kTileBytes >> 4);
        if (kAhead && !last) {
          wait_s(n + 1, false);
          issue_s(n + 1);
        }
        mbar_wait(&sh.v_full[s], (n / kSt) & 1, abort_flag, p.status, DEV_TIMEOUT_TMA);
        mbar_wait(&sh.p_half, n & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
        if (it == 0 && items > 0) mbar_wait(&sh.o_free, (items - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);      // O of the item before
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) umma_ts_lohi(t_o, tmem + kColP + kk * 8, v_lo + kk * 128u, mn_hi, idesc_o, it > 0 || kk > 0);
        }
        if (!kAhead && !last) wait_s(n + 1, false);
        mbar_wait(&sh.p_ready, n & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int kk = kTile / 32; kk < kTile / 16; ++kk) umma_ts_lohi(t_o, tmem + kColP + kk * 8, v_lo + kk * 128u, mn_hi, idesc_o, true);
          // (of the last tile V is free when O has left through its buffer, which the softmax warps say)
          if (kAhead || last) umma_commit(&sh.o_done);
          if (!last) umma_commit(&sh.v_empty[s]);
        }
        if (last) {      // (not before this item's last product: with items without tiles between, the next one may wait for its end)
          next = next_item();
          if (next > 0) wait_s(n + 1, true);
        }
        // the tensor pipe runs in order: where P lies over the scores it is consumed before they are written over it
        if (last ? next > 0 : !kAhead) issue_s(n + 1);
      }
      tiles = next;
      ++items;
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------------ scheduler: an item ahead of the others
    reg_dealloc<kRegsControl>();
    const int n_groups = p.N / p.tile_heads, per = p.tile_bound * p.head_group;
    const int64_t total = static_cast<int64_t>(p.tile_bound) * n_groups;
    uint32_t n = 0;
    bool more = true;
    for (int round = 0; more; ++round) {
      // Item numbers are dealt out there and back, as the heaviest come first; numbers past the last tile are nobody's.
      const int64_t number = static_cast<int64_t>(round) * gridDim.x + ((round & 1) == 0 ? blockIdx.x : gridDim.x - 1 - blockIdx.x);
      more = static_cast<int64_t>(round) * gridDim.x < total && *abort_flag == 0u;
      more = __any_sync(0xffffffffu, more);
      Work w = {};
      if (more) {
        if (number >= total) continue;
        const int hg = static_cast<int>(number / per), within = static_cast<int>(number % per);
        const int groups = min(p.head_group, n_groups - hg * p.head_group);
        const PackedItem x = finder.find(within / groups);
        const int token0 = x.tile * p.tile_tokens;
        w.tokens = min(p.tile_tokens, x.len_q - token0);
        if (w.tokens <= 0) continue;
        w.head0 = (hg * p.head_group + within % groups) * p.tile_heads;
        w.h_kv = w.head0 / p.kv_group;
        w.q_row = x.q0 + token0;
        w.k_row = x.k0;
        w.kv_len = x.len_k;
        w.tiles = (x.len_k + kTile - 1) / kTile;
        w.sees = x.len_k;
        if (causal) {
          w.sees = token0 + x.len_k - x.len_q + 1;
          const int last_key = w.sees + w.tokens - 2;
          w.tiles = last_key < 0 ? 0 : min(w.tiles, last_key / kTile + 1);
        }
      }
      if (n >= 2) mbar_wait(&sh.work_empty[n & 1], ((n >> 1) - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
      __syncwarp();
      if (elect_one()) {
        sh.work[n & 1] = w;
        mbar_arrive(&sh.work_full[n & 1]);
      }
      __syncwarp();
      ++n;
    }
  } else if (warp == 7) {
    // ------------------------------------------------------------------ stores of whole tiles
    reg_dealloc<kRegsControl>();
    uint32_t n = 0, whole = 0;      // K/V tiles, and whole tiles of O, so far
    for (uint32_t i = 0;; ++i) {
      const Work w = next_work(i);
      if (w.tokens == 0) break;
      n += w.tiles;
      if (w.tiles == 0 || w.tokens < p.tile_tokens) continue;
      mbar_wait(&sh.o_staged, whole++ & 1, abort_flag, p.status, DEV_TIMEOUT_SYNC);
      if (elect_one()) {
        const uint32_t s = (n - 1) % kSt;
        for (int nb = 0; nb < NB; ++nb)
          if (nb * 64 < p.D) tma_store_4d(&p.map_o, sV + s * kTileBytes + nb * 16384, nb * 64, w.head0, w.q_row, 0);
        tma_store_commit();
        tma_store_wait_read();
        mbar_arrive(&sh.v_empty[s]);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax
    reg_alloc<kRegsSoftmax>();
    const int token = tid / p.tile_heads, head = tid - token * p.tile_heads;      // of this thread's row
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t t_s = tmem + lanes, t_p = t_s + kColP, t_o = t_s + kColO;
    const float mult = p.scale_log2;
    const uint64_t mult2 = f2_pack(mult, mult);
    uint32_t n = 0, items = 0;      // tiles, and items that had any, so far

    for (uint32_t i = 0;; ++i) {
      // one warp takes the item for all four, so that they agree on it whatever happens
      if (warp == 0) {
        const Work mine = next_work(i);
        if (elect_one()) sh.softmax_work[i & 1] = mine;
      }
      named_barrier(1, 128);
      const Work& w = sh.softmax_work[i & 1];
      const int tiles = w.tiles, kv_len = w.kv_len, sees = w.sees;
      if (w.tokens == 0) break;
      // keys at or past `bound` do not exist for this row; `bound_tile` is the smallest bound of any row
      const int bound = causal ? min(kv_len, sees + token) : kv_len, bound_tile = min(kv_len, sees);

      float m_run = kNegInf, l_run = 0.f;
      for (int it = 0; it < tiles; ++it, ++n) {
        const int col_base = it * kTile;
        mbar_wait(&sh.s_full, n & 1, abort_flag, p.status, DEV_TIMEOUT_MMA);
        tc_fence_after_sync();
        // the whole score row in registers, one wait
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, s[c]);
        tmem_wait_ld();
        if constexpr (kAhead) {
          tc_fence_before_sync();
          mbar_arrive(&sh.s_free);
        }
        if (col_base + kTile > bound_tile) {      // positions that do not exist: a bit of a word decides, no compare per element
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int left = bound - col_base - c * 32;      // columns of the chunk that do
            const uint32_t gone = left >= 32 ? 0u : left <= 0 ? 0xffffffffu : 0xffffffffu << left;
#pragma unroll
            for (int j = 0; j < 32; ++j) s[c][j] = ((gone >> j) & 1u) != 0u ? __float_as_uint(kNegInf) : s[c][j];
          }
        }
        // one 32-column chunk: P = exp2(x * mult - m) packed to 16 bits, row sum into `l4`
        auto exp_chunk = [&](int c, uint64_t negm2, uint64_t (&l4)[4], uint32_t (&pk)[16]) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c][2 * j]), __uint_as_float(s[c][2 * j + 1])), mult2, negm2), x0, x1);
            const float p0 = ex2(x0), p1 = ex2(x1);
            l4[j & 3] = f2_add(l4[j & 3], f2_pack(p0, p1));
            pk[j] = pack2<BF16>(p0, p1);
          }
        };
        // from the second tile on the exponentials of chunk 0 start with the old maximum, and are done again if some row of the
        // warp needs a new one
        uint64_t l_part[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk0[16];
        const bool speculate = it > 0;
        if (speculate) {
          const float m_old = m_run == kNegInf ? 0.f : m_run;
          exp_chunk(0, f2_pack(-m_old, -m_old), l_part, pk0);
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][31]));
#pragma unroll
          for (int j = 1; j < 31; j += 2) mx[c] = fmax3(mx[c], __uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1]));
        }
        const float m_new = fmaxf(m_run, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mult);      // scale > 0
        const bool grow = (m_new > m_run + kRescaleThreshold) || (m_run == kNegInf && m_new != kNegInf);
        const bool any_grow = __any_sync(0xffffffffu, grow);
        float alpha = 1.0f;
        if (grow) {
          alpha = m_run == kNegInf ? 0.f : ex2(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
        }
        if constexpr (kAhead) {      // the tile before has left O, and its P is not needed any more
          if (it > 0) {
            mbar_wait(&sh.o_done, (n - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_MMA);
            tc_fence_after_sync();
          }
        }
        if (it > 0 && any_grow) {      // (otherwise O is complete because these scores were issued after the P V before)
#pragma unroll 1
          for (int c = 0; c < DPAD / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(t_o + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
            tmem_st32(t_o + c * 32, r);
          }
        }
        const float m_use = m_run == kNegInf ? 0.f : m_run;
        const uint64_t negm2 = f2_pack(-m_use, -m_use);
        if (!speculate || any_grow) {
#pragma unroll
          for (int j = 0; j < 4; ++j) l_part[j] = 0ull;
          exp_chunk(0, negm2, l_part, pk0);
        }
        // 16-bit P goes back; the first half is handed on as soon as it is stored
        tmem_st16(t_p, pk0);
        {
          uint32_t pk[16];
          exp_chunk(1, negm2, l_part, pk);
          tmem_st16(t_p + 16, pk);
          if (col_base + kTile > kv_len) {
            // Rows of V that are not this sequence's: 0 times what they hold might be a NaN.  (The last use of the buffer is over, as
            // the P V there has been waited for, here or before these scores were issued, and this tile's P V waits for this group: the
            // barrier can be in no other phase.)
            mbar_wait(&sh.v_full[n % kSt], (n / kSt) & 1, abort_flag, p.status, DEV_TIMEOUT_TMA);
            if (col_base + tid >= kv_len)
              for (int nb = 0; nb < NB; ++nb) {
                uint4* row = reinterpret_cast<uint4*>(sV + (n % kSt) * kTileBytes + nb * 16384 + tid * 128);
#pragma unroll
                for (int j = 0; j < 8; ++j) row[j] = make_uint4(0u, 0u, 0u, 0u);
              }
            fence_proxy_async_smem();
          }
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(&sh.p_half);
        }
        {
          uint32_t pk2[16], pk3[16], pk[32];
          exp_chunk(2, negm2, l_part, pk2);
          exp_chunk(3, negm2, l_part, pk3);
#pragma unroll
          for (int j = 0; j < 16; ++j) { pk[j] = pk2[j]; pk[16 + j] = pk3[j]; }
          tmem_st32(t_p + 32, pk);
        }
        float a0, a1;
        f2_unpack(f2_add(f2_add(l_part[0], l_part[1]), f2_add(l_part[2], l_part[3])), a0, a1);
        l_run += a0 + a1;
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&sh.p_ready);
      }

      // L = m + ln l straight to global memory, and O / l: of a whole tile through the V buffer and a TMA store, else by every thread
      // its row (the rows behind are the next sequence's)
      const int tokens = w.tokens, q_row = w.q_row, head0 = w.head0;
      const bool none = tiles == 0 || l_run == 0.f, there = token < tokens;      // a row that sees nothing: 0, also where V is not finite
      if (p.lse != nullptr && there)
        p.lse[static_cast<int64_t>(head0 + head) * p.T_q + q_row + token] = none ? kNegInf : m_run * kLn2 + logf(l_run);
      auto row_of_o = [&]() {
        int row = q_row + token, col = head0 + head;
        asm volatile("" : "+r"(row), "+r"(col));      // (nothing of the address is kept in registers over the tiles)
        return static_cast<uint16_t*>(p.o) + row * p.o_stride_s + col * p.o_stride_h;
      };
      if (tiles == 0) {      // no key at all: nothing has been loaded or multiplied
        uint16_t* out = row_of_o();
        for (int d = 0; there && d < p.D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      mbar_wait(&sh.o_done, (kAhead ? n - 1 : items) & 1, abort_flag, p.status, DEV_TIMEOUT_MMA);
      tc_fence_after_sync();
      ++items;
      const bool whole = tokens == p.tile_tokens;
      uint8_t* exit = sV + (n - 1) % kSt * kTileBytes;
      if (!whole && tid == 0) mbar_arrive(&sh.v_empty[(n - 1) % kSt]);
      const float inv_l = l_run > 0.f ? 1.0f / l_run : 0.f;
      const int n_chunks = (p.D + 31) / 32;
      // 32 columns of this thread's row, as 16-bit numbers
      auto row_chunk = [&](int c, uint4 (&u)[4]) {
        uint32_t r[32];
        tmem_ld32(t_o + c * 32, r);
        tmem_wait_ld();
        if (c + 1 == n_chunks) {      // O may be written over
          tc_fence_before_sync();
          mbar_arrive(&sh.o_free);
        }
        if (none) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0u;
        }
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) pk[j] = pack2<BF16>(__uint_as_float(r[2 * j]) * inv_l, __uint_as_float(r[2 * j + 1]) * inv_l);
#pragma unroll
        for (int g = 0; g < 4; ++g) u[g] = make_uint4(pk[4 * g], pk[4 * g + 1], pk[4 * g + 2], pk[4 * g + 3]);
      };
      if (whole) {
#pragma unroll 1
        for (int c = 0; c < n_chunks; ++c) {
          uint4 u[4];
          row_chunk(c, u);
#pragma unroll
          for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(exit + (c >> 1) * 16384u + swz128(tid, (c & 1) * 4 + g)) = u[g];
        }
        fence_proxy_async_smem();
        mbar_arrive(&sh.o_staged);
      } else {
        uint16_t* out = row_of_o();
#pragma unroll 1
        for (int c = 0; c < n_chunks; ++c) {
          uint4 u[4];
          row_chunk(c, u);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (there && c * 32 + g * 8 < p.D) *reinterpret_cast<uint4*>(out + c * 32 + g * 8) = u[g];
        }
      }
    }
    tc_fence_before_sync();
  }

  linger_after_abort(abort_flag);
  __syncthreads();
  if (warp == 4) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 256);
  }
}

}  // namespace

cudaError_t launch_fa_fwd_packed(const FwdParams& p, bool bf16, int sm_count, cudaStream_t stream) {
  const int dpad = p.D <= 64 ? 64 : 128;
  const size_t smem = static_cast<size_t>(dpad == 64 ? 5 : 6) * 16384 + 1024;      // Q and two K and V of 64 columns, or one of 128
  FwdParams pp = p;
  set_tile_tokens(pp, p.tile_tokens);
  // Heads that run at the same time share L2: as many as have their K and V in 48 MB of it.
  const int64_t fit = (48ll << 20) / (4ll * p.T_k * p.D + 1), per_kv = p.kv_group / p.tile_heads, groups = p.N / p.tile_heads;
  pp.head_group = static_cast<int>(fit < 1 ? per_kv : fit * per_kv < groups ? fit * per_kv : groups);
  void (*kern)(const FwdParams) = dpad == 64 ? (bf16 ? fa_fwd_packed_kernel<64, true> : fa_fwd_packed_kernel<64, false>)
                                             : (bf16 ? fa_fwd_packed_kernel<128, true> : fa_fwd_packed_kernel<128, false>);
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  const int64_t items = pp.tile_bound * groups;
  kern<<<static_cast<unsigned>(items < 2 * sm_count ? items : 2 * sm_count), kThreads, smem, stream>>>(pp);
  return cudaGetLastError();
}

}  // namespace acct
