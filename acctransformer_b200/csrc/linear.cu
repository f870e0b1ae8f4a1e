// Linear attention with a decay for each head, over whole sequences.
//
//   S_t = l S_(t-1) + b_t c_t^T,   y_t = scale S_t^T a_t,   l = exp(g)
//
// in chunks of 128 rows, r and i in a chunk of L rows, S the state before it:
//
//   P  = (A B^T) . l^(r - i) for i <= r     tensor cores, weighted in registers, back to tensor memory in 16 bits
//   y  = scale (P C + l^(r + 1) A S)        two products; their sum, weighted, in fp32
//   S' = l^L S + B^T (l^(L - 1 - i) C)      the product on tensor cores, the state itself in registers in fp32
//
// (reversed: i >= r, l^(i - r), l^(L - r), l^i, chunks from the last to the first).  A thread block has one head of a sequence and 64 columns
// of C: of two blocks per head at head_dim above 64 each loads A and B and forms P for itself; they run at the same time, so that
// the second load comes from L2, and P, half of the products at most, costs less than what the blocks would have to wait for each other.
//
// Roundings.  P and S are rounded once to the 16 bits that a product takes, like the probabilities of softmax attention; y is rounded
// once.  The weighted C goes into the state as a sum of 16-bit numbers, so the state keeps fp32: three for bfloat16 (24 bits), two for
// float16 (22), two for bfloat16 (16) where no state leaves the call and only 16-bit outputs follow from it.  float16 has no range to
// spare: the rows of P, the weighted C of a chunk and the state are scaled by powers of two that put their largest value near 2^15,
// and what follows is scaled back in fp32.
//
// What bounds it: 2 x 32 heads, 16 384 tokens of 128 take 240 us (164 at the copy rate) without and 275 us with states; a chunk of a block takes
// 3 000 to 3 400 clk, of which its products are 1 250 (head_dim up to 64) to 1 700, shared memory's traffic 2 600 and the loads 1 700.  Without any one of
// its parts it is 4 to 6 % faster, without all products 13 %: the rest are hand-offs between the warps.  (y straight to memory from the rows' threads,
// 845 wavefronts a chunk in the pipe that shared memory has too, instead of through the buffer of C: 281 us; twice the code, whose roles take each other's
// places in the instruction cache: 400 us with states.)
//
// Warps: 0-3 weight P (thread = row), 4-7 have the state (thread = row of S) and make y (thread = row), 8-11 split the weighted C, 12 loads,
// 13 issues products, 14 stores y.  The products of a chunk are issued as B^T C, A S, P C, the next chunk's A B^T (float16: these two the other way
// round): what each needs of the other warps is made while the ones before it run.
#include "fa_common.cuh"
#include "fa_kernels.cuh"
#include "linear.cuh"
#include "ptx.cuh"

namespace acct {
namespace {

constexpr int kThreads = 512;
constexpr int kRegsWork = 152, kRegsControl = 56;      // of 128 a thread at launch: 3 x 128 x 152 + 128 x 56 = 512 x 128
constexpr int kCols = 64;                              // columns of C, and of S, in a block
constexpr uint32_t kTileBytes = kLinChunk * 128;       // 128 rows of 64 16-bit values
// Tensor memory: P, twice 128 columns, of which P C takes the upper half once the scores there have been read; A S; B^T C, 64 columns for
// each number that stands for a weighted C.
constexpr uint32_t kColP = 0, kColIn = 64, kColOut = 256, kColState = 320;

struct Item {
  int b, h, c0, pass;
  int row0, rows;           // of the sequence
  int chunk0, chunks;       // of the segment
  int slot;                 // of the segment's state; -1: whole sequences
  int first, last;          // nothing is before, or behind, this segment in the order of the pass
};

struct LoadPlan {
  const CUtensorMap *a, *b, *c;
  int ha, hb, hc, row, step, batch, c0;
};

template <bool BF16>
struct Shared {
  uint64_t a_full[3], a_empty[3], b_full[3], b_empty[3], c_full[4], c_empty[4];
  uint64_t p_full[2], p_ready[2], split_ready, inc_done, inc_free, s_ready, s_read, o_done, o_free, y_staged[4];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
  Item item;
  float power[kLinChunk + 1];                                   // l^j
  float chunk_power[4];                                         // that of a whole chunk, and of one that is not, as sums of two numbers
  float p_back[BF16 ? 1 : 2][BF16 ? 1 : kLinChunk], c_back[4], s_back[4];      // float16: 1 / the scales of a chunk
  uint32_t most[2][2][4];
};

// mbar_wait in fewer instructions, of which this kernel has many copies in one instruction cache: a wait that runs out leaves its code in the
// block's abort flag, which ends all others, and the block records it before it retires.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, unsigned int code) {
  uint32_t polls = 0;
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (++polls >= kWaitPollLimit) *abort_flag = code;
    if (*abort_flag != 0u) break;
  }
}

// The power of two that brings `most` (>= 0) to [2^14, 2^15), and its inverse; 1 for 0 and what is not finite.
__device__ __forceinline__ void near_top(float most, float& scale, float& back) {
  const int e = static_cast<int>(__float_as_uint(most) >> 23);      // 127 + its exponent
  const bool usable = e > 0 && e < 255;
  const int up = usable ? min(max(141 - e, -126), 126) : 0;
  scale = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
  back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
}

template <bool BF16>
__device__ __forceinline__ uint64_t widen(uint32_t w) {      // two 16-bit values
  if constexpr (BF16) return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2_pack(f.x, f.y);
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow(uint64_t x) {
  float a, b;
  f2_unpack(x, a, b);
  return pack2<BF16>(a, b);
}

// The next 16-bit number of two values' sums, and what it leaves of them.  bfloat16: the leading 8 bits as they are, so that no conversion is
// needed and the rest has the same sign; the last number of a sum is rounded.
template <bool BF16, bool LAST>
__device__ __forceinline__ uint32_t next_part(uint64_t& v) {
  if constexpr (LAST) {
    return narrow<BF16>(v);
  } else if constexpr (BF16) {
    float a, b;
    f2_unpack(v, a, b);
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    v = f2_fma(f2_pack(__uint_as_float(ua & 0xffff0000u), __uint_as_float(ub & 0xffff0000u)), f2_pack(-1.f, -1.f), v);
    return __byte_perm(ua, ub, 0x7632);
  } else {
    const uint32_t w = narrow<BF16>(v);
    v = f2_fma(widen<BF16>(w), f2_pack(-1.f, -1.f), v);
    return w;
  }
}

// 32 bytes at a multiple of 32: a whole sector of L2
__device__ __forceinline__ void store32(void* to, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
               "r"(u[6]), "r"(u[7])
               : "memory");
}

// Blocks are numbered by columns of C, pass, head, and sequence or segment, fastest first: what reads the same rows runs at the same time.
__device__ __forceinline__ int slices_of(const LinParams& p) { return (p.D + kCols - 1) / kCols; }
__device__ __forceinline__ int pass_of_block(const LinParams& p) { return blockIdx.x / slices_of(p) % p.passes; }
__device__ __forceinline__ int head_of_block(const LinParams& p) { return blockIdx.x / (slices_of(p) * p.passes) % p.N; }

// What the block works on; by one warp.
__device__ __forceinline__ Item find_item(const LinParams& p) {
  const int lane = threadIdx.x & 31;
  Item x;
  x.c0 = blockIdx.x % slices_of(p) * kCols;
  x.pass = pass_of_block(p);
  x.h = head_of_block(p);
  const int at = blockIdx.x / (slices_of(p) * p.passes * p.N);
  x.chunks = 0; x.chunk0 = 0; x.slot = -1; x.first = x.last = 1;
  const bool reverse = p.pass[x.pass].reverse != 0;
  if (p.seg_chunks == 0) {
    x.b = at;
    if (p.cu != nullptr && p.B > 1 && p.B <= 64) {      // the at-th longest: a late start of a long one is what the SMs would wait for
      int n[2], rank[2] = {0, 0}, row;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        n[i] = -1;
        if (lane + 32 * i < p.B) lin_rows(p, lane + 32 * i, row, n[i]);
      }
#pragma unroll 1
      for (int j = 0; j < p.B; ++j) {
        const int other = __shfl_sync(0xffffffffu, n[j >> 5], j & 31);
#pragma unroll
        for (int i = 0; i < 2; ++i) rank[i] += other > n[i] || (other == n[i] && j < lane + 32 * i);
      }
      const unsigned int first = __ballot_sync(0xffffffffu, n[0] >= 0 && rank[0] == at), second = __ballot_sync(0xffffffffu, n[1] >= 0 && rank[1] == at);
      x.b = first != 0u ? __ffs(first) - 1 : 31 + __ffs(second);
    }
    lin_rows(p, x.b, x.row0, x.rows);
    x.chunks = (x.rows + kLinChunk - 1) / kLinChunk;
    return x;
  }
  x.slot = at;
  x.b = -1;
  x.row0 = x.rows = 0;
  int left = at;
#pragma unroll 1
  for (int b0 = 0; b0 < p.B && x.b < 0; b0 += 32) {      // the sequence that has the at-th segment
    int row = 0, n = 0;
    if (b0 + lane < p.B) lin_rows(p, b0 + lane, row, n);
    const int segs = (n + kLinChunk * p.seg_chunks - 1) / (kLinChunk * p.seg_chunks);
    int upto = segs;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += y;
    }
    const unsigned int past = __ballot_sync(0xffffffffu, upto > left);
    if (past != 0u) {
      const int from = __ffs(past) - 1;
      x.b = b0 + from;
      const int seg = left - __shfl_sync(0xffffffffu, upto - segs, from);
      x.row0 = __shfl_sync(0xffffffffu, row, from);
      x.rows = __shfl_sync(0xffffffffu, n, from);
      const int all = (x.rows + kLinChunk - 1) / kLinChunk;
      x.chunk0 = seg * p.seg_chunks;
      x.chunks = min(p.seg_chunks, all - x.chunk0);
      x.first = reverse ? x.chunk0 + x.chunks == all : seg == 0;
      x.last = reverse ? seg == 0 : x.chunk0 + x.chunks == all;
    } else {
      left -= __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  return x;
}

// STATES: only what each segment alone leaves behind.  SPLIT: 16-bit numbers that stand for a weighted value of C.
template <int DPAD, bool BF16, int SPLIT, bool STATES>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ LinParams p) {
  constexpr int NB = DPAD / 64;                    // 64-column blocks of A and B
  constexpr uint32_t kAB = NB * kTileBytes;
  // Buffers.  A chunk of C is needed from its split to P C, longer than its A and B.
  constexpr int kStAB = DPAD == 64 ? 3 : 2, kStC = DPAD == 64 ? 4 : SPLIT == 2 ? 3 : 2;
  constexpr bool kStaged = kStC > 2;               // whole chunks of y leave through the buffer of their C; with two it could not wait for that

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sB = sA + kStAB * kAB;
  uint8_t* sC = sB + kStAB * kAB;                  // (behind B: at head_dim up to 64 the product B^T C reads 128 columns of B, of which 64 are not)
  uint8_t* sSplit = sC + kStC * kTileBytes;
  uint8_t* sS = sSplit + SPLIT * kTileBytes;       // DPAD rows of 64 values
  __shared__ Shared<BF16> sh;

  const int tid = threadIdx.x;
  const int warp = static_cast<int>(warp_uniform(tid >> 5));
  volatile uint32_t* abort_flag = &sh.abort_flag;
  // The loads of the c-th chunk, one by one as buffers become free.  The first ones are under way before the block has set itself up.
  LoadPlan plan = {};
  auto load = [&](int c) {
    const int s = c % kStAB, sc = c % kStC, row = plan.row + c * plan.step;
    if constexpr (kStC > 2) {      // (in the order in which the buffers become free)
      if (c >= kStC) wait(&sh.c_empty[sc], (c / kStC - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
      mbar_expect_tx(&sh.c_full[sc], kTileBytes);
      tma_load_4d(sC + sc * kTileBytes, plan.c, &sh.c_full[sc], plan.c0, row, plan.hc, plan.batch);
    }
    if (c >= kStAB) wait(&sh.b_empty[s], (c / kStAB - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
    mbar_expect_tx(&sh.b_full[s], kAB);
    for (int nb = 0; nb < NB; ++nb) tma_load_4d(sB + s * kAB + nb * kTileBytes, plan.b, &sh.b_full[s], nb * 64, row, plan.hb, plan.batch);
    if constexpr (!STATES) {
      if (c >= kStAB) wait(&sh.a_empty[s], (c / kStAB - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
      mbar_expect_tx(&sh.a_full[s], kAB);
      for (int nb = 0; nb < NB; ++nb) tma_load_4d(sA + s * kAB + nb * kTileBytes, plan.a, &sh.a_full[s], nb * 64, row, plan.ha, plan.batch);
    }
    if constexpr (kStC == 2) {
      if (c >= kStC) wait(&sh.c_empty[sc], (c / kStC - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
      mbar_expect_tx(&sh.c_full[sc], kTileBytes);
      tma_load_4d(sC + sc * kTileBytes, plan.c, &sh.c_full[sc], plan.c0, row, plan.hc, plan.batch);
    }
  };
  const int h = head_of_block(p);
  if (warp == 12) {
    if (elect_one()) {
      const LinPass& pass = p.pass[pass_of_block(p)];
      prefetch_tmap(&pass.b.map);
      prefetch_tmap(&pass.c.map);
      if (!STATES) prefetch_tmap(&pass.a.map);
      for (int i = 0; i < kStAB; ++i) {
        mbar_init(&sh.a_full[i], 1); mbar_init(&sh.a_empty[i], 1);
        mbar_init(&sh.b_full[i], 1); mbar_init(&sh.b_empty[i], 1);
      }
      for (int i = 0; i < kStC; ++i) { mbar_init(&sh.c_full[i], 1); mbar_init(&sh.c_empty[i], 1); mbar_init(&sh.y_staged[i], 128); }
      for (int i = 0; i < 2; ++i) { mbar_init(&sh.p_full[i], 1); mbar_init(&sh.p_ready[i], 128); }
      mbar_init(&sh.split_ready, 128); mbar_init(&sh.inc_done, 1); mbar_init(&sh.inc_free, 128);
      mbar_init(&sh.s_ready, 128); mbar_init(&sh.s_read, 1);
      mbar_init(&sh.o_done, 1); mbar_init(&sh.o_free, 128);
      sh.abort_flag = 0;
      sh.s_back[0] = 1.f;
      mbar_fence_init();
    }
    __syncwarp();
    Item i = find_item(p);
    // what leaves no trace: a block past the last segment; with STATES the last segment of a sequence, which nothing comes behind
    if (i.b < 0 || (STATES && i.last)) { i.b = -1; i.chunks = 0; }
    const LinPass& pass = p.pass[i.pass];
    const bool reverse = pass.reverse != 0;
    plan.a = &pass.a.map; plan.b = &pass.b.map; plan.c = &pass.c.map;
    plan.ha = i.h / pass.a.group; plan.hb = i.h / pass.b.group; plan.hc = i.h / pass.c.group;
    plan.row = i.row0 + (i.chunk0 + (reverse ? i.chunks - 1 : 0)) * kLinChunk;
    plan.step = reverse ? -kLinChunk : kLinChunk;
    plan.batch = p.cu != nullptr ? 0 : i.b;
    plan.c0 = i.c0;
    if (elect_one()) {
      sh.item = i;
#pragma unroll 1
      for (int c = 0; c < min(i.chunks, kStAB < kStC ? kStAB : kStC); ++c) load(c);
    }
    __syncwarp();
    if ((tid & 31) < 2) {
      const LinPower w = lin_power(p.log_decay[h], (tid & 31) == 0 ? kLinChunk : i.rows % kLinChunk);
      sh.chunk_power[2 * (tid & 31)] = w.hi;
      sh.chunk_power[2 * (tid & 31) + 1] = w.lo;
      if ((tid & 31) == 0) sh.power[kLinChunk] = w.hi + w.lo;
    }
    __syncwarp();
  } else if (warp == 13) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  if (warp < 4) {
    const LinPower w = lin_power(p.log_decay[h], tid);
    sh.power[tid] = w.hi + w.lo;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = warp_uniform(sh.tmem_base);
  const Item x = sh.item;
  const LinPass& pass = p.pass[x.pass];
  const bool reverse = pass.reverse != 0;
  const bool idle = x.b < 0;
  const int n = x.chunks;
  const int batch = p.cu != nullptr ? 0 : x.b;
  // Nothing is before the first chunk, or nobody asks for what is behind the last one: the products that go with it are left out.
  const bool has_first = !x.first || p.state_in != nullptr;
  const bool has_last = STATES || (x.last && p.state_out != nullptr);
  const int s0 = has_first ? 0 : 1;                // the first chunk that has a state before it
  // the c-th chunk in the order of the pass: its first row, and how many
  auto first_row = [&](int c) { return (x.chunk0 + (reverse ? n - 1 - c : c)) * kLinChunk; };
  auto rows_of = [&](int c) { return min(kLinChunk, x.rows - first_row(c)); };
  void* const y = pass.y;
  const int64_t y_stride = pass.y_stride[2];
  const int64_t y_first = batch * pass.y_stride[0] + x.h * pass.y_stride[1] + (x.row0 + (tid & 127)) * y_stride + x.c0;
  const bool y_f32 = pass.y_f32 != 0, y_wide = pass.y_wide != 0;
  // y of chunk c; thread = row.  Whole chunks leave through the buffer of their C (kStaged), which P C was the last to read, others straight.
  auto write_y = [&](int c) {
    const int rows = rows_of(c), row = tid & 127;
    const uint32_t t_y = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint8_t* stage = sC + c % kStC * kTileBytes;
    float w = p.scale * sh.power[reverse ? max(rows - row, 0) : row + 1], in = p.scale;
    wait(&sh.o_done, c & 1, abort_flag, DEV_TIMEOUT_MMA);
    if (kStaged && c + 1 == n) wait(&sh.split_ready, c & 1, abort_flag, DEV_TIMEOUT_SYNC);      // (P C has not waited for it)
    tc_fence_after_sync();
    if constexpr (!BF16) {
      w *= sh.s_back[c & 3];
      in *= sh.p_back[c & 1][row];
    }
    const uint64_t w2 = f2_pack(w, w), in2 = f2_pack(in, in);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      uint32_t r[32], q[32];
      tmem_ld32(t_y + kColP + (c & 1) * 128 + kColIn + half * 32, r);
      tmem_ld32(t_y + kColOut + half * 32, q);
      tmem_wait_ld();
      if (half == 1) {
        tc_fence_before_sync();
        mbar_arrive(&sh.o_free);
      }
      uint64_t v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        v[j] = f2_fma(f2_pack(__uint_as_float(q[2 * j]), __uint_as_float(q[2 * j + 1])), w2,
                      f2_mul(f2_pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), in2));
      const int64_t at = y_first + static_cast<int64_t>(first_row(c)) * y_stride + half * 32;
      const int left = row < rows ? p.D - x.c0 - half * 32 : 0;      // values that exist
      if (y_f32) {
        float* out = static_cast<float*>(y) + at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t u[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a, b;
            f2_unpack(v[4 * j + e], a, b);
            u[2 * e] = __float_as_uint(a);
            u[2 * e + 1] = __float_as_uint(b);
          }
          if (8 * j < left) store32(out + 8 * j, u);
        }
      } else {
        uint16_t* out = static_cast<uint16_t*>(y) + at;
        uint32_t u[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) u[j] = narrow<BF16>(v[j]);
        if (kStaged && rows == kLinChunk) {
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stage + swz128(row, half * 4 + j)) = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
        } else if (!kStaged && y_wide && left >= 32) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x8[8] = {u[8 * j], u[8 * j + 1], u[8 * j + 2], u[8 * j + 3], u[8 * j + 4], u[8 * j + 5], u[8 * j + 6], u[8 * j + 7]};
            store32(out + 16 * j, x8);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (8 * j < left) *reinterpret_cast<uint4*>(out + 8 * j) = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
        }
      }
    }
    if constexpr (kStaged) {
      fence_proxy_async_smem();
      mbar_arrive(&sh.y_staged[c % kStC]);
    }
  };

  if (warp == 12) {
    // ------------------------------------------------------------------ loads
    reg_dealloc<kRegsControl>();
    if (elect_one())
#pragma unroll 1
      for (int c = kStAB < kStC ? kStAB : kStC; c < n; ++c) load(c);
    __syncwarp();
  } else if (warp == 13) {
    // ------------------------------------------------------------------ products
    reg_dealloc<kRegsControl>();
    const uint32_t idesc_p = make_idesc(BF16, 128, 128, false, false), idesc_in = make_idesc(BF16, 128, kCols, false, true);
    const uint32_t idesc_s = make_idesc(BF16, 128, SPLIT * kCols, true, true);
    const uint64_t kmajor = make_sdesc_base(16, 1024), mnmajor = make_sdesc_base(kTileBytes, 1024);
    const uint32_t k_hi = static_cast<uint32_t>(kmajor >> 32), mn_hi = static_cast<uint32_t>(mnmajor >> 32);
    auto at = [](uint64_t base, const uint8_t* t) { return static_cast<uint32_t>(base) | ((smem_u32(t) >> 4) & 0x3fffu); };
    const uint32_t a_lo = at(kmajor, sA), b_lo = at(kmajor, sB), bt_lo = at(mnmajor, sB), c_lo = at(mnmajor, sC);
    const uint32_t split_lo = at(mnmajor, sSplit), s_lo = at(mnmajor, sS);
    const int k_steps = (p.D + 15) / 16;
    // (each product stands here once: the roles share an instruction cache)
#pragma unroll 1
    for (int j = STATES ? 0 : -1; j <= n; ++j) {
      // B^T C of chunk j; of the last one behind what y needs, if at all
      const int inc = STATES ? j : j < n - 1 ? j : j == n && has_last ? n - 1 : -1;
      if (inc >= 0 && inc < n) {
        const int s = inc % kStAB;
        if constexpr (STATES) wait(&sh.b_full[s], (inc / kStAB) & 1, abort_flag, DEV_TIMEOUT_TMA);
        if (inc > 0) wait(&sh.inc_free, (inc - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
        wait(&sh.split_ready, inc & 1, abort_flag, DEV_TIMEOUT_SYNC);
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll 4
          for (int kk = 0; kk < kLinChunk / 16; ++kk)
            umma_ss_lohi(tmem + kColState, bt_lo + s * (kAB >> 4) + kk * 128u, mn_hi, split_lo + kk * 128u, mn_hi, idesc_s, kk > 0);
          umma_commit(&sh.inc_done);
          umma_commit(&sh.b_empty[s]);
          if constexpr (STATES) umma_commit(&sh.c_empty[inc % kStC]);
        }
        __syncwarp();
      }
      if constexpr (!STATES) {
        if (j >= 0 && j < n) {      // A S of chunk j
          const int s = j % kStAB;
          if (j >= s0) wait(&sh.s_ready, (j - s0) & 1, abort_flag, DEV_TIMEOUT_SYNC);
          if (j > 0) wait(&sh.o_free, (j - 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
          tc_fence_after_sync();
          if (elect_one()) {
            if (j >= s0) {
#pragma unroll 2
              for (int kk = 0; kk < k_steps; ++kk)
                umma_ss_lohi(tmem + kColOut, a_lo + s * (kAB >> 4) + (kk >> 2) * (kTileBytes >> 4) + (kk & 3) * 2u, k_hi, s_lo + kk * 128u, mn_hi, idesc_in, kk > 0);
              umma_commit(&sh.s_read);
            }
            umma_commit(&sh.a_empty[s]);
          }
          __syncwarp();
        }
        auto issue_p = [&]() {      // P of chunk j + 1 (what it goes over has been consumed, as products run in the order of their issue, and P C read)
          const int c = j + 1, s = c % kStAB;
          wait(&sh.a_full[s], (c / kStAB) & 1, abort_flag, DEV_TIMEOUT_TMA);
          wait(&sh.b_full[s], (c / kStAB) & 1, abort_flag, DEV_TIMEOUT_TMA);
          if (elect_one()) {
#pragma unroll 2
            for (int kk = 0; kk < k_steps; ++kk) {
              const uint32_t o = s * (kAB >> 4) + (kk >> 2) * (kTileBytes >> 4) + (kk & 3) * 2u;
              umma_ss_lohi(tmem + kColP + (c & 1) * 128, a_lo + o, k_hi, b_lo + o, k_hi, idesc_p, kk > 0);
            }
            umma_commit(&sh.p_full[c & 1]);
          }
          __syncwarp();
        };
        auto issue_pc = [&]() {     // P C of chunk j
          const int sc = j % kStC;
          const uint32_t t_p = tmem + kColP + (j & 1) * 128;
          if (j + 1 == n) {         // (its B^T C has not waited yet: for C, and for rows of C to be set to 0)
            wait(&sh.c_full[sc], (j / kStC) & 1, abort_flag, DEV_TIMEOUT_TMA);
            if (rows_of(j) < kLinChunk) wait(&sh.split_ready, j & 1, abort_flag, DEV_TIMEOUT_SYNC);
          }
          wait(&sh.p_ready[j & 1], (j >> 1) & 1, abort_flag, DEV_TIMEOUT_SYNC);
          tc_fence_after_sync();
          if (elect_one()) {
#pragma unroll 4
            for (int kk = 0; kk < kLinChunk / 16; ++kk)
              umma_ts_lohi(t_p + kColIn, t_p + kk * 8, c_lo + sc * (kTileBytes >> 4) + kk * 128u, mn_hi, idesc_in, kk > 0);
            umma_commit(&sh.o_done);
            if constexpr (!kStaged) umma_commit(&sh.c_empty[sc]);
          }
          __syncwarp();
        };
        // P C first, which frees C early; float16, whose P takes the warps that weight it twice as long, gives them the time of P's product
        // (2 x 32 heads, 8 192 tokens, with states: bfloat16 145 -> 137 us, float16 171 -> 146 us).
        if (BF16 && j >= 0 && j < n) issue_pc();
        if (j + 1 < n) issue_p();
        if (!BF16 && j >= 0 && j < n) issue_pc();
      }
    }
  } else if (warp == 14) {
    // ------------------------------------------------------------------ stores of whole chunks
    reg_dealloc<kRegsControl>();
    if constexpr (!STATES && kStaged) {
      for (int c = 0; c < n; ++c) {
        wait(&sh.y_staged[c % kStC], (c / kStC) & 1, abort_flag, DEV_TIMEOUT_SYNC);
        if (elect_one()) {
          if (rows_of(c) == kLinChunk && !y_f32) {
            tma_store_4d(&pass.map_y, sC + c % kStC * kTileBytes, x.c0, x.row0 + first_row(c), x.h, batch);
            tma_store_commit();
            tma_store_wait_read();
          }
          mbar_arrive(&sh.c_empty[c % kStC]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ weights of P
    reg_alloc<kRegsWork>();
    if constexpr (!STATES) {
      const int lane = tid & 31;
      const uint32_t t_p = tmem + kColP + (static_cast<uint32_t>(warp * 32) << 16);
      // A column block of 32 is 32 (warp - block) + lane - j before the row: on the diagonal its weights are the same for all warps;
      // elsewhere the power is one of the row and the block times one of the column, both <= 1.
      uint64_t diagonal[16], column[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float d[2], w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int apart = reverse ? 2 * j + u - lane : lane - 2 * j - u;
          d[u] = apart >= 0 ? sh.power[max(apart, 0)] : 0.f;
          w[u] = sh.power[reverse ? 2 * j + u : 31 - 2 * j - u];
        }
        diagonal[j] = f2_pack(d[0], d[1]);
        column[j] = f2_pack(w[0], w[1]);
      }
      for (int c = 0; c < n; ++c) {
        const int rows = rows_of(c);
        const uint32_t t = t_p + (c & 1) * 128;
        wait(&sh.p_full[c & 1], (c >> 1) & 1, abort_flag, DEV_TIMEOUT_MMA);
        tc_fence_after_sync();
        // one block of 32 columns, weighted
        auto weighted = [&](int block, uint64_t (&v)[16]) {
          uint32_t r[32];
          tmem_ld32(t + block * 32, r);
          tmem_wait_ld();
          if (block == warp) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = f2_mul(f2_pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), diagonal[j]);
          } else {
            const float w = sh.power[reverse ? 32 * (block - warp) - lane : 32 * (warp - block) + lane - 31];
            const uint64_t w2 = f2_pack(w, w);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = f2_mul(f2_mul(f2_pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), column[j]), w2);
          }
          const int left = rows - block * 32;
          if (left < 32) {      // columns behind the last row
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float a, b;
              f2_unpack(v[j], a, b);
              v[j] = f2_pack(2 * j < left ? a : 0.f, 2 * j + 1 < left ? b : 0.f);
            }
          }
        };
        // float16: the largest value of the row first
        float most = 0.f;
        uint64_t scale2 = 0;
#pragma unroll 1
        for (int round = BF16 ? 4 : 0; round < 8; ++round) {
          const int block = round & 3;
          if constexpr (!BF16) {
            if (round == 4) {
              float scale, back;
              near_top(most, scale, back);
              scale2 = f2_pack(scale, scale);
              sh.p_back[c & 1][tid] = back;
            }
          }
          uint64_t v[16];
          const bool seen = reverse ? block >= warp : block <= warp;
          if (seen) {
            weighted(block, v);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0ull;
          }
          if (!BF16 && round < 4) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float a, b;
              f2_unpack(v[j], a, b);
              most = fmax3(most, fabsf(a), fabsf(b));
            }
          } else {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) pk[j] = narrow<BF16>(BF16 ? v[j] : f2_mul(v[j], scale2));
            tmem_st16(t + block * 16, pk);      // (over scores that have been read, or that nobody needs)
          }
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&sh.p_ready[c & 1]);
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ warps 4-7: the state, and y; 8-11: weighted C
    reg_alloc<kRegsWork>();
    const int row = tid & 127, lane = tid & 31;      // of the state, or of C
    const bool keeps_state = warp < 8;
    const uint32_t t_s = tmem + kColState + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const LinPower step = {sh.chunk_power[0], sh.chunk_power[1]}, part = {sh.chunk_power[2], sh.chunk_power[3]};
    const int width = min(kCols, p.D - x.c0);      // columns that exist
    const int64_t one = (static_cast<int64_t>(x.b) * p.N + x.h) * p.D * p.D, mine = static_cast<int64_t>(row) * p.D + x.c0;
    const int64_t slot = ((static_cast<int64_t>(x.slot) * p.passes + x.pass) * p.N + x.h) * p.D * p.D;
    // (of a sequence in several segments the first one reads a copy, too: the last one's block may be done before this one begins, and what it
    // writes may be what the call was given)
    const bool whole = x.first && x.last;
    const float* from = STATES || idle || !has_first ? nullptr : whole ? p.state_in + one : p.seg_states + slot;
    float* to = idle ? nullptr : STATES ? p.seg_states + slot : has_last ? p.state_out + one : nullptr;
    uint64_t s[kCols / 2];
#pragma unroll
    for (int j = 0; j < kCols / 4; ++j) {
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (keeps_state && from != nullptr && row < p.D && 4 * j < width) f = *reinterpret_cast<const float4*>(from + mine + 4 * j);
      s[2 * j] = f2_pack(f.x, f.y);
      s[2 * j + 1] = f2_pack(f.z, f.w);
    }
    // The state before chunk c, to shared memory in 16 bits; from chunk 1 on it is made from the one before first.
    auto advance = [&](int c) {
      if (c > 0) {
        const int rows = rows_of(c - 1);
        const LinPower w = rows == kLinChunk ? step : part;
        const uint64_t hi2 = f2_pack(w.hi, w.hi), lo2 = f2_pack(w.lo, w.lo);
        wait(&sh.inc_done, (c - 1) & 1, abort_flag, DEV_TIMEOUT_MMA);
        tc_fence_after_sync();
        uint64_t back2 = 0;
        if constexpr (!BF16) back2 = f2_pack(sh.c_back[(c - 1) & 3], sh.c_back[(c - 1) & 3]);
#pragma unroll
        for (int part = 0; part < kCols / 16; ++part) {
          uint32_t r[SPLIT][16];
#pragma unroll
          for (int i = 0; i < SPLIT; ++i) tmem_ld16(t_s + i * kCols + part * 16, r[i]);
          tmem_wait_ld();
          if (part + 1 == kCols / 16) {
            tc_fence_before_sync();
            mbar_arrive(&sh.inc_free);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint64_t inc = f2_pack(__uint_as_float(r[SPLIT - 1][2 * j]), __uint_as_float(r[SPLIT - 1][2 * j + 1]));
#pragma unroll
            for (int i = SPLIT - 2; i >= 0; --i) inc = f2_add(inc, f2_pack(__uint_as_float(r[i][2 * j]), __uint_as_float(r[i][2 * j + 1])));
            if constexpr (!BF16) inc = f2_mul(inc, back2);
            uint64_t& v = s[part * 8 + j];
            v = f2_fma(v, hi2, f2_fma(v, lo2, inc));
          }
        }
      }
      if (STATES || c >= n) return;
      uint64_t scale2 = 0;
      if constexpr (!BF16) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) {
          float a, b;
          f2_unpack(s[j], a, b);
          most = fmax3(most, fabsf(a), fabsf(b));
        }
        const uint32_t of_warp = __reduce_max_sync(0xffffffffu, DPAD == 128 || warp < 6 ? __float_as_uint(most) : 0u);
        if (lane == 0) sh.most[0][c & 1][warp - 4] = of_warp;
        named_barrier(1, 128);
        const float of_all = __uint_as_float(max(max(sh.most[0][c & 1][0], sh.most[0][c & 1][1]), max(sh.most[0][c & 1][2], sh.most[0][c & 1][3])));
        float scale, back;
        near_top(of_all, scale, back);
        scale2 = f2_pack(scale, scale);
        if (row == 0) sh.s_back[c & 3] = back;
      }
      if (c > s0) wait(&sh.s_read, (c - 1 - s0) & 1, abort_flag, DEV_TIMEOUT_MMA);
      if (row < DPAD) {
#pragma unroll
        for (int j = 0; j < kCols / 8; ++j) {
          uint32_t pk[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) pk[u] = narrow<BF16>(BF16 ? s[4 * j + u] : f2_mul(s[4 * j + u], scale2));
          *reinterpret_cast<uint4*>(sS + swz128(row, j)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.s_ready);
    };
    // C of chunk c, weighted, as sums of 16-bit numbers
    auto split = [&](int c) {
      const int rows = rows_of(c);
      uint8_t *its_c = sC + c % kStC * kTileBytes, *its_b = sB + c % kStAB * kAB;
      const bool there = row < rows;
      float w = there ? sh.power[reverse ? row : rows - 1 - row] : 0.f;
      wait(&sh.c_full[c % kStC], (c / kStC) & 1, abort_flag, DEV_TIMEOUT_TMA);
      if (!there) {      // rows that are not this sequence's: 0 times what they hold might be a NaN
        wait(&sh.b_full[c % kStAB], (c / kStAB) & 1, abort_flag, DEV_TIMEOUT_TMA);
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          for (int nb = 0; nb < NB; ++nb) *reinterpret_cast<uint4*>(its_b + nb * kTileBytes + swz128(row, j)) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(its_c + swz128(row, j)) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      __syncwarp();
      if (c + 1 == n && !has_last) {      // into no state
        if (c > 0) wait(&sh.inc_done, (c - 1) & 1, abort_flag, DEV_TIMEOUT_MMA);      // (the barrier's phase before has been seen)
        fence_proxy_async_smem();
        mbar_arrive(&sh.split_ready);
        return;
      }
      if constexpr (!BF16) {
        uint32_t most = 0;      // of the absolute values, as 16-bit patterns, which have their order
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 raw = *reinterpret_cast<const uint4*>(its_c + swz128(row, j));
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu)));
        }
        // times this row's weight
        const float of_row = __half2float(__ushort_as_half(static_cast<unsigned short>(max(most >> 16, most & 0xffffu)))) * w;
        const uint32_t of_warp = __reduce_max_sync(0xffffffffu, __float_as_uint(of_row));
        if (lane == 0) sh.most[1][c & 1][warp - 8] = of_warp;
        named_barrier(2, 128);
        const float of_all = __uint_as_float(max(max(sh.most[1][c & 1][0], sh.most[1][c & 1][1]), max(sh.most[1][c & 1][2], sh.most[1][c & 1][3])));
        float scale, back;
        near_top(of_all, scale, back);
        w *= scale;
        if (row == 0) sh.c_back[c & 3] = back;
      }
      const uint64_t w2 = f2_pack(w, w);
      if (c > 0) wait(&sh.inc_done, (c - 1) & 1, abort_flag, DEV_TIMEOUT_MMA);
#pragma unroll 2
      for (int j = 0; j < 8; ++j) {
        const uint4 raw = *reinterpret_cast<const uint4*>(its_c + swz128(row, j));
        const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t out[3][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint64_t v = f2_mul(widen<BF16>(in[u]), w2);
          out[0][u] = next_part<BF16, false>(v);
          if constexpr (SPLIT == 3) out[1][u] = next_part<BF16, false>(v);
          out[SPLIT - 1][u] = next_part<BF16, true>(v);
        }
#pragma unroll
        for (int i = 0; i < SPLIT; ++i)
          *reinterpret_cast<uint4*>(sSplit + i * kTileBytes + swz128(row, j)) = make_uint4(out[i][0], out[i][1], out[i][2], out[i][3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.split_ready);
    };
    if (keeps_state && !has_first) {      // A S of the first chunk; these threads read it
      uint32_t zero[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) zero[j] = 0u;
      const uint32_t t_out = tmem + kColOut + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      tmem_st32(t_out, zero);
      tmem_st32(t_out + 32, zero);
      tmem_wait_st();
    }
    if (keeps_state) {
#pragma unroll 1
      for (int c = has_first && !STATES ? -1 : 0; c <= n; ++c) {      // (advance stands here once)
        if (!STATES && c > 0) write_y(c - 1);
        if (has_last ? c < n : c + 1 < n) advance(c + 1);
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < n; ++c) split(c);
    }
    if (keeps_state && to != nullptr && row < p.D) {
#pragma unroll
      for (int j = 0; j < kCols / 4; ++j) {
        float4 f;
        f2_unpack(s[2 * j], f.x, f.y);
        f2_unpack(s[2 * j + 1], f.z, f.w);
        if (4 * j < width) *reinterpret_cast<float4*>(to + mine + 4 * j) = f;
      }
    }
  } else {
    reg_dealloc<kRegsControl>();
  }

  tc_fence_before_sync();
  linger_after_abort(abort_flag);
  __syncthreads();
  if (tid == 0 && *abort_flag != 0u) atomicMax(p.status, *abort_flag);
  if (warp == 13) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// From what each segment alone leaves to the states before each of them, in its place; a thread has 4 neighbouring elements.  (And sequences
// without rows, which no block of the other kernel works on: their states stay as they are.)
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ LinParams p) {
  const int quads = p.D * p.D / 4, i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y % p.N, pass = blockIdx.y / p.N % p.passes, b = blockIdx.y / p.N / p.passes;
  int slot0 = 0, row0, rows;
  const int per = kLinChunk * p.seg_chunks;
  for (int j = threadIdx.x & 31; j < b; j += 32) {
    lin_rows(p, j, row0, rows);
    slot0 += (rows + per - 1) / per;
  }
  slot0 = __reduce_add_sync(0xffffffffu, slot0);
  if (i >= quads) return;
  lin_rows(p, b, row0, rows);
  const int segs = (rows + per - 1) / per;
  const int64_t one = (static_cast<int64_t>(b) * p.N + h) * quads + i, stride = static_cast<int64_t>(p.passes) * p.N * quads;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.state_in != nullptr) s = reinterpret_cast<const float4*>(p.state_in)[one];
  if (segs == 0 && p.state_out != nullptr) reinterpret_cast<float4*>(p.state_out)[one] = s;
  if (segs < 2 || slot0 + segs > p.seg_slots) return;      // (sequences that share rows make more segments than there are slots)
  const bool reverse = p.pass[pass].reverse != 0;
  const float g = p.log_decay[h];
  float4* slots = reinterpret_cast<float4*>(p.seg_states) + slot0 * stride + (static_cast<int64_t>(pass) * p.N + h) * quads + i;
  auto slot = [&](int at) { return slots + (reverse ? segs - 1 - at : at) * stride; };
  const LinPower whole = lin_power(g, per), first = reverse ? lin_power(g, rows - (segs - 1) * per) : whole;
  float4 add = *slot(0);
  if (p.state_in != nullptr) *slot(0) = s;             // (zeros otherwise, which nothing reads)
  for (int at = 0; at + 1 < segs; ++at) {
    const LinPower w = at == 0 ? first : whole;      // (of a segment that is not whole, the last one, reversed the first)
    float4 next = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at + 2 < segs) next = *slot(at + 1);         // (before its place is taken)
    s.x = fmaf(s.x, w.hi, fmaf(s.x, w.lo, add.x)); s.y = fmaf(s.y, w.hi, fmaf(s.y, w.lo, add.y));
    s.z = fmaf(s.z, w.hi, fmaf(s.z, w.lo, add.z)); s.w = fmaf(s.w, w.hi, fmaf(s.w, w.lo, add.w));
    *slot(at + 1) = s;
    add = next;
  }
}

// a thread: 4 neighbouring values
template <bool BF16>
__global__ void __launch_bounds__(256) linear_reduce_kernel(const LinReduce p) {
  const int quads = p.D / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, which = blockIdx.y;
  if (i >= static_cast<int64_t>(p.B) * p.N_kv * p.S * quads) return;
  const int d = static_cast<int>(i % quads) * 4, s = static_cast<int>(i / quads % p.S);
  const int h = static_cast<int>(i / quads / p.S % p.N_kv), b = static_cast<int>(i / quads / p.S / p.N_kv);
  if (p.lens != nullptr && s >= p.lens[b]) return;
  const float* from = (which ? p.parts[1] : p.parts[0]) + ((static_cast<int64_t>(b) * p.N_kv + h) * p.group * p.S + s) * p.D + d;
  float4 sum = *reinterpret_cast<const float4*>(from);
  for (int g = 1; g < p.group; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(g) * p.S * p.D);
    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
  }
  uint16_t* to = static_cast<uint16_t*>(which ? p.out[1] : p.out[0]) + b * p.out_stride[0] + h * p.out_stride[1] + s * p.out_stride[2] + d;
  *reinterpret_cast<uint2*>(to) = make_uint2(pack2<BF16>(sum.x, sum.y), pack2<BF16>(sum.z, sum.w));
}

template <int DPAD, bool BF16, int SPLIT, bool STATES>
cudaError_t launch(const LinParams& p, unsigned int blocks, cudaStream_t stream) {
  const size_t tiles = DPAD == 64 ? 3 * 2 + 4 : 2 * 4 + (SPLIT == 2 ? 3 : 2);      // (A, B and C as in the kernel)
  const size_t smem = (tiles + SPLIT) * kTileBytes + DPAD * 128 + 1024;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(linear_kernel<DPAD, BF16, SPLIT, STATES>), smem);
  if (e != cudaSuccess) return e;
  linear_kernel<DPAD, BF16, SPLIT, STATES><<<blocks, kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <int DPAD, bool BF16, int SPLIT>
cudaError_t launch_all(const LinParams& p, cudaStream_t stream) {
  const int slices = (p.D + kCols - 1) / kCols;
  const unsigned int per = static_cast<unsigned int>(p.passes) * slices * p.N;
  if (p.seg_chunks == 0) return launch<DPAD, BF16, SPLIT, false>(p, per * p.B, stream);
  cudaError_t e = launch<DPAD, BF16, SPLIT, true>(p, per * p.seg_slots, stream);
  if (e != cudaSuccess) return e;
  linear_join_kernel<<<dim3((p.D * p.D / 4 + 255) / 256, p.N * p.passes * p.B), 256, 0, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return launch<DPAD, BF16, SPLIT, false>(p, per * p.seg_slots, stream);
}

}  // namespace

// In halves of a chunk of the whole computation (0.8 to 1.1 us), for which a block has one SM to itself: a chunk of a segment's state alone takes one, and
// the two launches more, with what a block needs to begin and end, 20.  (Packed sequences count as equally long, since the host does not know
// them.)  Cut or whole, us: 1 x 8 heads of 128, 2 048 tokens 33 and 39, 8 192 tokens 54 and 109, 1 x 16, 4 096 tokens 53 and 69; whole: 2 x 16, 4 096 tokens 72
// (cut 80), 2 x 8, 2 048 tokens 39 (41), 1 x 1, 1 024 tokens 24 (25).
void linear_segments(LinParams& p, int sm_count) {
  const int64_t items = static_cast<int64_t>((p.D + kCols - 1) / kCols) * p.passes * p.N * p.B;
  const int64_t rows = p.cu != nullptr ? (p.S + p.B - 1) / p.B : p.S, chunks = (rows + kLinChunk - 1) / kLinChunk;
  auto waves = [&](int64_t blocks) { return (blocks + sm_count - 1) / sm_count; };
  int64_t best = 2 * waves(items) * chunks, segs = 1;
  for (int64_t n = 2; n <= chunks && items * (n - 1) < 2 * sm_count; ++n) {
    const int64_t per = (chunks + n - 1) / n, cost = 2 * waves(items * n) * per + waves(items * (n - 1)) * per + 20;
    if (cost < best) {
      best = cost;
      segs = n;
    }
  }
  p.seg_chunks = p.seg_slots = 0;
  if (segs == 1) return;
  const int64_t per = (chunks + segs - 1) / segs;
  p.seg_chunks = static_cast<int>(per);
  p.seg_slots = static_cast<int>(p.cu != nullptr ? p.S / (per * kLinChunk) + p.B : p.B * ((chunks + per - 1) / per));
}

cudaError_t launch_linear(const LinParams& p, bool bf16, cudaStream_t stream) {
  const bool exact = p.state_out != nullptr;
  if (p.D <= 64) return !bf16 ? launch_all<64, false, 2>(p, stream) : exact ? launch_all<64, true, 3>(p, stream) : launch_all<64, true, 2>(p, stream);
  return !bf16 ? launch_all<128, false, 2>(p, stream) : exact ? launch_all<128, true, 3>(p, stream) : launch_all<128, true, 2>(p, stream);
}

cudaError_t launch_linear_reduce(const LinReduce& p, bool bf16, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(p.B) * p.N_kv * p.S * (p.D / 4);
  const dim3 grid(static_cast<unsigned int>((threads + 255) / 256), 2);
  (bf16 ? linear_reduce_kernel<true> : linear_reduce_kernel<false>)<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace acct
