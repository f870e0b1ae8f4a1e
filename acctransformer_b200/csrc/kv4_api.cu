// C-ABI entry points of the cache in 4 bits: argument checks and launches.
#include <algorithm>

#include "common.cuh"
#include "fa_kernels.cuh"
#include "kv4_common.cuh"

namespace acct {
namespace {

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_cache(const char* name, const acct_kv4_cache* c, Kv4Cache* out) {
  if (c == nullptr) return fail(ACCT_ERR_NULL, "%s is NULL", name);
  if (c->dtype != ACCT_F16 && c->dtype != ACCT_BF16) return fail(ACCT_ERR_DTYPE, "%s: dtype must be ACCT_F16 or ACCT_BF16", name);
  if (c->B <= 0 || c->N_kv <= 0 || c->S_max <= 0) return fail(ACCT_ERR_SHAPE, "%s: B, N_kv, S_max must be positive", name);
  if (static_cast<int64_t>(c->B) * c->N_kv > 65535) return fail(ACCT_ERR_SHAPE, "%s: B*N_kv = %lld exceeds 65535", name, (long long)c->B * c->N_kv);
  if (c->D <= 0 || c->D % 8 != 0 || c->D > 32 * kKv4MaxGroups)
    return fail(ACCT_ERR_UNSUPPORTED_D, "%s: head_dim %d must be a multiple of 8 in (0, %d]", name, c->D, 32 * kKv4MaxGroups);
  if (c->records == nullptr) return fail(ACCT_ERR_NULL, "%s: records is NULL", name);
  if (misaligned(c->records)) return fail(ACCT_ERR_ALIGN, "%s: records must be 16-byte aligned", name);
  out->records = static_cast<uint8_t*>(c->records);
  out->table = c->block_table;
  out->B = c->B; out->N_kv = c->N_kv; out->D = c->D; out->S_max = c->S_max;
  out->recs = (c->S_max - 1) / kKv4Rows + 1;
  out->page_shift = 0;
  out->max_pages = out->num_pages = 0;
  if (c->block_table != nullptr) {
    if (c->page_size < kKv4Rows || (c->page_size & (c->page_size - 1)) != 0)
      return fail(ACCT_ERR_SHAPE, "%s: page_size = %d must be a power of two >= %d", name, c->page_size, kKv4Rows);
    if (c->num_pages <= 0) return fail(ACCT_ERR_SHAPE, "%s: num_pages must be positive", name);
    if (c->max_pages <= 0 || static_cast<int64_t>(c->max_pages) * c->page_size < c->S_max)
      return fail(ACCT_ERR_SHAPE, "%s: block_table with %d pages of %d rows cannot hold S_max = %d", name, c->max_pages, c->page_size, c->S_max);
    while ((kKv4Rows << out->page_shift) < c->page_size) ++out->page_shift;
    out->max_pages = c->max_pages;
    out->num_pages = c->num_pages;
  }
  return 0;
}

// bytes of a cache's records (of its whole pool, where it is paged)
size_t cache_bytes(const Kv4Cache& c) {
  const size_t recs = c.table != nullptr ? static_cast<size_t>(c.num_pages) << c.page_shift : static_cast<size_t>(c.B) * c.recs;
  return recs * c.N_kv * acct_kv4_record_bytes(c.D);
}

bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y ? y - x < a_bytes : x - y < b_bytes;
}

int check_rows(const acct_kv4_cache* c, const acct_kv4_rows* r, Kv4Rows* out) {
  if (r == nullptr) return fail(ACCT_ERR_NULL, "rows is NULL");
  if (r->T < 0) return fail(ACCT_ERR_SHAPE, "T must not be negative");
  if (!r->start || (r->T > 0 && (!r->k || !r->v))) return fail(ACCT_ERR_NULL, "k, v and start must be non-NULL");
  if (misaligned(r->k) || misaligned(r->v)) return fail(ACCT_ERR_ALIGN, "k and v must be 16-byte aligned");
  if (r->cu_seqlens == nullptr && r->T != c->B) return fail(ACCT_ERR_SHAPE, "without cu_seqlens there is one row per sequence: T = %d is not B = %d", r->T, c->B);
  for (int i = 0; i < 2; ++i) {
    const int64_t packed = i == 0 ? static_cast<int64_t>(c->N_kv) * c->D : c->D;
    out->k_stride[i] = packed_or(r->k_stride[i], packed);
    out->v_stride[i] = packed_or(r->v_stride[i], packed);
    if (out->k_stride[i] < c->D || out->v_stride[i] < c->D) return fail(ACCT_ERR_SHAPE, "row strides must not be smaller than head_dim");
    if (out->k_stride[i] % 8 != 0 || out->v_stride[i] % 8 != 0) return fail(ACCT_ERR_ALIGN, "row strides must be multiples of 8 elements");
  }
  out->k = r->k; out->v = r->v;
  out->cu = r->cu_seqlens; out->start = r->start; out->T = r->T;
  return 0;
}

int rows_call(const acct_kv4_cache* c, const acct_kv4_rows* r, bool append, void* stream) {
  Kv4Cache cache;
  Kv4Rows rows;
  int rc;
  if ((rc = check_cache("cache", c, &cache)) || (rc = check_rows(c, r, &rows))) return rc;
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  if (r->T == 0) return ACCT_OK;
  const cudaError_t e = (append ? launch_kv4_append : launch_kv4_read)(cache, rows, c->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, append ? "launching the cache write kernel" : "launching the cache read kernel");
  return ACCT_OK;
}

// scratch of one decode call: the parts' results, then (with weights) the scores
size_t parts_bytes(int B, int N, int D, int splits) {
  return (static_cast<size_t>(B) * N * splits * (static_cast<size_t>(D) + 2) * 4 + 15) / 16 * 16;
}
int padded_slots(int S_max) { return static_cast<int>((static_cast<int64_t>(S_max) + kKv4Rows - 1) / kKv4Rows * kKv4Rows); }
int padded_group(int N, int N_kv) { return (N / N_kv + 1) / 2 * 2; }
size_t scores_bytes(int B, int N, int N_kv, int S_max) { return static_cast<size_t>(B) * N_kv * padded_group(N, N_kv) * padded_slots(S_max) * 4; }

constexpr int kMaxSplits = 64;
// the most parts that a sequence is cut into where the library chooses: of 512 slots or more
int most_splits(int S_max) { return static_cast<int>(std::min<int64_t>(kMaxSplits, (static_cast<int64_t>(S_max) + 511) / 512)); }

}  // namespace
}  // namespace acct

using namespace acct;

extern "C" {

size_t acct_kv4_record_bytes(int32_t D) { return D > 0 && D % 8 == 0 && D <= 32 * kKv4MaxGroups ? static_cast<size_t>(640) * ((D + 31) / 32) : 0; }

int acct_kv4_append(const acct_kv4_cache* c, const acct_kv4_rows* r, void* stream) { return rows_call(c, r, true, stream); }

int acct_kv4_read(const acct_kv4_cache* c, const acct_kv4_rows* r, void* stream) { return rows_call(c, r, false, stream); }

size_t acct_kv4_decode_workspace_bytes(const acct_kv4_cache* c, int32_t N, int32_t num_splits, int32_t with_weights) {
  if (c == nullptr || c->B <= 0 || c->N_kv <= 0 || c->D <= 0 || c->S_max <= 0 || N < c->N_kv || num_splits > kMaxSplits) return 0;
  const int splits = num_splits > 0 ? num_splits : num_splits == 0 ? kMaxSplits : most_splits(c->S_max);
  return parts_bytes(c->B, N, c->D, splits) + (with_weights ? scores_bytes(c->B, N, c->N_kv, c->S_max) : 0);
}

int acct_kv4_decode(const acct_kv4_cache* c, const acct_kv4_decode_args* a, void* stream) {
  Kv4DecodeParams p;
  int rc = check_cache("cache", c, &p.cache);
  if (rc) return rc;
  if (a == nullptr) return fail(ACCT_ERR_NULL, "args is NULL");
  if (!a->q || !a->y) return fail(ACCT_ERR_NULL, "q and y must be non-NULL");
  if (misaligned(a->q) || misaligned(a->y)) return fail(ACCT_ERR_ALIGN, "q and y must be 16-byte aligned");
  if (a->N <= 0 || a->N % c->N_kv != 0) return fail(ACCT_ERR_SHAPE, "N = %d must be a multiple of N_kv = %d", a->N, c->N_kv);
  const int group = a->N / c->N_kv;
  if (group > 16) return fail(ACCT_ERR_SHAPE, "decode takes up to 16 query heads per cache head, got %d", group);
  if (!(a->scale > 0.f) || !(a->scale < 1e30f)) return fail(ACCT_ERR_SHAPE, "scale must be a positive finite number");
  if (a->num_splits < 0 || a->num_splits > kMaxSplits) return fail(ACCT_ERR_SHAPE, "num_splits must be in [0, %d]", kMaxSplits);
  const size_t scores = a->weights != nullptr ? scores_bytes(c->B, a->N, c->N_kv, c->S_max) : 0;
  const size_t given = a->workspace != nullptr ? a->workspace_bytes : 0;
  const size_t least = parts_bytes(c->B, a->N, c->D, a->num_splits > 0 ? a->num_splits : 1) + scores;
  if (given < least) return fail(ACCT_ERR_WORKSPACE, "decode workspace: need %zu bytes, got %zu", least, given);
  if (misaligned(a->workspace)) return fail(ACCT_ERR_ALIGN, "workspace must be 16-byte aligned");
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  const int64_t units = static_cast<int64_t>(c->B) * c->N_kv;
  p.B = c->B; p.N = a->N; p.D = c->D; p.kv_group = group;
  p.clustered = 0;
  int64_t splits = a->num_splits;
  p.parts = 0;
  if (splits == 0) {
    // Parts for one round of resident thread blocks (a sequence wastes half a part on average), or for two where a part of one round
    // has 160 steps (5 120 keys) or more of the slots.  One round and two, us, by steps: groups of 4 heads 80 34.9 / 37.5, 120 43.6 /
    // 47.1, 161 53.3 / 55.3, 174 60.4 / 60.8, 210 59.0 / 53.3, 261 82.9 / 81.1, 321 107.8 / 93.0, 420 101.5 / 99.0.  Groups of 16,
    // whose rounds are of fewer blocks, scatter with how the parts divide the lengths: 141 65.7 / 53.2, 186 59.4 / 65.1, 248 98.3 /
    // 73.8, 282 81.1 / 84.1, 390 100.4 / 82.2, 496 120.5 / 144.8, 780 176.2 / 144.8.
    const int64_t slots = static_cast<int64_t>(info.sm_count) * kv4_decode_blocks_per_sm(group);
    const int64_t steps = static_cast<int64_t>(c->B) * ((static_cast<int64_t>(c->S_max) + 31) / 32);
    auto parts = [&](int64_t rounds) { return std::max<int64_t>(1, slots * rounds / c->N_kv - c->B / 2); };
    const int64_t rounds = (units + slots - 1) / slots;
    p.parts = static_cast<int>(parts(steps >= 160 * parts(rounds) ? 2 * rounds : rounds));
    splits = most_splits(c->S_max);
    while (splits > 1 && parts_bytes(c->B, a->N, c->D, static_cast<int>(splits)) + scores > given) --splits;
    // Short contexts of few slices: the parts of a slice are one cluster and finish without a second kernel.  All clusters have to
    // be resident at once (16 x 8 slices of 1 024 keys in 2 parts, 128 of 222 that fit: 12.5 us against 17.7 of two kernels, in 4,
    // of 104 that fit: 18.5), and no part may be long, since the longest sequence decides (a group of 4 heads, 8 192 keys in 8
    // parts, 32 slices 18.8 -> 16.7 us, 8 slices 14.7 -> 14.7; 32 768 keys 22.7 -> 33.0; of 12 heads, 4 096 keys 16.6 -> 14.5, 8 192
    // 18.8 -> 20.8) or shorter than 128 keys.  One part is no cluster and need not be resident: 64 x 8 slices of 512 keys 18.8 -> 15.7.
    const int longest = group > 8 ? 512 : 1024;
    for (int parts : {8, 4, 2, 1}) {
      if (parts > 1 && parts * 128ll > c->S_max + 127ll) continue;
      if (static_cast<int64_t>(parts) * longest < c->S_max) break;
      Kv4DecodeParams q = p;
      q.clustered = 1;
      q.splits = parts;
      q.parts = 0;
      int resident = 0;
      if (parts > 1 && launch_kv4_decode(q, c->dtype == ACCT_BF16, nullptr, &resident) != cudaSuccess) {
        cudaGetLastError();      // a device that will not say gets no clusters
        resident = 0;
      }
      if (parts > 1 && units > resident) continue;
      p = q;
      splits = parts;
      break;
    }
  }
  p.q = a->q; p.y = a->y; p.seq_lens = a->seq_lens; p.weights = a->weights;
  p.B = c->B; p.N = a->N; p.D = c->D; p.kv_group = group;
  p.splits = static_cast<int>(splits);
  p.S_pad = padded_slots(c->S_max);
  p.G_pad = padded_group(a->N, c->N_kv);
  p.part_acc = static_cast<float*>(a->workspace);
  p.part_ml = p.part_acc + static_cast<size_t>(c->B) * a->N * p.splits * c->D;
  p.scores = a->weights == nullptr ? nullptr
             : p.clustered         ? p.part_acc      // (no results of parts then)
                                   : reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + parts_bytes(c->B, a->N, c->D, p.splits));
  p.status = device_status_ptr();
  p.scale_log2 = a->scale * kLog2e;
  const cudaError_t e = launch_kv4_decode(p, c->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the 4-bit decode kernels");
  return ACCT_OK;
}

int acct_kv4_evict(const acct_kv4_cache* src, const acct_kv4_cache* dst, const acct_kv4_evict_args* a, void* stream) {
  Kv4EvictParams p;
  int rc;
  if ((rc = check_cache("src", src, &p.src)) || (rc = check_cache("dst", dst, &p.dst))) return rc;
  if (a == nullptr) return fail(ACCT_ERR_NULL, "args is NULL");
  if (src->dtype != dst->dtype) return fail(ACCT_ERR_DTYPE, "src and dst must have one dtype");
  if (src->B != dst->B || src->N_kv != dst->N_kv || src->D != dst->D) return fail(ACCT_ERR_SHAPE, "src and dst must agree on B, N_kv and D");
  if (!a->weights || !a->weights_out || !a->kept || !a->seq_lens || !a->seq_lens_out)
    return fail(ACCT_ERR_NULL, "weights, weights_out, kept, seq_lens and seq_lens_out must be non-NULL");
  if (a->keep < 1 || a->recent < 0 || a->recent > a->keep) return fail(ACCT_ERR_SHAPE, "need 0 <= recent <= keep and keep >= 1, got recent = %d, keep = %d", a->recent, a->keep);
  if (a->keep > dst->S_max) return fail(ACCT_ERR_SHAPE, "keep = %d does not fit dst with S_max = %d", a->keep, dst->S_max);
  // The copy of one record reads where others are written, so nothing may be in both.  Of two tables over one pool only the caller
  // knows that they share no page.
  const size_t lens = static_cast<size_t>(src->B) * sizeof(int32_t), heads = static_cast<size_t>(src->B) * src->N_kv * sizeof(float);
  if (overlap(a->weights, heads * src->S_max, a->weights_out, heads * dst->S_max)) return fail(ACCT_ERR_SHAPE, "eviction does not work in place: weights and weights_out overlap");
  if (overlap(a->seq_lens, lens, a->seq_lens_out, lens)) return fail(ACCT_ERR_SHAPE, "eviction does not work in place: seq_lens and seq_lens_out overlap");
  const bool one_pool = src->block_table != nullptr && dst->block_table != nullptr && src->records == dst->records && src->block_table != dst->block_table;
  if (!one_pool && overlap(src->records, cache_bytes(p.src), dst->records, cache_bytes(p.dst)))
    return fail(ACCT_ERR_SHAPE, "eviction does not work in place: dst must be other memory than src, or other pages of its pool");
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  p.weights = a->weights; p.weights_out = a->weights_out; p.kept = a->kept;
  p.seq_lens = a->seq_lens; p.seq_lens_out = a->seq_lens_out;
  p.keep = a->keep; p.recent = a->recent;
  const cudaError_t e = launch_kv4_evict(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the eviction kernels");
  return ACCT_OK;
}

}  // extern "C"
