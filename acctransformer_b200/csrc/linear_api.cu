// C-ABI entry points of linear attention and of rotary positions: argument checks and launches.
#include <algorithm>

#include "common.cuh"
#include "fa_kernels.cuh"
#include "linear.cuh"

namespace acct {
namespace {

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_width(int D) {
  if (D <= 0 || D % 8 != 0 || D > kLinMaxHeadDim) return fail(ACCT_ERR_UNSUPPORTED_D, "head_dim %d must be a multiple of 8 in (0, %d]", D, kLinMaxHeadDim);
  return 0;
}

// Strides of batch entry, head and row; 0 = packed: [rows, heads, D] where sequences are packed, else [B, heads, rows, D].
int strides_of(const char* name, const int64_t (&given)[3], const acct_linear_args* a, int heads, int64_t (&out)[3]) {
  const int64_t D = a->D, S = a->S;
  const bool packed = a->cu_seqlens != nullptr;
  const int64_t dense[3] = {D * S * heads, packed ? D : D * S, packed ? D * heads : D};
  for (int i = 0; i < 3; ++i) {
    out[i] = packed_or(given[i], std::max(dense[i], D));      // (no rows: nothing is read)
    if (out[i] < D) return fail(ACCT_ERR_SHAPE, "%s strides must not be smaller than head_dim", name);
    if (out[i] % 8 != 0) return fail(ACCT_ERR_ALIGN, "%s stride (%lld elements) is not a multiple of 8", name, (long long)out[i]);
  }
  return 0;
}

// One [B, heads, S, D] operand, for the tensor maps and for plain addresses.
struct Rows {
  const char* name;
  const void* ptr;
  int heads;
  int64_t stride[3];
  CUtensorMap map;
};

int check_linear(const acct_linear_args* a, LinParams* p, Rows* q, Rows* k, Rows* v) {
  if (a == nullptr) return fail(ACCT_ERR_NULL, "args is NULL");
  if (a->dtype != ACCT_F16 && a->dtype != ACCT_BF16) return fail(ACCT_ERR_DTYPE, "dtype must be ACCT_F16 or ACCT_BF16");
  if (a->B <= 0 || a->N <= 0) return fail(ACCT_ERR_SHAPE, "B, N must be positive");
  if (a->S < 0 || (a->S == 0 && a->cu_seqlens == nullptr)) return fail(ACCT_ERR_SHAPE, "S must be positive (0 only for packed sequences)");
  if (a->N_kv < 0 || (a->N_kv > 0 && a->N % a->N_kv != 0)) return fail(ACCT_ERR_SHAPE, "N_kv = %d must be 0 or a divisor of N = %d", a->N_kv, a->N);
  if (static_cast<int64_t>(a->B) * a->N > (1 << 24)) return fail(ACCT_ERR_SHAPE, "B*N = %lld is too large", (long long)a->B * a->N);
  int rc = check_width(a->D);
  if (rc) return rc;
  if (!a->log_decay) return fail(ACCT_ERR_NULL, "log_decay is NULL");
  if (a->cu_seqlens != nullptr && a->seq_lens != nullptr) return fail(ACCT_ERR_SHAPE, "seq_lens does not go with packed sequences");
  if (a->S > 0 && (!a->q || !a->k || !a->v)) return fail(ACCT_ERR_NULL, "q, k, v must be non-NULL");
  if (misaligned(a->q) || misaligned(a->k) || misaligned(a->v)) return fail(ACCT_ERR_ALIGN, "q, k, v must be 16-byte aligned");
  if (!(a->scale > -1e30f) || !(a->scale < 1e30f)) return fail(ACCT_ERR_SHAPE, "scale must be a finite number");
  const int n_kv = a->N_kv > 0 ? a->N_kv : a->N;
  *q = {"q", a->q, a->N, {0, 0, 0}, {}};
  *k = {"k", a->k, n_kv, {0, 0, 0}, {}};
  *v = {"v", a->v, n_kv, {0, 0, 0}, {}};
  if ((rc = strides_of("q", a->q_stride, a, a->N, q->stride)) || (rc = strides_of("k", a->k_stride, a, n_kv, k->stride)) ||
      (rc = strides_of("v", a->v_stride, a, n_kv, v->stride)))
    return rc;
  memset(p, 0, sizeof(*p));
  p->B = a->B; p->N = a->N; p->S = a->S; p->D = a->D;
  p->log_decay = a->log_decay;
  p->cu = a->cu_seqlens;
  p->lens = a->seq_lens;
  p->scale = a->scale;
  return 0;
}

int make_map(const acct_linear_args* a, Rows& x, CUtensorMap* map = nullptr) {
  TensorDesc4 t;
  t.ptr = x.ptr;
  t.dtype = a->dtype;
  t.dims[0] = a->D; t.dims[1] = a->S; t.dims[2] = x.heads; t.dims[3] = a->cu_seqlens != nullptr ? 1 : a->B;
  t.strides[0] = x.stride[2]; t.strides[1] = x.stride[1]; t.strides[2] = x.stride[0];
  return make_tmap_4d(map != nullptr ? map : &x.map, t, kLinChunk);
}

void set_pass(const acct_linear_args* a, const Rows& x, const Rows& y, const Rows& z, LinPass* pass) {
  const Rows* from[3] = {&x, &y, &z};
  LinOperand* to[3] = {&pass->a, &pass->b, &pass->c};
  for (int i = 0; i < 3; ++i) {
    to[i]->group = a->N / from[i]->heads;
    to[i]->map = from[i]->map;
  }
}
int make_output(const acct_linear_args* a, Rows& y, LinPass* pass) {
  pass->y = const_cast<void*>(y.ptr);
  pass->y_wide = (reinterpret_cast<uintptr_t>(y.ptr) & 31u) == 0;
  for (int i = 0; i < 3; ++i) {
    pass->y_stride[i] = y.stride[i];
    pass->y_wide = pass->y_wide && y.stride[i] % 16 == 0;
  }
  return make_map(a, y, &pass->map_y);
}

// fp32 parts of dk and dv by query head, where heads share their keys and values
size_t partial_bytes(const acct_linear_args* a) {
  return a->N_kv > 0 && a->N_kv != a->N ? static_cast<size_t>(2) * a->B * a->N * a->S * a->D * 4 : 0;
}

// Bytes of the segments' states of a call, and (in `p`, unless it is null) how its sequences are cut.  (By the arguments alone: what a
// workspace was sized for is what a call does.)
constexpr int kSms = 148;
size_t segments_of(const acct_linear_args* a, int passes, LinParams* p) {
  if (a == nullptr || a->B <= 0 || a->N <= 0 || a->S <= 0 || a->D <= 0) return 0;
  LinParams own;
  if (p == nullptr) p = &own;
  p->B = a->B; p->N = a->N; p->S = a->S; p->D = a->D;
  p->cu = a->cu_seqlens;
  p->passes = passes;
  linear_segments(*p, kSms);
  return (linear_segment_bytes(*p) + 31) / 32 * 32;
}

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (need > 0 && (workspace == nullptr || bytes < need)) return fail(ACCT_ERR_WORKSPACE, "workspace of %zu bytes is too small: %zu are needed", bytes, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 31u) != 0) return fail(ACCT_ERR_ALIGN, "workspace must be 32-byte aligned");
  return 0;
}

// no rows at all: the states stay as they are
int copy_states(const acct_linear_args* a, void* stream) {
  if (a->state_out == nullptr || a->state_out == a->state_in) return ACCT_OK;
  const size_t bytes = static_cast<size_t>(a->B) * a->N * a->D * a->D * 4;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->state_in != nullptr ? cudaMemcpyAsync(a->state_out, a->state_in, bytes, cudaMemcpyDeviceToDevice, s)
                                               : cudaMemsetAsync(a->state_out, 0, bytes, s);
  return e == cudaSuccess ? ACCT_OK : fail_cuda(e, "copying the states");
}

// positions of 32 or of 64 bits
int rotary(const acct_rotary_args* a, const int32_t* positions, const int64_t* wide, void* stream) {
  if (a == nullptr) return fail(ACCT_ERR_NULL, "args is NULL");
  if (a->dtype != ACCT_F16 && a->dtype != ACCT_BF16) return fail(ACCT_ERR_DTYPE, "dtype must be ACCT_F16 or ACCT_BF16");
  if (a->B < 0 || a->S < 0 || a->N < 0 || a->N_kv < 0) return fail(ACCT_ERR_SHAPE, "sizes must not be negative");
  if (a->D <= 0 || a->D % 8 != 0 || a->D > 256) return fail(ACCT_ERR_UNSUPPORTED_D, "head_dim %d must be a multiple of 8 in (0, 256]", a->D);
  if (a->rotated <= 0 || a->rotated % 2 != 0 || a->rotated > a->D) return fail(ACCT_ERR_SHAPE, "rotated = %d must be even, in (0, head_dim = %d]", a->rotated, a->D);
  if ((!positions && !wide) || !a->turns || !a->axis) return fail(ACCT_ERR_NULL, "positions, turns, axis must be non-NULL");
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  const int64_t rows = static_cast<int64_t>(a->B) * a->S;
  const struct { const char* name; const void* x; void* y; const int64_t *xs, *ys; int heads; } t[2] = {
      {"q", a->q, a->q_out, a->q_stride, a->q_out_stride, a->N}, {"k", a->k, a->k_out, a->k_stride, a->k_out_stride, a->N_kv}};
  for (int w = 0; w < 2; ++w) {
    if (t[w].heads == 0 || rows == 0) continue;
    if (!t[w].x || !t[w].y) return fail(ACCT_ERR_NULL, "%s and its output must be non-NULL", t[w].name);
    if (misaligned(t[w].x) || misaligned(t[w].y)) return fail(ACCT_ERR_ALIGN, "%s and its output must be 16-byte aligned", t[w].name);
    const int64_t dense[3] = {static_cast<int64_t>(a->D) * a->S * t[w].heads, static_cast<int64_t>(a->D) * a->S, a->D};
    for (int i = 0; i < 3; ++i) {
      p.t[w].x_stride[i] = packed_or(t[w].xs[i], dense[i]);
      p.t[w].y_stride[i] = packed_or(t[w].ys[i], dense[i]);
      for (int64_t s : {p.t[w].x_stride[i], p.t[w].y_stride[i]}) {
        if (s < a->D) return fail(ACCT_ERR_SHAPE, "%s strides must not be smaller than head_dim", t[w].name);
        if (s % 8 != 0) return fail(ACCT_ERR_ALIGN, "%s stride (%lld elements) is not a multiple of 8", t[w].name, (long long)s);
      }
    }
    p.t[w].x = t[w].x; p.t[w].y = t[w].y;
    p.t[w].heads = t[w].heads;
  }
  if (rows > INT32_MAX || static_cast<double>(rows) * (static_cast<double>(a->N) + a->N_kv) * a->D >= 0x1p34)      // (a few launches at most)
    return fail(ACCT_ERR_SHAPE, "B*S = %lld rows are too many for one call", (long long)rows);
  p.positions = positions;
  p.wide_positions = reinterpret_cast<const long long*>(wide);
  for (int i = 0; i < 3; ++i) p.pos_stride[i] = a->pos_stride[i];
  p.turns = reinterpret_cast<const unsigned long long*>(a->turns);
  p.axis = a->axis;
  p.B = a->B; p.S = a->S; p.D = a->D; p.rotated = a->rotated;
  p.adjacent = a->adjacent; p.inverse = a->inverse;
  DeviceInfo info;
  int rc = device_info(&info);
  if (rc) return rc;
  if (rows == 0 || a->N + a->N_kv == 0) return ACCT_OK;
  const cudaError_t e = launch_rotary(p, a->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the rotary kernel");
  return ACCT_OK;
}

}  // namespace
}  // namespace acct

using namespace acct;

extern "C" {

size_t acct_linear_fwd_workspace_bytes(const acct_linear_args* a) { return segments_of(a, 1, nullptr); }

int acct_linear_fwd(const acct_linear_args* a, void* stream) {
  LinParams p;
  Rows q, k, v, y;
  int rc = check_linear(a, &p, &q, &k, &v);
  if (rc) return rc;
  if (a->S > 0 && !a->y) return fail(ACCT_ERR_NULL, "y must be non-NULL");
  if (misaligned(a->y) || misaligned(a->state_in) || misaligned(a->state_out)) return fail(ACCT_ERR_ALIGN, "y and the states must be 16-byte aligned");
  y = {"y", a->y, a->N, {0, 0, 0}, {}};
  if ((rc = strides_of("y", a->y_stride, a, a->N, y.stride))) return rc;
  if ((rc = check_workspace(segments_of(a, 1, &p), a->workspace, a->workspace_bytes))) return rc;
  p.seg_states = static_cast<float*>(a->workspace);
  p.state_in = a->state_in;
  p.state_out = a->state_out;
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  p.status = device_status_ptr();
  if (a->S == 0) return copy_states(a, stream);
  if ((rc = make_map(a, q)) || (rc = make_map(a, k)) || (rc = make_map(a, v)) || (rc = make_output(a, y, &p.pass[0]))) return rc;
  set_pass(a, q, k, v, &p.pass[0]);
  const cudaError_t e = launch_linear(p, a->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the linear attention kernel");
  return ACCT_OK;
}

size_t acct_linear_bwd_workspace_bytes(const acct_linear_args* a) {
  if (a == nullptr || a->B <= 0 || a->N <= 0 || a->S <= 0 || a->D <= 0) return 0;
  return segments_of(a, 3, nullptr) + partial_bytes(a);
}

int acct_linear_bwd(const acct_linear_args* a, const acct_linear_bwd_io* g, void* stream) {
  LinParams p;
  Rows q, k, v;
  int rc = check_linear(a, &p, &q, &k, &v);
  if (rc) return rc;
  if (a->cu_seqlens != nullptr) return fail(ACCT_ERR_SHAPE, "packed sequences have no backward");
  if (a->state_in != nullptr || a->state_out != nullptr) return fail(ACCT_ERR_SHAPE, "states have no backward");
  if (g == nullptr || !g->d_y || !g->dq || !g->dk || !g->dv) return fail(ACCT_ERR_NULL, "d_y, dq, dk, dv must be non-NULL");
  if (misaligned(g->d_y) || misaligned(g->dq) || misaligned(g->dk) || misaligned(g->dv)) return fail(ACCT_ERR_ALIGN, "d_y, dq, dk, dv must be 16-byte aligned");
  const size_t segment_bytes = segments_of(a, 3, &p);
  if ((rc = check_workspace(segment_bytes + partial_bytes(a), g->workspace, g->workspace_bytes))) return rc;
  p.seg_states = static_cast<float*>(g->workspace);
  const int64_t zero[3] = {0, 0, 0};
  Rows d = {"d_y", g->d_y, a->N, {0, 0, 0}, {}}, dq = {"dq", g->dq, a->N, {0, 0, 0}, {}};
  Rows dk = {"dk", g->dk, k.heads, {0, 0, 0}, {}}, dv = {"dv", g->dv, k.heads, {0, 0, 0}, {}};
  if ((rc = strides_of("d_y", g->d_y_stride, a, a->N, d.stride)) || (rc = strides_of("dq", zero, a, a->N, dq.stride)) ||
      (rc = strides_of("dk", zero, a, k.heads, dk.stride)))
    return rc;
  std::copy(dk.stride, dk.stride + 3, dv.stride);
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  p.status = device_status_ptr();
  if ((rc = make_map(a, q)) || (rc = make_map(a, k)) || (rc = make_map(a, v)) || (rc = make_map(a, d)) || (rc = make_output(a, dq, &p.pass[0])) || (rc = make_output(a, dk, &p.pass[1])) || (rc = make_output(a, dv, &p.pass[2])))
    return rc;
  set_pass(a, d, v, k, &p.pass[0]);
  set_pass(a, v, d, q, &p.pass[1]);
  set_pass(a, k, q, d, &p.pass[2]);
  p.pass[1].reverse = p.pass[2].reverse = 1;
  const int group = a->N / k.heads;
  LinReduce r;
  memset(&r, 0, sizeof(r));
  if (group > 1) {      // every query head's part in fp32, then their sums
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(g->workspace) + segment_bytes);
    for (int i = 0; i < 2; ++i) {
      LinPass& pass = p.pass[1 + i];
      pass.y = parts + i * (partial_bytes(a) / 8);      // (rows of a multiple of 8 fp32 values)
      pass.y_f32 = 1;
      std::copy(dq.stride, dq.stride + 3, pass.y_stride);
      r.parts[i] = static_cast<const float*>(pass.y);
    }
    std::copy(dk.stride, dk.stride + 3, r.out_stride);
    r.out[0] = g->dk; r.out[1] = g->dv;
    r.lens = a->seq_lens;
    r.B = a->B; r.N_kv = k.heads; r.group = group; r.S = a->S; r.D = a->D;
  }
  cudaError_t e = launch_linear(p, a->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess && group > 1) e = launch_linear_reduce(r, a->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the linear attention backward");
  return ACCT_OK;
}

int acct_linear_step(const acct_linear_step_args* a, void* stream) {
  if (a == nullptr) return fail(ACCT_ERR_NULL, "args is NULL");
  if (a->dtype != ACCT_F16 && a->dtype != ACCT_BF16) return fail(ACCT_ERR_DTYPE, "dtype must be ACCT_F16 or ACCT_BF16");
  if (a->B <= 0 || a->N <= 0) return fail(ACCT_ERR_SHAPE, "B, N must be positive");
  if (a->N_kv < 0 || (a->N_kv > 0 && a->N % a->N_kv != 0)) return fail(ACCT_ERR_SHAPE, "N_kv = %d must be 0 or a divisor of N = %d", a->N_kv, a->N);
  if (static_cast<int64_t>(a->B) * a->N > (1 << 24)) return fail(ACCT_ERR_SHAPE, "B*N = %lld is too large", (long long)a->B * a->N);
  int rc = check_width(a->D);
  if (rc) return rc;
  if (!a->q || !a->k || !a->v || !a->y || !a->state || !a->log_decay) return fail(ACCT_ERR_NULL, "q, k, v, y, state, log_decay must be non-NULL");
  if (misaligned(a->q) || misaligned(a->k) || misaligned(a->v) || misaligned(a->y) || misaligned(a->state))
    return fail(ACCT_ERR_ALIGN, "q, k, v, y, state must be 16-byte aligned");
  if (!(a->scale > -1e30f) || !(a->scale < 1e30f)) return fail(ACCT_ERR_SHAPE, "scale must be a finite number");
  const int n_kv = a->N_kv > 0 ? a->N_kv : a->N;
  LinStepParams p;
  memset(&p, 0, sizeof(p));
  const struct { const char* name; const int64_t* given; int heads; int64_t* out; } rows[3] = {
      {"q", a->q_stride, a->N, p.q_stride}, {"k", a->k_stride, n_kv, p.k_stride}, {"v", a->v_stride, n_kv, p.v_stride}};
  for (const auto& x : rows)
    for (int i = 0; i < 2; ++i) {
      x.out[i] = packed_or(x.given[i], i == 0 ? static_cast<int64_t>(x.heads) * a->D : a->D);
      if (x.out[i] < a->D) return fail(ACCT_ERR_SHAPE, "%s strides must not be smaller than head_dim", x.name);
      if (x.out[i] % 8 != 0) return fail(ACCT_ERR_ALIGN, "%s stride (%lld elements) is not a multiple of 8", x.name, (long long)x.out[i]);
    }
  p.q = a->q; p.k = a->k; p.v = a->v; p.y = a->y;
  p.state = a->state;
  p.log_decay = a->log_decay;
  p.B = a->B; p.N = a->N; p.D = a->D; p.group = a->N / n_kv;
  p.scale = a->scale;
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  const cudaError_t e = launch_linear_step(p, a->dtype == ACCT_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "launching the linear attention step");
  return ACCT_OK;
}

int acct_rotary(const acct_rotary_args* a, void* stream) { return rotary(a, a != nullptr ? a->positions : nullptr, nullptr, stream); }
int acct_rotary_wide(const acct_rotary_args* a, const int64_t* positions, void* stream) { return rotary(a, nullptr, positions, stream); }

}  // extern "C"
