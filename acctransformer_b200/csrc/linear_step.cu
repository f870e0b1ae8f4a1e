// Linear attention, one token per sequence: S = exp(g) S + k v^T in place, y = scale S^T q.
//
// Bound by the state's way in and out of memory, 8 D^2 bytes a head.  A thread block has 32 columns of one head's state: 8 lanes read
// 128 bytes of a row, the 32 row groups of a block all rows of it, each thread its rows' 16 bytes all at once, before anything waits.
// 128 sequences, 32 heads of 128: 85 us, 97 % of the copy rate; 4 sequences: 4.2 us, which is latency.
#include "fa_common.cuh"
#include "linear.cuh"

namespace acct {
namespace {

constexpr int kCols = 32, kThreads = 256, kRowGroups = kThreads / (kCols / 4), kRows = kLinMaxHeadDim / kRowGroups;

template <bool BF16>
__global__ void __launch_bounds__(kThreads) linear_step_kernel(const LinStepParams p) {
  __shared__ float4 part[kThreads / 32][kCols / 4];
  const int slices = (p.D + kCols - 1) / kCols, tid = threadIdx.x;
  const int slice = blockIdx.x % slices, h = blockIdx.x / slices % p.N, b = blockIdx.x / slices / p.N;
  const int quad = tid % (kCols / 4), group = tid / (kCols / 4), e = slice * kCols + quad * 4;
  const bool there = e < p.D;
  float4* state = reinterpret_cast<float4*>(p.state + (static_cast<int64_t>(b) * p.N + h) * p.D * p.D);
  const int64_t q0 = b * p.q_stride[0] + h * p.q_stride[1], k0 = b * p.k_stride[0] + (h / p.group) * p.k_stride[1];
  const int64_t v0 = b * p.v_stride[0] + (h / p.group) * p.v_stride[1];
  float4 s[kRows];
  float q[kRows], k[kRows], v[4];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int d = group + kRowGroups * i;
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    q[i] = k[i] = 0.f;
    if (d < p.D && there) {
      s[i] = state[(d * p.D + e) / 4];
      q[i] = load16<BF16>(p.q, q0 + d);
      k[i] = load16<BF16>(p.k, k0 + d);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = there ? load16<BF16>(p.v, v0 + e + j) : 0.f;
  const LinPower lambda = lin_power(p.log_decay[h], 1);      // (over thousands of steps a rounding of it each time would add up)
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int d = group + kRowGroups * i;
    s[i].x = fmaf(lambda.hi, s[i].x, fmaf(lambda.lo, s[i].x, k[i] * v[0])); s[i].y = fmaf(lambda.hi, s[i].y, fmaf(lambda.lo, s[i].y, k[i] * v[1]));
    s[i].z = fmaf(lambda.hi, s[i].z, fmaf(lambda.lo, s[i].z, k[i] * v[2])); s[i].w = fmaf(lambda.hi, s[i].w, fmaf(lambda.lo, s[i].w, k[i] * v[3]));
    if (d < p.D && there) state[(d * p.D + e) / 4] = s[i];
    y.x = fmaf(q[i], s[i].x, y.x); y.y = fmaf(q[i], s[i].y, y.y); y.z = fmaf(q[i], s[i].z, y.z); y.w = fmaf(q[i], s[i].w, y.w);
  }
#pragma unroll
  for (int d = kCols / 4; d < 32; d <<= 1) {
    y.x += __shfl_xor_sync(0xffffffffu, y.x, d); y.y += __shfl_xor_sync(0xffffffffu, y.y, d);
    y.z += __shfl_xor_sync(0xffffffffu, y.z, d); y.w += __shfl_xor_sync(0xffffffffu, y.w, d);
  }
  if (tid % 32 < kCols / 4) part[tid / 32][quad] = y;
  __syncthreads();
  if (tid < kCols / 4 && there) {
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) {
      const float4 x = part[w][quad];
      y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
    }
    uint16_t* to = static_cast<uint16_t*>(p.y) + (static_cast<int64_t>(b) * p.N + h) * p.D + e;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<BF16>(y.x * p.scale, y.y * p.scale), pack2<BF16>(y.z * p.scale, y.w * p.scale));
  }
}

}  // namespace

cudaError_t launch_linear_step(const LinStepParams& p, bool bf16, cudaStream_t stream) {
  const unsigned int blocks = static_cast<unsigned int>((p.D + kCols - 1) / kCols) * p.N * p.B;
  (bf16 ? linear_step_kernel<true> : linear_step_kernel<false>)<<<blocks, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace acct
