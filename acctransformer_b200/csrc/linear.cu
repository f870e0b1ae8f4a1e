// Linear attention with a decay for each head, over whole sequences.
//
//   S_t = exp(g) S_(t-1) + b_t c_t^T,   y_t = scale S_t^T a_t
//
// A thread block has 32 columns of one head's state in registers and walks the sequence's tokens: a warp has 4 columns, a lane 1/8 of
// a column.  16 tokens at a time are staged in shared memory in fp32.
#include "fa_common.cuh"
#include "linear.cuh"

namespace acct {
namespace {

constexpr int kCols = 32, kStage = 16, kParts = 8, kPer = kLinMaxHeadDim / kParts;

template <bool BF16>
__global__ void __launch_bounds__(kCols * kParts) linear_kernel(const LinParams p) {
  __shared__ float sa[kStage][kLinMaxHeadDim], sb[kStage][kLinMaxHeadDim], sc[kStage][kCols];
  const int slices = (p.D + kCols - 1) / kCols, tid = threadIdx.x;
  int item = blockIdx.x;
  const LinPass& pass = p.pass[item % p.passes];
  item /= p.passes;
  const int e0 = item % slices * kCols, h = item / slices % p.N, b = item / slices / p.N;
  int row0, n;
  lin_rows(p, b, row0, n);
  const int col = tid / kParts, part = tid % kParts, e = e0 + col;
  const float lambda = static_cast<float>(exp(static_cast<double>(p.log_decay[h])));
  float s[kPer];
  for (int i = 0; i < kPer; ++i) {
    const int d = part + kParts * i;
    s[i] = p.state_in != nullptr && d < p.D && e < p.D ? p.state_in[((static_cast<int64_t>(b) * p.N + h) * p.D + d) * p.D + e] : 0.f;
  }
  const int64_t batch = p.cu != nullptr ? 0 : b;
  auto at = [&](const LinOperand& o, int row, int d) {
    return load16<BF16>(o.ptr, batch * o.stride[0] + (h / o.group) * o.stride[1] + row * o.stride[2] + d);
  };
  for (int t0 = 0; t0 < n; t0 += kStage) {
    __syncthreads();
    for (int i = tid; i < kStage * kLinMaxHeadDim; i += blockDim.x) {
      const int t = i / kLinMaxHeadDim, d = i % kLinMaxHeadDim, row = row0 + (pass.reverse ? n - 1 - (t0 + t) : t0 + t);
      const bool there = t0 + t < n && d < p.D;
      sa[t][d] = there ? at(pass.a, row, d) : 0.f;
      sb[t][d] = there ? at(pass.b, row, d) : 0.f;
      if (d < kCols) sc[t][d] = there && e0 + d < p.D ? at(pass.c, row, e0 + d) : 0.f;
    }
    __syncthreads();
    for (int t = 0; t < kStage && t0 + t < n; ++t) {
      float y = 0.f;
      for (int i = 0; i < kPer; ++i) {
        s[i] = fmaf(lambda, s[i], sb[t][part + kParts * i] * sc[t][col]);
        y = fmaf(sa[t][part + kParts * i], s[i], y);
      }
      for (int d = 1; d < kParts; d <<= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
      if (part == 0 && e < p.D) {
        const int row = row0 + (pass.reverse ? n - 1 - (t0 + t) : t0 + t);
        const int64_t to = batch * pass.y_stride[0] + h * pass.y_stride[1] + row * pass.y_stride[2] + e;
        if (pass.y_f32) static_cast<float*>(pass.y)[to] = y * p.scale;
        else if (BF16) static_cast<__nv_bfloat16*>(pass.y)[to] = __float2bfloat16(y * p.scale);
        else static_cast<__half*>(pass.y)[to] = __float2half(y * p.scale);
      }
    }
  }
  if (p.state_out != nullptr)
    for (int i = 0; i < kPer; ++i) {
      const int d = part + kParts * i;
      if (d < p.D && e < p.D) p.state_out[((static_cast<int64_t>(b) * p.N + h) * p.D + d) * p.D + e] = s[i];
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
  const float* from = p.parts[which] + ((static_cast<int64_t>(b) * p.N_kv + h) * p.group * p.S + s) * p.D + d;
  float4 sum = *reinterpret_cast<const float4*>(from);
  for (int g = 1; g < p.group; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(g) * p.S * p.D);
    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
  }
  uint16_t* to = static_cast<uint16_t*>(p.out[which]) + b * p.out_stride[which][0] + h * p.out_stride[which][1] + s * p.out_stride[which][2] + d;
  *reinterpret_cast<uint2*>(to) = make_uint2(pack2<BF16>(sum.x, sum.y), pack2<BF16>(sum.z, sum.w));
}

}  // namespace

cudaError_t launch_linear(const LinParams& p, bool bf16, cudaStream_t stream) {
  const unsigned int blocks = static_cast<unsigned int>(p.passes) * ((p.D + kCols - 1) / kCols) * p.N * p.B;
  (bf16 ? linear_kernel<true> : linear_kernel<false>)<<<blocks, kCols * kParts, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_linear_reduce(const LinReduce& p, bool bf16, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(p.B) * p.N_kv * p.S * (p.D / 4);
  const dim3 grid(static_cast<unsigned int>((threads + 255) / 256), 2);
  (bf16 ? linear_reduce_kernel<true> : linear_reduce_kernel<false>)<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace acct
