// Gradient of the RMS norm.  With r = 1 / sqrt(mean(x^2) + eps) of a row and s = mean(g * alpha * x):
//   dx = r * (g * alpha - x * r^2 * s) + grad_sum        dalpha = sum over rows of g * x * r
// A row needs two sums (x^2 and g * alpha * x) before its dx can be written; dalpha is a sum over rows, held in
// f32 per block of rows and added up by a second kernel in a fixed order.
#include "launch.h"

namespace cb200 {

namespace {

constexpr int kThreads = 256;

// Sums of two values over the CTA, returned to every thread.  `scratch` holds 2 * warps floats; a later call may
// reuse it after a __syncthreads.
__device__ __forceinline__ float2 block_sum2(float a, float b, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  a = warp_sum(a);
  b = warp_sum(b);
  if (lane == 0) {
    scratch[2 * warp] = a;
    scratch[2 * warp + 1] = b;
  }
  __syncthreads();
  float2 t = make_float2(0.0f, 0.0f);
  for (int w = 0; w < warps; ++w) {
    t.x += scratch[2 * w];
    t.y += scratch[2 * w + 1];
  }
  return t;
}

// r and r^3 * mean(g alpha x) of a row from its two sums.
__device__ __forceinline__ float2 row_factors(float sum_xx, float sum_gax, int n, float eps) {
  const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum_xx, static_cast<float>(n)), eps)));
  return make_float2(r, r * (r * (r * __fdiv_rn(sum_gax, static_cast<float>(n)))));
}

// ---- any shape, any alignment: three passes -----------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(kThreads) factors_kernel(const RmsBackwardArgs a, float2* factors) {
  __shared__ float scratch[2 * kThreads / 32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float xx = 0.0f, gax = 0.0f;
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
      const float x = load_elem<DT>(a.x, row * a.n + c);
      const float ga = load_elem<DT>(a.grad, row * a.n + c) * load_elem<DT>(a.alpha, c);
      xx = fmaf(x, x, xx);
      gax = fmaf(ga, x, gax);
    }
    const float2 t = block_sum2(xx, gax, scratch);
    if (threadIdx.x == 0) factors[row] = row_factors(t.x, t.y, a.n, a.eps);
    __syncthreads();
  }
}

// Block (i, p): 256 columns of the rows of slice p.
template <int DT>
__global__ void __launch_bounds__(kThreads) alpha_partials_kernel(const RmsBackwardArgs a, const float2* factors, float* partials) {
  const int64_t begin = a.rows * blockIdx.y / gridDim.y, end = a.rows * (blockIdx.y + 1) / gridDim.y;
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.n) return;
  float acc = 0.0f;
  for (int64_t row = begin; row < end; ++row)
    acc = fmaf(load_elem<DT>(a.grad, row * a.n + c) * load_elem<DT>(a.x, row * a.n + c), factors[row].x, acc);
  partials[static_cast<int64_t>(blockIdx.y) * a.n + c] = acc;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) dx_kernel(const RmsBackwardArgs a, const float2* factors) {
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float2 f = factors[row];
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
      const int64_t at = row * a.n + c;
      const float ga = load_elem<DT>(a.grad, at) * load_elem<DT>(a.alpha, c);
      float d = fmaf(f.x, ga, -f.y * load_elem<DT>(a.x, at));
      if (a.grad_sum != nullptr) d += load_elem<DT>(a.grad_sum, at);
      store_elem<DT>(a.dx, at, d);
    }
  }
}

// 32 columns per CTA, its eight warps over the partial rows.
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* partials, int n_partials, int cols, float* out) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float acc = 0.0f;
  if (c < cols)
    for (int p = warp; p < n_partials; p += 8) acc += partials[static_cast<int64_t>(p) * cols + c];
  part[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && c < cols) {
    for (int w = 1; w < 8; ++w) acc += part[w][lane];
    out[c] = acc;
  }
}

int max_partials() { return 2 * sm_count(); }

template <int DT>
cudaError_t launch_any(const RmsBackwardArgs& a, float* partials, float2* factors, cudaStream_t stream) {
  int64_t grid = static_cast<int64_t>(sm_count()) * 8;
  if (grid > a.rows) grid = a.rows;
  factors_kernel<DT><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, factors);
  const int slices = static_cast<int>(a.rows < max_partials() ? a.rows : max_partials());
  const dim3 blocks((a.n + kThreads - 1) / kThreads, slices);
  alpha_partials_kernel<DT><<<blocks, kThreads, 0, stream>>>(a, factors, partials);
  dx_kernel<DT><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, factors);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_sum_partials(partials, slices, a.n, a.dalpha, stream);
}

}  // namespace

cudaError_t launch_sum_partials(const float* partials, int n_partials, int cols, float* out, cudaStream_t stream) {
  sum_partials_kernel<<<(cols + 31) / 32, 256, 0, stream>>>(partials, n_partials, cols, out);
  return cudaGetLastError();
}

int64_t rms_backward_workspace(int64_t rows, int n) {
  const int64_t partials = (static_cast<int64_t>(max_partials()) * n * 4 + 15) & ~int64_t(15);
  return partials + rows * 8;
}

cudaError_t launch_rms_backward(int dtype, const RmsBackwardArgs& a, void* workspace, cudaStream_t stream) {
  if (a.rows == 0) return cudaMemsetAsync(a.dalpha, 0, static_cast<size_t>(a.n) * 4, stream);
  float* partials = static_cast<float*>(workspace);
  float2* factors = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) +
                                              ((static_cast<int64_t>(max_partials()) * a.n * 4 + 15) & ~int64_t(15)));
  switch (dtype) {
    case kDtF32: return launch_any<kDtF32>(a, partials, factors, stream);
    case kDtF16: return launch_any<kDtF16>(a, partials, factors, stream);
    default: return launch_any<kDtBF16>(a, partials, factors, stream);
  }
}

}  // namespace cb200
