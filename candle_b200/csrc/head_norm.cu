// RMS norm of every query and key head with the rotary embedding in the same pass, and its gradient.
//   forward   u = x r w,  r = 1 / sqrt(mean(x^2) + eps);   out = R u   (R: the rotation of the token's position)
//   gradient  v = R^T g;  dx = r (v w - x r^2 mean(v w x));  dw = sum over rows of v x r
// A row is one head of one token.  As separate operators (norm, rotation) queries and keys make two trips through
// memory and are rounded twice; here one.
#include "launch.h"

namespace cb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct HeadRows {
  unsigned char* base;
  int64_t batch_stride, token_stride, head_stride;  // bytes
};

struct Common {
  const void *q_weight, *k_weight, *cos, *sin, *positions;
  int64_t n_tokens;     // batch * tokens
  int64_t tokens;
  int64_t max_positions;
  int q_heads, k_heads;
  int dim, rotary;
  float eps;
  int interleaved, position_dtype;
  cb200_status* status;
};

struct ForwardArgs {
  Common c;
  HeadRows in[2], out[2];  // queries, keys
};

struct BackwardArgs {
  Common c;
  HeadRows grad[2], x[2], dx[2];
  float* partials;  // [2][workers][dim]
  int workers;
};

__device__ __forceinline__ unsigned char* row_of(const HeadRows& h, int64_t b, int64_t t, int head) {
  return h.base + b * h.batch_stride + t * h.token_stride + head * h.head_stride;
}

// The position of token `n` (b, t), or -1 after reporting one that the tables do not have.
__device__ __forceinline__ int64_t position_of(const Common& c, int64_t n, int64_t t, bool report) {
  if (c.positions == nullptr) return t;
  const uint64_t p = read_id(c.positions, c.position_dtype, n);
  if (p < static_cast<uint64_t>(c.max_positions)) return static_cast<int64_t>(p);
  if (report) report_status(c.status, CB200_STATUS_INVALID_INDEX, n, static_cast<int64_t>(p), c.max_positions);
  return -1;
}

__device__ __forceinline__ float inverse_rms(float sum, int dim, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(dim)), eps)));
}

// ---- any head size, any alignment: a warp per row, element by element -------------------------------------------
// Work item p of a row: pair p of the rotated part for p < rotary / 2, else one column behind it.
__device__ __forceinline__ void pair_columns(const Common& c, int p, int& c1, int& c2) {
  const int half = c.rotary / 2;
  if (p < half) {
    c1 = c.interleaved ? 2 * p : p;
    c2 = c.interleaved ? 2 * p + 1 : p + half;
  } else {
    c1 = c.rotary + p - half;
    c2 = -1;
  }
}

template <int DT, int DTC>
__global__ void __launch_bounds__(kThreads) forward_any_kernel(const ForwardArgs a) {
  const Common& c = a.c;
  const int lane = threadIdx.x & 31;
  const int heads = c.q_heads + c.k_heads, half = c.rotary / 2, items = c.dim - half;
  const int64_t n_rows = c.n_tokens * heads;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); row < n_rows;
       row += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t n = row / heads;
    int head = static_cast<int>(row - n * heads);
    const int64_t b = n / c.tokens, t = n - b * c.tokens;
    const int64_t pos = position_of(c, n, t, head == 0 && lane == 0);
    if (pos < 0) continue;
    const int side = head < c.q_heads ? 0 : 1;
    head -= side ? c.q_heads : 0;
    const void* weight = side ? c.k_weight : c.q_weight;
    const unsigned char* x = row_of(a.in[side], b, t, head);
    unsigned char* y = row_of(a.out[side], b, t, head);
    float sum = 0.0f;
    for (int i = lane; i < c.dim; i += 32) {
      const float v = load_elem<DT>(x, i);
      sum = fmaf(v, v, sum);
    }
    const float r = inverse_rms(warp_sum(sum), c.dim, c.eps);
    for (int p = lane; p < items; p += 32) {
      int c1, c2;
      pair_columns(c, p, c1, c2);
      const float u1 = load_elem<DT>(x, c1) * r * load_elem<DT>(weight, c1);
      if (c2 < 0) {
        store_elem<DT>(y, c1, u1);
        continue;
      }
      const float u2 = load_elem<DT>(x, c2) * r * load_elem<DT>(weight, c2);
      const float co = load_elem<DTC>(c.cos, pos * half + p), si = load_elem<DTC>(c.sin, pos * half + p);
      store_elem<DT>(y, c1, u1 * co - u2 * si);
      store_elem<DT>(y, c2, u1 * si + u2 * co);
    }
  }
}

// A warp keeps the weights' gradient of its rows in its own line of `partials` (each lane its own columns).
template <int DT, int DTC>
__global__ void __launch_bounds__(kThreads) backward_any_kernel(const BackwardArgs a) {
  const Common& c = a.c;
  const int lane = threadIdx.x & 31;
  const int half = c.rotary / 2, items = c.dim - half;
  const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
  for (int side = 0; side < 2; ++side) {
    const int heads = side ? c.k_heads : c.q_heads;
    const void* weight = side ? c.k_weight : c.q_weight;
    float* dw = a.partials + (static_cast<int64_t>(side) * a.workers + worker) * c.dim;
    for (int p = lane; p < items; p += 32) {
      int c1, c2;
      pair_columns(c, p, c1, c2);
      dw[c1] = 0.0f;
      if (c2 >= 0) dw[c2] = 0.0f;
    }
    const int64_t n_rows = c.n_tokens * heads;
    for (int64_t row = worker; row < n_rows; row += a.workers) {
      const int64_t n = row / heads;
      const int head = static_cast<int>(row - n * heads);
      const int64_t b = n / c.tokens, t = n - b * c.tokens;
      const int64_t pos = position_of(c, n, t, head == 0 && lane == 0);
      if (pos < 0) continue;
      const unsigned char* x = row_of(a.x[side], b, t, head);
      const unsigned char* g = row_of(a.grad[side], b, t, head);
      unsigned char* dx = row_of(a.dx[side], b, t, head);
      float r = 0.0f, s = 0.0f;
      for (int pass = 0; pass < 2; ++pass) {
        float xx = 0.0f, vwx = 0.0f;
        for (int p = lane; p < items; p += 32) {
          int c1, c2;
          pair_columns(c, p, c1, c2);
          const float x1 = load_elem<DT>(x, c1), g1 = load_elem<DT>(g, c1), w1 = load_elem<DT>(weight, c1);
          float x2 = 0.0f, v1 = g1, v2 = 0.0f, w2 = 0.0f;
          if (c2 >= 0) {
            const float g2 = load_elem<DT>(g, c2);
            const float co = load_elem<DTC>(c.cos, pos * half + p), si = load_elem<DTC>(c.sin, pos * half + p);
            x2 = load_elem<DT>(x, c2);
            w2 = load_elem<DT>(weight, c2);
            v1 = g1 * co + g2 * si;
            v2 = g2 * co - g1 * si;
          }
          if (pass == 0) {
            xx = fmaf(x1, x1, fmaf(x2, x2, xx));
            vwx = fmaf(v1 * w1, x1, fmaf(v2 * w2, x2, vwx));
          } else {
            store_elem<DT>(dx, c1, r * fmaf(v1, w1, -x1 * s));
            dw[c1] = fmaf(v1 * x1, r, dw[c1]);
            if (c2 >= 0) {
              store_elem<DT>(dx, c2, r * fmaf(v2, w2, -x2 * s));
              dw[c2] = fmaf(v2 * x2, r, dw[c2]);
            }
          }
        }
        if (pass == 0) {
          r = inverse_rms(warp_sum(xx), c.dim, c.eps);
          s = r * (r * __fdiv_rn(warp_sum(vwx), static_cast<float>(c.dim)));
        }
      }
    }
  }
}

HeadRows rows_of(const cb200_heads& h, int elem) {
  return HeadRows{static_cast<unsigned char*>(h.data), h.batch_stride * elem, h.token_stride * elem, h.head_stride * elem};
}

Common common_of(const cb200_qk_args& a, int q_heads, int k_heads, cb200_status* status) {
  Common c{};
  c.q_weight = a.q_weight;
  c.k_weight = a.k_weight;
  c.cos = a.cos;
  c.sin = a.sin;
  c.positions = a.positions;
  c.n_tokens = a.batch * a.tokens;
  c.tokens = a.tokens;
  c.max_positions = a.max_positions;
  c.q_heads = q_heads;
  c.k_heads = k_heads;
  c.dim = a.dim;
  c.rotary = a.rotary;
  c.eps = a.eps;
  c.interleaved = a.interleaved;
  c.position_dtype = a.position_dtype;
  c.status = status;
  return c;
}

template <int DT, int DTC>
cudaError_t launch_forward(const ForwardArgs& a, cudaStream_t stream) {
  const int64_t n_rows = a.c.n_tokens * (a.c.q_heads + a.c.k_heads);
  int64_t grid = (n_rows + kWarps - 1) / kWarps;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  if (grid > cap) grid = cap;
  forward_any_kernel<DT, DTC><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

int max_workers() { return sm_count() * 4 * kWarps; }

template <int DT, int DTC>
cudaError_t launch_backward(BackwardArgs& a, float* dq_weight, float* dk_weight, cudaStream_t stream) {
  const int64_t n_rows = a.c.n_tokens * (a.c.q_heads > a.c.k_heads ? a.c.q_heads : a.c.k_heads);
  int64_t grid = (n_rows + kWarps - 1) / kWarps;
  if (grid * kWarps > max_workers()) grid = max_workers() / kWarps;
  a.workers = static_cast<int>(grid) * kWarps;
  backward_any_kernel<DT, DTC><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_sum_partials(a.partials, a.workers, a.c.dim, dq_weight, stream);
  if (e == cudaSuccess)
    e = launch_sum_partials(a.partials + static_cast<int64_t>(a.workers) * a.c.dim, a.workers, a.c.dim, dk_weight, stream);
  return e;
}

template <typename F>
cudaError_t by_types(int dtype, int table_dtype, F&& f) {
  if (dtype == kDtF32) return f(std::integral_constant<int, kDtF32>{}, std::integral_constant<int, kDtF32>{});
  if (dtype == kDtF16)
    return table_dtype == kDtF32 ? f(std::integral_constant<int, kDtF16>{}, std::integral_constant<int, kDtF32>{})
                                 : f(std::integral_constant<int, kDtF16>{}, std::integral_constant<int, kDtF16>{});
  return table_dtype == kDtF32 ? f(std::integral_constant<int, kDtBF16>{}, std::integral_constant<int, kDtF32>{})
                               : f(std::integral_constant<int, kDtBF16>{}, std::integral_constant<int, kDtBF16>{});
}

}  // namespace

cudaError_t launch_qk_norm_rope(const cb200_heads& q, const cb200_heads& k, const cb200_heads& q_out,
                                const cb200_heads& k_out, const cb200_qk_args& args, cb200_status* status,
                                cudaStream_t stream) {
  const int elem = args.dtype == kDtF32 ? 4 : 2;
  ForwardArgs a{};
  a.c = common_of(args, q.heads, k.heads, status);
  a.in[0] = rows_of(q, elem);
  a.in[1] = rows_of(k, elem);
  a.out[0] = rows_of(q_out, elem);
  a.out[1] = rows_of(k_out, elem);
  if (a.c.n_tokens * (q.heads + k.heads) == 0) return cudaSuccess;
  return by_types(args.dtype, args.table_dtype, [&](auto dt, auto dtc) {
    return launch_forward<decltype(dt)::value, decltype(dtc)::value>(a, stream);
  });
}

int64_t qk_backward_workspace(int dim) { return int64_t(2) * max_workers() * dim * 4; }

cudaError_t launch_qk_norm_rope_backward(const cb200_heads& grad_q, const cb200_heads& grad_k, const cb200_heads& q,
                                         const cb200_heads& k, const cb200_heads& dq, const cb200_heads& dk,
                                         float* dq_weight, float* dk_weight, const cb200_qk_args& args, void* workspace,
                                         cb200_status* status, cudaStream_t stream) {
  const int elem = args.dtype == kDtF32 ? 4 : 2;
  BackwardArgs a{};
  a.c = common_of(args, q.heads, k.heads, status);
  if (a.c.n_tokens * (q.heads + k.heads) == 0) {
    const cudaError_t e = cudaMemsetAsync(dq_weight, 0, static_cast<size_t>(args.dim) * 4, stream);
    return e != cudaSuccess ? e : cudaMemsetAsync(dk_weight, 0, static_cast<size_t>(args.dim) * 4, stream);
  }
  a.grad[0] = rows_of(grad_q, elem);
  a.grad[1] = rows_of(grad_k, elem);
  a.x[0] = rows_of(q, elem);
  a.x[1] = rows_of(k, elem);
  a.dx[0] = rows_of(dq, elem);
  a.dx[1] = rows_of(dk, elem);
  a.partials = static_cast<float*>(workspace);
  return by_types(args.dtype, args.table_dtype, [&](auto dt, auto dtc) {
    return launch_backward<decltype(dt)::value, decltype(dtc)::value>(a, dq_weight, dk_weight, stream);
  });
}

}  // namespace cb200
