// Gradient of the RMS norm.  With r = 1 / sqrt(mean(x^2) + eps) of a row and s = mean(g * alpha * x):
//   dx = r * (g * alpha - x * r^2 * s) + grad_sum        dalpha = sum over rows of g * x * r
// A row needs two sums (x^2 and g * alpha * x) before its dx can be written; dalpha is a sum over rows, held in
// f32 per block of rows and added up by a second kernel in a fixed order.  f32 inside, dx rounded once.
//
// Bound by memory: 65536 x 8192 bf16 with grad_sum (4.3 GB) 640 us, 6.7 TB/s, a little above a plain copy's rate (three
// reads per write); 32768 x 8192 f32 (3.2 GB) 534 us; 1000000 x 256 bf16 with grad_sum (2.0 GB) 325 us.
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

// ---- rows too long for the kernels below: three passes, element by element ----------------------------------------
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
  follow_previous();
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

// 32 columns per CTA, its warps over the partial rows: warp w takes rows w, w + 32, ... and the warps' sums are added
// in order.  Columns from `split` on go to out2.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(kSumWarps * 32) sum_partials_kernel(const float* partials, int n_partials, int cols,
                                                                      float* out, int split, float* out2) {
  __shared__ float part[kSumWarps][33];
  follow_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float acc = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int p = warp; p < n_partials; p += kSumWarps) acc += partials[static_cast<int64_t>(p) * cols + c];
  }
  part[warp][lane] = acc;
  __syncthreads();
  // warp w adds up column w: lane k holds the sum of warp k
  const float sum = warp_sum(part[lane][warp]);
  const int column = blockIdx.x * 32 + warp;
  if (lane == 0 && column < cols) {
    if (column < split) out[column] = sum;
    else out2[column - split] = sum;
  }
}

int max_partials() { return 4 * sm_count(); }

// ---- one pass ----------------------------------------------------------------------------------------------------
// TPR threads take a row, up to 64 bytes of it each, as vectors of VB bytes (the widest of 16, 8 and 4 that rows and
// pointers are aligned to; columns fixed per thread, so dalpha accumulates in registers).  A CTA works on kThreads / TPR
// rows at a time and walks over the rows persistently.  Every thread brings its own vectors of the rows to come into
// its own slots of shared memory by asynchronous copies, kStages - 1 rows ahead, and reads back only what it copied
// itself: no barrier guards the ring, and the only one per row is that of the row sums (none for rows of up to 32
// threads).
// U: 16-byte units per thread.
template <int U>
struct Ring {
  static constexpr int kStages = U >= 3 ? 2 : 4;
};

template <int PENDING>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// A vector of VB bytes in shared memory and what it holds, as pairs.
template <int VB>
struct VecOf;
template <>
struct VecOf<16> {
  using type = uint4;
};
template <>
struct VecOf<8> {
  using type = uint2;
};
template <>
struct VecOf<4> {
  using type = uint32_t;
};
template <int VB>
__device__ __forceinline__ void copy_async(void* slot, const void* src) {
  if constexpr (VB == 16) cp_async16(slot, src);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(slot)), "l"(src), "n"(VB) : "memory");
}
template <int DT, int VB>
__device__ __forceinline__ void widen(const typename VecOf<VB>::type& v, F2 (&f)[VB / Elem<DT>::kBytes / 2]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int j = 0; j < VB / Elem<DT>::kBytes / 2; ++j) {
    if constexpr (DT == kDtF32) {
      f[j] = pair(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    } else {
      const float2 t = unpack2<DT>(w[j]);
      f[j] = pair(t.x, t.y);
    }
  }
}
template <int DT, int VB>
__device__ __forceinline__ void store_pairs(void* to, const F2 (&f)[VB / Elem<DT>::kBytes / 2]) {
  uint32_t w[VB / 4];
#pragma unroll
  for (int j = 0; j < VB / Elem<DT>::kBytes / 2; ++j) {
    const float2 t = unpair(f[j]);
    if constexpr (DT == kDtF32) {
      w[2 * j] = __float_as_uint(t.x);
      w[2 * j + 1] = __float_as_uint(t.y);
    } else {
      w[j] = pack2<DT>(t.x, t.y);
    }
  }
  if constexpr (VB == 16) stg_stream(static_cast<uint4*>(to), make_uint4(w[0], w[1], w[2], w[3]));
  else if constexpr (VB == 8) asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(to), "r"(w[0]), "r"(w[1]) : "memory");
  else asm volatile("st.global.cs.u32 [%0], %1;" ::"l"(to), "r"(w[0]) : "memory");
}

struct FastArgs {
  RmsBackwardArgs a;
  float* partials;  // [grid][n]
  int tpr_shift, V; // threads per row, vectors per row
};

constexpr int kWideThreads = 512;  // CTAs for rows that 256 threads do not hold
constexpr int kScratchBytes = 2 * kWideThreads / 32 * 8;

// The row sums (x^2, g alpha x) over the tpr threads of a row, to all of them.  `scratch` is [2][warps]; a CTA's calls
// use its halves in turn, since a thread may still be reading the last call's.
__device__ __forceinline__ float2 row_sums(float2 sums, int tpr, int sub, float2* scratch, int& turn) {
  for (int o = tpr < 32 ? tpr >> 1 : 16; o > 0; o >>= 1) {
    sums.x += __shfl_xor_sync(0xFFFFFFFFu, sums.x, o);
    sums.y += __shfl_xor_sync(0xFFFFFFFFu, sums.y, o);
  }
  if (tpr > 32) {
    if ((threadIdx.x & 31) == 0) scratch[turn + (threadIdx.x >> 5)] = sums;
    __syncthreads();
    const int warps = tpr >> 5, first = sub * warps;
    sums = make_float2(0.0f, 0.0f);
    for (int i = 0; i < warps; ++i) {
      sums.x += scratch[turn + first + i].x;
      sums.y += scratch[turn + first + i].y;
    }
    turn ^= blockDim.x / 32;
  }
  return sums;
}

// Adds the lines [group][n] of this CTA's row groups into its line of the partial sums.
__device__ __forceinline__ void add_groups(const float* line, int groups, int n, float* partials) {
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    float t = line[c];
    for (int i = 1; i < groups; ++i) t += line[i * n + c];
    partials[static_cast<int64_t>(blockIdx.x) * n + c] = t;
  }
}

template <int DT, int VB, int U, bool SUM, int T>
__global__ void __launch_bounds__(T, 512 / T) rows_kernel(const FastArgs f) {
  follow_previous();
  extern __shared__ __align__(16) unsigned char shared[];
  using V = typename VecOf<VB>::type;
  constexpr int P2 = VB / Elem<DT>::kBytes / 2, kInputs = SUM ? 3 : 2, kStages = Ring<U>::kStages, VPT = U * 16 / VB;
  float2* scratch = reinterpret_cast<float2*>(shared);     // [2][warps]
  V* ring = reinterpret_cast<V*>(shared + kScratchBytes);  // [stage][input][vector][thread]
  const RmsBackwardArgs& a = f.a;
  const int tpr = 1 << f.tpr_shift, sub = threadIdx.x >> f.tpr_shift, at0 = threadIdx.x & (tpr - 1);
  const int rows_at_once = T >> f.tpr_shift;
  const int n_vec = f.V;
  const float inv_n = 1.0f / static_cast<float>(a.n);
  const V* src[3] = {static_cast<const V*>(a.x), static_cast<const V*>(a.grad), static_cast<const V*>(a.grad_sum)};
  const int64_t n_tiles = (a.rows + rows_at_once - 1) / rows_at_once;

  auto fetch = [&](int64_t tile, int stage) {
    const int64_t row = tile * rows_at_once + sub;
    if (row < a.rows) {
#pragma unroll
      for (int i = 0; i < kInputs; ++i)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
          if (at0 + k * tpr < n_vec)
            copy_async<VB>(&ring[((stage * kInputs + i) * VPT + k) * T + threadIdx.x], src[i] + row * n_vec + at0 + k * tpr);
    }
    cp_async_commit();
  };

  F2 acc[VPT][P2];
  V w[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    w[k] = V{};
    if (at0 + k * tpr < n_vec) w[k] = __ldg(static_cast<const V*>(a.alpha) + at0 + k * tpr);
#pragma unroll
    for (int j = 0; j < P2; ++j) acc[k][j] = 0;
  }

  int64_t ahead = blockIdx.x;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    fetch(ahead, s);
    ahead += gridDim.x;
  }
  int stage = 0, turn = 0;
  for (int64_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
    fetch(ahead, stage == 0 ? kStages - 1 : stage - 1);
    ahead += gridDim.x;
    copies_wait<kStages - 1>();
    const V* slot = ring + stage * kInputs * VPT * T + threadIdx.x;
    stage = stage == kStages - 1 ? 0 : stage + 1;
    const int64_t row = tile * rows_at_once + sub;
    const bool live = row < a.rows;
    F2 xx = 0, gax = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!live || at0 + k * tpr >= n_vec) continue;
      F2 x[P2], g[P2], u[P2];
      widen<DT, VB>(slot[k * T], x);
      widen<DT, VB>(slot[(VPT + k) * T], g);
      widen<DT, VB>(w[k], u);
#pragma unroll
      for (int j = 0; j < P2; ++j) {
        xx = fma2(x[j], x[j], xx);
        gax = fma2(mul2(g[j], u[j]), x[j], gax);
      }
    }
    const float2 t1 = unpair(xx), t2 = unpair(gax);
    const float2 sums = row_sums(make_float2(t1.x + t1.y, t2.x + t2.y), tpr, sub, scratch, turn);
    const float r = rsqrtf(fmaf(sums.x, inv_n, a.eps));
    const float along = -r * (r * (r * (sums.y * inv_n)));
    const F2 r2 = pair(r, r), along2 = pair(along, along);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!live || at0 + k * tpr >= n_vec) continue;
      F2 x[P2], g[P2], u[P2], d[P2];
      widen<DT, VB>(slot[k * T], x);
      widen<DT, VB>(slot[(VPT + k) * T], g);
      widen<DT, VB>(w[k], u);
#pragma unroll
      for (int j = 0; j < P2; ++j) {
        const F2 gr = mul2(g[j], r2);
        acc[k][j] = fma2(gr, x[j], acc[k][j]);
        d[j] = fma2(gr, u[j], mul2(x[j], along2));
      }
      if constexpr (SUM) {
        F2 e[P2];
        widen<DT, VB>(slot[(2 * VPT + k) * T], e);
#pragma unroll
        for (int j = 0; j < P2; ++j) d[j] = add2(d[j], e[j]);
      }
      store_pairs<DT, VB>(static_cast<V*>(a.dx) + row * n_vec + at0 + k * tpr, d);
    }
  }

  // the rows' groups of this CTA, added through shared memory (the ring is idle now): [group][n]
  __syncthreads();
  float* line = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (at0 + k * tpr >= n_vec) continue;
#pragma unroll
    for (int j = 0; j < P2; ++j)
      *reinterpret_cast<F2*>(line + sub * a.n + (at0 + k * tpr) * 2 * P2 + 2 * j) = acc[k][j];
  }
  add_groups(line, rows_at_once, a.n, f.partials);
}

// Rows of any alignment, up to E elements per thread.  The rows of a visit lie next to one another in memory and come
// into shared memory as they lie, whole 16-byte vectors by asynchronous copies, the ends by elements, while the visit
// before is worked on; the threads then pick their elements.  (Loads of single elements out of memory leave too few
// bytes in flight: 60000 rows of 4097 bf16 took 2.6 ms.)
// Bytes of a visit's rows in shared memory: they begin where their first byte does within 16.
__host__ __device__ inline int64_t visit_bytes(int64_t rows, int n, int elem) { return (rows * n * elem + 15 + 15) / 16 * 16; }

template <int DT>
__device__ __forceinline__ void bring_rows(unsigned char* to, const void* from, int64_t bytes) {
  using T = typename Elem<DT>::type;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(from), end = begin + bytes;
  const uintptr_t base = begin & ~uintptr_t(15), whole = (begin + 15) & ~uintptr_t(15), behind = end & ~uintptr_t(15);
  for (uintptr_t p = whole + threadIdx.x * 16; p + 16 <= end; p += kThreads * 16) cp_async16(to + (p - base), reinterpret_cast<const void*>(p));
  // fewer than 16 bytes at either end; all of them where no whole vector lies between
  const uintptr_t head_end = whole < end ? whole : end, tail = behind > head_end ? behind : head_end;
  for (uintptr_t p = begin + threadIdx.x * sizeof(T); p < head_end; p += kThreads * sizeof(T)) *reinterpret_cast<T*>(to + (p - base)) = *reinterpret_cast<const T*>(p);
  for (uintptr_t p = tail + threadIdx.x * sizeof(T); p < end; p += kThreads * sizeof(T)) *reinterpret_cast<T*>(to + (p - base)) = *reinterpret_cast<const T*>(p);
}

template <int DT, int E, bool SUM>
__global__ void __launch_bounds__(kThreads, 2) rows_any_kernel(const FastArgs f) {
  follow_previous();
  extern __shared__ __align__(16) unsigned char shared[];
  constexpr int kInputs = SUM ? 3 : 2, kBytes = Elem<DT>::kBytes;
  const RmsBackwardArgs& a = f.a;
  const int tpr = 1 << f.tpr_shift, sub = threadIdx.x >> f.tpr_shift, at0 = threadIdx.x & (tpr - 1);
  const int rows_at_once = kThreads >> f.tpr_shift;
  const float inv_n = 1.0f / static_cast<float>(a.n);
  float2* scratch = reinterpret_cast<float2*>(shared);
  unsigned char* ring = shared + kScratchBytes;  // [stage][input][visit_bytes]
  const int64_t piece = visit_bytes(rows_at_once, a.n, kBytes);
  const void* src[3] = {a.x, a.grad, a.grad_sum};
  auto address = [&](int i, int64_t row) { return static_cast<const unsigned char*>(src[i]) + row * a.n * kBytes; };
  auto bring = [&](int64_t first, int stage) {
    if (first < a.rows) {
      const int64_t rows = a.rows - first < rows_at_once ? a.rows - first : rows_at_once;
#pragma unroll
      for (int i = 0; i < kInputs; ++i) bring_rows<DT>(ring + (stage * kInputs + i) * piece, address(i, first), rows * a.n * kBytes);
    }
    cp_async_commit();
  };

  float acc[E] = {}, w[E];
#pragma unroll
  for (int k = 0; k < E; ++k) w[k] = at0 + k * tpr < a.n ? load_elem<DT>(a.alpha, at0 + k * tpr) : 0.0f;
  int turn = 0, stage = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows_at_once;
  int64_t first = static_cast<int64_t>(blockIdx.x) * rows_at_once;
  bring(first, 0);
  for (; first < a.rows; first += step) {
    cp_async_wait_all();
    __syncthreads();  // the visit's rows are here, and the visit before is done with the other stage
    bring(first + step, stage ^ 1);
    const int64_t row = first + sub;
    const int n = row < a.rows ? a.n : 0;
    const unsigned char* at[3];
#pragma unroll
    for (int i = 0; i < kInputs; ++i)
      at[i] = ring + (stage * kInputs + i) * piece + (reinterpret_cast<uintptr_t>(address(i, first)) & 15) + static_cast<int64_t>(sub) * a.n * kBytes;
    stage ^= 1;
    float xx = 0.0f, gax = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int c = at0 + k * tpr;
      if (c >= n) continue;
      const float x = load_elem<DT>(at[0], c);
      xx = fmaf(x, x, xx);
      gax = fmaf(load_elem<DT>(at[1], c) * w[k], x, gax);
    }
    const float2 sums = row_sums(make_float2(xx, gax), tpr, sub, scratch, turn);
    const float r = rsqrtf(fmaf(sums.x, inv_n, a.eps));
    const float along = -r * (r * (r * (sums.y * inv_n)));
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int c = at0 + k * tpr;
      if (c >= n) continue;
      const float x = load_elem<DT>(at[0], c), gr = load_elem<DT>(at[1], c) * r;
      acc[k] = fmaf(gr, x, acc[k]);
      float d = fmaf(gr, w[k], x * along);
      if constexpr (SUM) d += load_elem<DT>(at[2], c);
      store_elem<DT>(a.dx, row * a.n + c, d);
    }
  }
  __syncthreads();
  float* line = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int k = 0; k < E; ++k)
    if (at0 + k * tpr < a.n) line[sub * a.n + at0 + k * tpr] = acc[k];
  add_groups(line, rows_at_once, a.n, f.partials);
}

// The same grid with and without grad_sum (per_sm: what fits with it), so that dalpha is summed in the same order.
template <typename K>
cudaError_t launch_persistent(K kern, const FastArgs& f, int threads, size_t smem, int per_sm, cudaStream_t stream) {
  cudaError_t e = kernel_launch_config(reinterpret_cast<const void*>(kern), threads, smem, -1, nullptr);
  if (e != cudaSuccess) return e;
  const int rows_at_once = threads >> f.tpr_shift;
  int64_t grid = static_cast<int64_t>(sm_count()) * per_sm;
  if (grid > max_partials()) grid = max_partials();
  const int64_t tiles = (f.a.rows + rows_at_once - 1) / rows_at_once;
  if (grid > tiles) grid = tiles;
  kern<<<static_cast<unsigned>(grid), threads, smem, stream>>>(f);
  e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_sum_partials(f.partials, static_cast<int>(grid), f.a.n, f.a.dalpha, f.a.n, nullptr, stream);
}

template <int DT, int VB, int U, int T>
cudaError_t launch_rows(const FastArgs& f, cudaStream_t stream) {
  const size_t input = static_cast<size_t>(Ring<U>::kStages) * U * T * 16;
  int per_sm = 1;
  const cudaError_t e = kernel_launch_config(reinterpret_cast<const void*>(rows_kernel<DT, VB, U, true, T>), T, kScratchBytes + input * 3, -1, &per_sm);
  if (e != cudaSuccess) return e;
  return f.a.grad_sum != nullptr ? launch_persistent(rows_kernel<DT, VB, U, true, T>, f, T, kScratchBytes + input * 3, per_sm, stream)
                                 : launch_persistent(rows_kernel<DT, VB, U, false, T>, f, T, kScratchBytes + input * 2, per_sm, stream);
}

// The fewest threads per row (8 .. max_threads) that leave at most `most` vectors to each; how many that are, or more
// than `most`.
int split_row(FastArgs& f, int most, int max_threads) {
  const auto per_thread = [&] { return (f.V + (1 << f.tpr_shift) - 1) >> f.tpr_shift; };
  f.tpr_shift = 3;
  while ((1 << f.tpr_shift) < max_threads && per_thread() > most) ++f.tpr_shift;
  return per_thread();
}

// false: the row is too long for the vectors.
template <int DT, int VB>
bool launch_fast(const RmsBackwardArgs& a, float* partials, cudaStream_t stream, cudaError_t* e) {
  FastArgs f{a, partials, 3, a.n * Elem<DT>::kBytes / VB};
  const int units = (split_row(f, 64 / VB, kWideThreads) * VB + 15) / 16;
  if (units > 4) return false;
  if (f.tpr_shift == 9) {  // more than half of what the 512 threads hold
    *e = units == 3 ? launch_rows<DT, VB, 3, kWideThreads>(f, stream) : launch_rows<DT, VB, 4, kWideThreads>(f, stream);
    return true;
  }
  switch (units) {
    case 1: *e = launch_rows<DT, VB, 1, kThreads>(f, stream); break;
    case 2: *e = launch_rows<DT, VB, 2, kThreads>(f, stream); break;
    case 3: *e = launch_rows<DT, VB, 3, kThreads>(f, stream); break;
    default: *e = launch_rows<DT, VB, 4, kThreads>(f, stream); break;
  }
  return true;
}

constexpr int kMaxElements = 32;  // per thread

template <int DT, int E>
cudaError_t launch_elements(const FastArgs& f, cudaStream_t stream) {
  const size_t input = 2 * static_cast<size_t>(visit_bytes(kThreads >> f.tpr_shift, f.a.n, Elem<DT>::kBytes));
  int per_sm = 1;
  const cudaError_t e = kernel_launch_config(reinterpret_cast<const void*>(rows_any_kernel<DT, E, true>), kThreads, kScratchBytes + 3 * input, -1, &per_sm);
  if (e != cudaSuccess) return e;
  return f.a.grad_sum != nullptr ? launch_persistent(rows_any_kernel<DT, E, true>, f, kThreads, kScratchBytes + 3 * input, per_sm, stream)
                                 : launch_persistent(rows_any_kernel<DT, E, false>, f, kThreads, kScratchBytes + 2 * input, per_sm, stream);
}

template <int DT>
cudaError_t launch_long(const RmsBackwardArgs& a, float* partials, float2* factors, cudaStream_t stream) {
  int64_t grid = static_cast<int64_t>(sm_count()) * 8;
  if (grid > a.rows) grid = a.rows;
  factors_kernel<DT><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, factors);
  const int slices = static_cast<int>(a.rows < max_partials() ? a.rows : max_partials());
  const dim3 blocks((a.n + kThreads - 1) / kThreads, slices);
  alpha_partials_kernel<DT><<<blocks, kThreads, 0, stream>>>(a, factors, partials);
  dx_kernel<DT><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, factors);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_sum_partials(partials, slices, a.n, a.dalpha, a.n, nullptr, stream);
}

template <int DT>
cudaError_t launch_dt(const RmsBackwardArgs& a, float* partials, float2* factors, cudaStream_t stream) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.grad) | reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.alpha) |
                       reinterpret_cast<uintptr_t>(a.grad_sum) | reinterpret_cast<uintptr_t>(a.dx) |
                       static_cast<uintptr_t>(a.n) * Elem<DT>::kBytes;
  cudaError_t e = cudaSuccess;
  if (at % 16 == 0 && launch_fast<DT, 16>(a, partials, stream, &e)) return e;
  if (at % 8 == 0 && launch_fast<DT, 8>(a, partials, stream, &e)) return e;
  if constexpr (DT != kDtF32)
    if (at % 4 == 0 && launch_fast<DT, 4>(a, partials, stream, &e)) return e;
  FastArgs f{a, partials, 3, a.n};
  const int elements = split_row(f, kMaxElements, kThreads);
  if (elements > kMaxElements) return launch_long<DT>(a, partials, factors, stream);
  if (elements <= 8) return launch_elements<DT, 8>(f, stream);
  if (elements <= 16) return launch_elements<DT, 16>(f, stream);
  return elements <= 24 ? launch_elements<DT, 24>(f, stream) : launch_elements<DT, 32>(f, stream);
}

}  // namespace

cudaError_t launch_sum_partials(const float* partials, int n_partials, int cols, float* out, int split, float* out2,
                                cudaStream_t stream) {
  return launch_dependent(true, sum_partials_kernel, static_cast<unsigned>((cols + 31) / 32), kSumWarps * 32, 0, stream, partials, n_partials,
                          cols, out, split, out2);
}

// Bytes of the lines of partial sums: no grid has more CTAs, or slices, than there are rows.
static int64_t partial_bytes(int64_t rows, int n) {
  const int64_t lines = rows < max_partials() ? rows : max_partials();
  return (lines * n * 4 + 15) & ~int64_t(15);
}

// Behind them the factors of the rows, for lengths that may take the three passes.
int64_t rms_backward_workspace(int64_t rows, int n) {
  return partial_bytes(rows, n) + (n > kThreads * kMaxElements ? rows * 8 : 0);
}

cudaError_t launch_rms_backward(int dtype, const RmsBackwardArgs& a, void* workspace, cudaStream_t stream) {
  if (a.rows == 0) return cudaMemsetAsync(a.dalpha, 0, static_cast<size_t>(a.n) * 4, stream);
  float* partials = static_cast<float*>(workspace);
  float2* factors = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + partial_bytes(a.rows, a.n));
  switch (dtype) {
    case kDtF32: return launch_dt<kDtF32>(a, partials, factors, stream);
    case kDtF16: return launch_dt<kDtF16>(a, partials, factors, stream);
    default: return launch_dt<kDtBF16>(a, partials, factors, stream);
  }
}

}  // namespace cb200
