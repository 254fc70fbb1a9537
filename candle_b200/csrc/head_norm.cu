// RMS norm of every query and key head with the rotary embedding in the same pass, and its gradient.
//   forward   u = x r w,  r = 1 / sqrt(mean(x^2) + eps);   out = R u   (R: the rotation of the token's position)
//   gradient  v = R^T g;  dx = r (v w - x r^2 mean(v w x));  dw = sum over rows of v x r
// A row is one head of one token.  As separate operators (norm, rotation) queries and keys make two trips through
// memory and are rounded twice; here one.  Everything is f32 inside, rounded once to T when it is stored; the sums of the
// weights' gradients stay in f32.
//
// Measured (B200, 32 + 8 heads of 128 columns, bf16): forward, 16384 tokens, 336 MB: 61 us, 5.5 TB/s, 0.85 of a copy's rate
// (the same kernel with scalar arithmetic and IEEE divisions: 72 us, bound by issue slots at 22 instructions per
// element); gradient, 16384 tokens, 504 MB: 97 us, 5.2 TB/s with the sum of the partial gradients (with v computed twice
// instead of kept 106 us; rows staged through shared memory instead of registers 104 us).  64 tokens: 2.6 us on the
// device, a launch's latency.
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
  float* partials;  // [workers][2][dim]
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
  follow_previous();
  const Common& c = a.c;
  const int lane = threadIdx.x & 31;
  const int half = c.rotary / 2, items = c.dim - half;
  const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
  for (int side = 0; side < 2; ++side) {
    const int heads = side ? c.k_heads : c.q_heads;
    const void* weight = side ? c.k_weight : c.q_weight;
    float* dw = a.partials + (static_cast<int64_t>(worker) * 2 + side) * c.dim;
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

// ---- vector kernels ----------------------------------------------------------------------------------------------
// A group of G lanes (a power of two) takes a row.  Lane p of the group holds item p of the row (and p + G with
// NI == 2): two vectors of PV elements that make PV pairs -- columns [p PV, ...) and their partners rotary / 2 further
// on, or with interleaved pairs 2 PV columns in a row -- so the rotation needs no exchange between lanes and its PV
// cosines and sines are one vector of each table.  Behind the rotated columns an item is two vectors as they are.
// A warp's unit of work is R rows for each of its 32 / G groups, all of one token: the angles are fetched once for
// them, and all loads are issued before the first is used.
template <int W>
struct Words {
  uint32_t w[W];
};

template <int W>
__device__ __forceinline__ Words<W> load_words(const void* p) {
  Words<W> r;
  if constexpr (W == 1) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
  } else if constexpr (W == 2) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  } else {
    static_assert(W == 4, "4, 8 or 16 bytes");
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                 : "l"(p));
  }
  return r;
}
template <int W>
__device__ __forceinline__ void store_words(void* p, const Words<W>& r) {
  if constexpr (W == 1) {
    asm volatile("st.global.cs.u32 [%0], %1;" ::"l"(p), "r"(r.w[0]) : "memory");
  } else if constexpr (W == 2) {
    asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]) : "memory");
  } else {
    stg_stream(static_cast<uint4*>(p), make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]));
  }
}
template <int DT, int PV>
struct Vec {
  static constexpr int kWords = PV * Elem<DT>::kBytes / 4;
  using type = Words<kWords>;
};
// PV elements of a table that stays in cache.
template <int DT, int PV>
__device__ __forceinline__ typename Vec<DT, PV>::type load_table(const void* base, int64_t elem) {
  const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(base) + elem * Elem<DT>::kBytes);
  constexpr int kWords = Vec<DT, PV>::kWords;
  typename Vec<DT, PV>::type v;
  if constexpr (kWords % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
      v.w[4 * i] = q.x, v.w[4 * i + 1] = q.y, v.w[4 * i + 2] = q.z, v.w[4 * i + 3] = q.w;
    }
  } else if constexpr (kWords == 2) {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
    v.w[0] = q.x, v.w[1] = q.y;
  } else {
    v.w[0] = __ldg(p);
  }
  return v;
}

// Pair j (elements 2 j, 2 j + 1) of a vector, widened.
template <int DT, int PV>
__device__ __forceinline__ F2 widen2(const typename Vec<DT, PV>::type& v, int j) {
  if constexpr (DT == kDtF32) {
    return pair(__uint_as_float(v.w[2 * j]), __uint_as_float(v.w[2 * j + 1]));
  } else {
    const float2 t = unpack2<DT>(v.w[j]);
    return pair(t.x, t.y);
  }
}
template <int DT, int PV>
__device__ __forceinline__ void narrow2(typename Vec<DT, PV>::type& v, int j, F2 f) {
  const float2 t = unpair(f);
  if constexpr (DT == kDtF32) {
    v.w[2 * j] = __float_as_uint(t.x);
    v.w[2 * j + 1] = __float_as_uint(t.y);
  } else {
    v.w[j] = pack2<DT>(t.x, t.y);
  }
}
// Element e of a vector, widened.
template <int DT, int PV>
__device__ __forceinline__ float element(const typename Vec<DT, PV>::type& v, int e) {
  if constexpr (DT == kDtF32) {
    return __uint_as_float(v.w[e]);
  } else {
    const float2 t = unpack2<DT>(v.w[e / 2]);
    return e & 1 ? t.y : t.x;
  }
}

// First columns of the two vectors of item p (second < 0: there is none), and whether they are rotated.
template <int PV, bool INTER>
__device__ __forceinline__ bool item_columns(const Common& c, int p, int& c1, int& c2) {
  const int half = c.rotary / 2;
  const bool turned = p * PV < half;
  if (turned) {
    c1 = INTER ? 2 * p * PV : p * PV;
    c2 = INTER ? c1 + PV : c1 + half;
  } else {
    c1 = c.rotary + 2 * (p * PV - half);
    c2 = c1 + PV < c.dim ? c1 + PV : -1;
  }
  return turned;
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// How a warp walks over its units (token, block of heads of one side): the steps are computed on the host, so the
// loop has no division.
struct Walk {
  int64_t n_units, stride;  // units, and units between a warp's visits
  int q_blocks, blocks;     // head blocks of the queries, and of both sides, per token
  int d_block, d_b, d_t;    // the stride as (batch, token, block)
  int group_shift;          // G = 1 << group_shift lanes per row
  int items;                // items per row
};

struct Place {
  int64_t unit;
  int b, t, block;
  __device__ __forceinline__ void start(const Walk& w, int64_t first, int64_t tokens) {
    unit = first;
    const int64_t n = first / w.blocks;
    block = static_cast<int>(first - n * w.blocks);
    b = static_cast<int>(n / tokens);
    t = static_cast<int>(n - b * tokens);
  }
  __device__ __forceinline__ void next(const Walk& w, int tokens) {
    unit += w.stride;
    block += w.d_block;
    b += w.d_b;
    unsigned u = static_cast<unsigned>(t) + w.d_t;
    if (block >= w.blocks) {
      block -= w.blocks;
      ++u;
    }
    if (u >= static_cast<unsigned>(tokens)) {
      u -= tokens;
      ++b;
    }
    t = static_cast<int>(u);
  }
};

// A unit's rows share token and weight, so weight and angle are multiplied once per unit: with half-split pairs
// (r: a row's inverse root mean square, by the approximate reciprocal square root, off by at most 2 ulp)
//   y1 = (x1 r) (w1 cos) - (x2 r) (w2 sin),   y2 = (x1 r) (w1 sin) + (x2 r) (w2 cos).
template <int DT, int DTC, int PV, int NI, int R, bool INTER>
__global__ void __launch_bounds__(kThreads, NI == 2 ? 2 : 3) forward_kernel(const ForwardArgs a, const Walk walk) {
  const Common& c = a.c;
  constexpr int kBytes = Elem<DT>::kBytes, kWords = Vec<DT, PV>::kWords, P2 = PV / 2;
  using V = typename Vec<DT, PV>::type;
  const int lane = threadIdx.x & 31;
  const int group = 1 << walk.group_shift, rows_at_once = 32 >> walk.group_shift;
  const int sub = lane >> walk.group_shift, p0 = lane & (group - 1);
  const int half = c.rotary / 2, tokens = static_cast<int>(c.tokens);
  const float inv_dim = 1.0f / static_cast<float>(c.dim);
  int c1[NI], c2[NI];
  bool turned[NI], here[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    here[i] = p0 + i * group < walk.items;
    turned[i] = item_columns<PV, INTER>(c, p0 + i * group, c1[i], c2[i]);
  }
  Place at;
  at.start(walk, static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5), c.tokens);
  for (; at.unit < walk.n_units; at.next(walk, tokens)) {
    const int side = at.block < walk.q_blocks ? 0 : 1;
    const int first = (at.block - (side ? walk.q_blocks : 0)) * (R * rows_at_once) + sub;
    const int live = (side ? c.k_heads : c.q_heads) - first;  // rows r with r * rows_at_once < live exist
    const unsigned char* in = row_of(a.in[side], at.b, at.t, first);
    const int64_t in_step = a.in[side].head_stride * rows_at_once;
    V x[R][NI][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        x[r][i][0] = V{};
        x[r][i][1] = V{};
        if (r * rows_at_once < live && here[i]) {
          x[r][i][0] = load_words<kWords>(in + r * in_step + c1[i] * kBytes);
          if (c2[i] >= 0) x[r][i][1] = load_words<kWords>(in + r * in_step + c2[i] * kBytes);
        }
      }
    const int64_t pos = position_of(c, static_cast<int64_t>(at.b) * tokens + at.t, at.t, at.block == 0 && lane == 0);
    if (pos < 0) continue;
    const void* weight = side ? c.k_weight : c.q_weight;
    F2 k1[NI][PV], k2[NI][PV];  // half-split: k1 = {w1 cos, w1 sin}, k2 = {-w2 sin, w2 cos}; see below for INTER
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (!here[i]) continue;
      const V w1 = load_table<DT, PV>(weight, c1[i]);
      V w2{};
      if (c2[i] >= 0) w2 = load_table<DT, PV>(weight, c2[i]);
      if (turned[i]) {
        const auto co = load_table<DTC, PV>(c.cos, pos * half + (p0 + i * group) * PV);
        const auto si = load_table<DTC, PV>(c.sin, pos * half + (p0 + i * group) * PV);
        if constexpr (INTER) {
          // pair j = (x1, x2) in one register pair: y = (x1, x2) (w1 cos, w2 cos) + (x2, x1) (-w2 sin, w1 sin)
#pragma unroll
          for (int j = 0; j < PV; ++j) {
            const F2 w = widen2<DT, PV>(j < P2 ? w1 : w2, j % P2);
            const float cj = element<DTC, PV>(co, j), sj = element<DTC, PV>(si, j);
            k1[i][j] = mul2(w, pair(cj, cj));
            k2[i][j] = mul2(swapped(w), pair(-sj, sj));
          }
        } else {
#pragma unroll
          for (int j = 0; j < P2; ++j) {
            const F2 u1 = widen2<DT, PV>(w1, j), u2 = widen2<DT, PV>(w2, j);
            const F2 cj = widen2<DTC, PV>(co, j), sj = widen2<DTC, PV>(si, j);
            k1[i][j] = mul2(u1, cj);
            k1[i][P2 + j] = mul2(u1, sj);
            k2[i][j] = mul2(mul2(u2, sj), pair(-1.0f, -1.0f));
            k2[i][P2 + j] = mul2(u2, cj);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < P2; ++j) {
          k1[i][j] = widen2<DT, PV>(w1, j);
          k1[i][P2 + j] = widen2<DT, PV>(w2, j);
        }
      }
    }
    unsigned char* out = row_of(a.out[side], at.b, at.t, first);
    const int64_t out_step = a.out[side].head_stride * rows_at_once;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      F2 sum2 = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < PV; ++j) {
          const F2 f = widen2<DT, PV>(x[r][i][j / P2], j % P2);
          sum2 = fma2(f, f, sum2);
        }
      const float2 s = unpair(sum2);
      const float inv = rsqrtf(fmaf(group_sum(s.x + s.y, group), inv_dim, c.eps));
      const F2 inv2 = pair(inv, inv);
      if (r * rows_at_once >= live) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (!here[i]) continue;
        V y1, y2;
        if (!turned[i]) {
#pragma unroll
          for (int j = 0; j < P2; ++j) {
            narrow2<DT, PV>(y1, j, mul2(mul2(widen2<DT, PV>(x[r][i][0], j), inv2), k1[i][j]));
            narrow2<DT, PV>(y2, j, mul2(mul2(widen2<DT, PV>(x[r][i][1], j), inv2), k1[i][P2 + j]));
          }
        } else if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < PV; ++j) {
            const F2 u = mul2(widen2<DT, PV>(x[r][i][j / P2], j % P2), inv2);
            narrow2<DT, PV>(j < P2 ? y1 : y2, j % P2, fma2(u, k1[i][j], mul2(swapped(u), k2[i][j])));
          }
        } else {
#pragma unroll
          for (int j = 0; j < P2; ++j) {
            const F2 u1 = mul2(widen2<DT, PV>(x[r][i][0], j), inv2), u2 = mul2(widen2<DT, PV>(x[r][i][1], j), inv2);
            narrow2<DT, PV>(y1, j, fma2(u1, k1[i][j], mul2(u2, k2[i][j])));
            narrow2<DT, PV>(y2, j, fma2(u1, k1[i][P2 + j], mul2(u2, k2[i][P2 + j])));
          }
        }
        store_words(out + r * out_step + c1[i] * kBytes, y1);
        if (c2[i] >= 0) store_words(out + r * out_step + c2[i] * kBytes, y2);
      }
    }
  }
}

// The same units, first all of the queries, then all of the keys: a lane's columns are the same in every row, so it
// keeps their part of the weight's gradient in registers and the CTA adds its lanes' parts once per side.
// The rows' sums are taken for all R rows before the first of them is finished.
template <int DT, int DTC, int PV, int NI, int R, bool INTER>
__global__ void __launch_bounds__(kThreads, NI == 2 ? 1 : 2) backward_kernel(const BackwardArgs a, const Walk q_walk,
                                                                                  const Walk k_walk) {
  follow_previous();
  extern __shared__ float line[];  // [warp][dim]
  const Common& c = a.c;
  constexpr int kBytes = Elem<DT>::kBytes, kWords = Vec<DT, PV>::kWords, P2 = PV / 2;
  using V = typename Vec<DT, PV>::type;
  using VC = typename Vec<DTC, PV>::type;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group_shift = q_walk.group_shift;
  const int group = 1 << group_shift, rows_at_once = 32 >> group_shift;
  const int sub = lane >> group_shift, p0 = lane & (group - 1);
  const int half = c.rotary / 2, tokens = static_cast<int>(c.tokens);
  const float inv_dim = 1.0f / static_cast<float>(c.dim);
  int c1[NI], c2[NI];
  bool turned[NI], here[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    here[i] = p0 + i * group < q_walk.items;
    turned[i] = item_columns<PV, INTER>(c, p0 + i * group, c1[i], c2[i]);
  }
  for (int side = 0; side < 2; ++side) {
    const Walk& walk = side ? k_walk : q_walk;
    const int heads = side ? c.k_heads : c.q_heads;
    F2 acc[NI][PV], w[NI][PV];
    const void* weight = side ? c.k_weight : c.q_weight;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      V u[2] = {V{}, V{}};
      if (here[i]) {
        u[0] = load_table<DT, PV>(weight, c1[i]);
        if (c2[i] >= 0) u[1] = load_table<DT, PV>(weight, c2[i]);
      }
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        w[i][j] = widen2<DT, PV>(u[j / P2], j % P2);
        acc[i][j] = 0;
      }
    }
    if (walk.n_units > 0) {
      Place at;
      at.start(walk, static_cast<int64_t>(blockIdx.x) * kWarps + warp, c.tokens);
      for (; at.unit < walk.n_units; at.next(walk, tokens)) {
        const int first = at.block * (R * rows_at_once) + sub;
        const int live = heads - first;
        const unsigned char* px = row_of(a.x[side], at.b, at.t, first);
        const unsigned char* pg = row_of(a.grad[side], at.b, at.t, first);
        const int64_t x_step = a.x[side].head_stride * rows_at_once, g_step = a.grad[side].head_stride * rows_at_once;
        V x[R][NI][2], g[R][NI][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            x[r][i][0] = x[r][i][1] = g[r][i][0] = g[r][i][1] = V{};
            if (r * rows_at_once < live && here[i]) {
              x[r][i][0] = load_words<kWords>(px + r * x_step + c1[i] * kBytes);
              g[r][i][0] = load_words<kWords>(pg + r * g_step + c1[i] * kBytes);
              if (c2[i] >= 0) {
                x[r][i][1] = load_words<kWords>(px + r * x_step + c2[i] * kBytes);
                g[r][i][1] = load_words<kWords>(pg + r * g_step + c2[i] * kBytes);
              }
            }
          }
        const int64_t pos = position_of(c, static_cast<int64_t>(at.b) * tokens + at.t, at.t, at.block == 0 && lane == 0);
        if (pos < 0) continue;
        VC co[NI], si[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          co[i] = si[i] = VC{};
          if (here[i] && turned[i]) {
            co[i] = load_table<DTC, PV>(c.cos, pos * half + (p0 + i * group) * PV);
            si[i] = load_table<DTC, PV>(c.sin, pos * half + (p0 + i * group) * PV);
          }
        }
        // v = R^T g of row r, item i: pairs of elements j < P2 from the first vector, the others from the second
        auto back = [&](int r, int i, F2(&v)[PV]) {
          if (!turned[i]) {
#pragma unroll
            for (int j = 0; j < PV; ++j) v[j] = widen2<DT, PV>(g[r][i][j / P2], j % P2);
          } else if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < PV; ++j) {
              const F2 u = widen2<DT, PV>(g[r][i][j / P2], j % P2);
              const float cj = element<DTC, PV>(co[i], j), sj = element<DTC, PV>(si[i], j);
              v[j] = fma2(u, pair(cj, cj), mul2(swapped(u), pair(sj, -sj)));
            }
          } else {
#pragma unroll
            for (int j = 0; j < P2; ++j) {
              const F2 u1 = widen2<DT, PV>(g[r][i][0], j), u2 = widen2<DT, PV>(g[r][i][1], j);
              const F2 cj = widen2<DTC, PV>(co[i], j), sj = widen2<DTC, PV>(si[i], j);
              v[j] = fma2(u1, cj, mul2(u2, sj));
              const float2 n = unpair(sj);
              v[P2 + j] = fma2(u2, cj, mul2(u1, pair(-n.x, -n.y)));
            }
          }
        };
        float xx[R], vwx[R];
        F2 v[R][NI][PV];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          F2 s1 = 0, s2 = 0;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            back(r, i, v[r][i]);
#pragma unroll
            for (int j = 0; j < PV; ++j) {
              const F2 f = widen2<DT, PV>(x[r][i][j / P2], j % P2);
              s1 = fma2(f, f, s1);
              s2 = fma2(mul2(v[r][i][j], w[i][j]), f, s2);
            }
          }
          const float2 t1 = unpair(s1), t2 = unpair(s2);
          xx[r] = t1.x + t1.y;
          vwx[r] = t2.x + t2.y;
        }
        for (int o = group >> 1; o > 0; o >>= 1)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            xx[r] += __shfl_xor_sync(0xFFFFFFFFu, xx[r], o);
            vwx[r] += __shfl_xor_sync(0xFFFFFFFFu, vwx[r], o);
          }
        unsigned char* pd = row_of(a.dx[side], at.b, at.t, first);
        const int64_t d_step = a.dx[side].head_stride * rows_at_once;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r * rows_at_once >= live) continue;
          const float inv = rsqrtf(fmaf(xx[r], inv_dim, c.eps));
          const float along = -inv * (inv * (inv * (vwx[r] * inv_dim)));
          const F2 inv2 = pair(inv, inv), along2 = pair(along, along);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            if (!here[i]) continue;
            V y[2];
#pragma unroll
            for (int j = 0; j < PV; ++j) {
              const F2 f = widen2<DT, PV>(x[r][i][j / P2], j % P2), vr = mul2(v[r][i][j], inv2);
              acc[i][j] = fma2(vr, f, acc[i][j]);
              narrow2<DT, PV>(y[j / P2], j % P2, fma2(vr, w[i][j], mul2(f, along2)));
            }
            store_words(pd + r * d_step + c1[i] * kBytes, y[0]);
            if (c2[i] >= 0) store_words(pd + r * d_step + c2[i] * kBytes, y[1]);
          }
        }
      }
    }
    // the lanes of a warp that hold the same columns, then the warps
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        float2 t = unpair(acc[i][j]);
        for (int o = group; o < 32; o <<= 1) {
          t.x += __shfl_xor_sync(0xFFFFFFFFu, t.x, o);
          t.y += __shfl_xor_sync(0xFFFFFFFFu, t.y, o);
        }
        if (sub == 0 && here[i] && (j < P2 || c2[i] >= 0)) {
          const int column = (j < P2 ? c1[i] : c2[i]) + 2 * (j % P2);
          line[warp * c.dim + column] = t.x;
          line[warp * c.dim + column + 1] = t.y;
        }
      }
    __syncthreads();
    for (int d = threadIdx.x; d < c.dim; d += kThreads) {
      float t = line[d];
#pragma unroll
      for (int k = 1; k < kWarps; ++k) t += line[k * c.dim + d];
      a.partials[(static_cast<int64_t>(blockIdx.x) * 2 + side) * c.dim + d] = t;
    }
    __syncthreads();
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

bool aligned_rows(const HeadRows& h, uint64_t bytes) {
  return ((reinterpret_cast<uint64_t>(h.base) | static_cast<uint64_t>(h.batch_stride) | static_cast<uint64_t>(h.token_stride) |
           static_cast<uint64_t>(h.head_stride)) & (bytes - 1)) == 0;
}

// Elements per vector: the widest (up to 16 bytes) that the rotated part and the rows' alignment allow; 0: none.
int vector_elements(const Common& c, const HeadRows* rows, int n_rows, int elem, int table_elem) {
  for (int pv = 16 / elem; pv * elem >= 4 && pv >= 2; pv /= 2) {
    bool ok = c.rotary % (2 * pv) == 0 && c.dim % pv == 0;
    for (int i = 0; i < n_rows && ok; ++i) ok = aligned_rows(rows[i], static_cast<uint64_t>(pv) * elem);
    const uint64_t weights = reinterpret_cast<uint64_t>(c.q_weight) | reinterpret_cast<uint64_t>(c.k_weight);
    const uint64_t tables = reinterpret_cast<uint64_t>(c.cos) | reinterpret_cast<uint64_t>(c.sin);
    const int table_bytes = pv * table_elem < 16 ? pv * table_elem : 16;
    if (ok && weights % (pv * elem) == 0 && tables % table_bytes == 0) return pv;
  }
  return 0;
}

// The walk over (token, block of heads of one side) for rows of `items` items, `rows` rows per lane, by `grid` CTAs;
// `grid` == 0 is replaced by as many as there is work for, at most max_grid.
Walk plan_walk(const Common& c, int q_heads, int k_heads, int items, int rows, int64_t max_grid, int64_t& grid) {
  Walk w{};
  w.items = items;
  while ((1 << w.group_shift) < items && w.group_shift < 5) ++w.group_shift;
  const int per_block = (32 >> w.group_shift) * rows;
  w.q_blocks = (q_heads + per_block - 1) / per_block;
  w.blocks = w.q_blocks + (k_heads + per_block - 1) / per_block;
  w.n_units = c.n_tokens * w.blocks;
  if (grid == 0) {
    grid = (w.n_units + kWarps - 1) / kWarps;
    if (grid > max_grid) grid = max_grid;
  }
  w.stride = grid * kWarps;
  if (w.blocks == 0) return w;
  const int64_t d_token = w.stride / w.blocks;
  w.d_block = static_cast<int>(w.stride - d_token * w.blocks);
  w.d_b = static_cast<int>(d_token / c.tokens);
  w.d_t = static_cast<int>(d_token - w.d_b * c.tokens);
  return w;
}

int row_items(const Common& c, int pv) { return c.rotary / 2 / pv + ((c.dim - c.rotary) / pv + 1) / 2; }

template <int DT, int DTC, int PV, int NI, int R>
cudaError_t launch_forward_vec(const ForwardArgs& a, const Walk& w, int64_t grid, cudaStream_t stream) {
  if (a.c.interleaved) forward_kernel<DT, DTC, PV, NI, R, true><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, w);
  else forward_kernel<DT, DTC, PV, NI, R, false><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a, w);
  return cudaGetLastError();
}

// Rows per lane and unit: 32 bytes of each vector's elements, however narrow the vectors.
template <int DT, int PV>
constexpr int kUnitRows = 2 * Elem<DT>::kPerVec / PV;

template <int DT, int DTC, int PV>
cudaError_t launch_forward_pv(const ForwardArgs& a, cudaStream_t stream, bool* done) {
  const Common& c = a.c;
  const int items = row_items(c, PV);
  const int64_t cap = static_cast<int64_t>(sm_count()) * (items > 32 ? 2 : 3);
  int64_t grid = 0;
  *done = items <= 64;
  if (!*done) return cudaSuccess;
  if (items > 32) {
    const Walk w = plan_walk(c, c.q_heads, c.k_heads, items, 1, cap, grid);
    return launch_forward_vec<DT, DTC, PV, 2, 1>(a, w, grid, stream);
  }
  // Few units: a row per lane and unit, so that more warps have one.  Device times so and with kRows: 32 + 8 bf16 heads of 128 (the
  // limit is 1421 tokens) 64 tokens 2.3 and 2.7 us, 256 3.1 both, 1024 6.7 and 5.9, 2048 10.9 and 8.8; 16 + 2 f32 heads of 64
  // (2368 tokens) 256 2.7 and 2.8, 900 4.0 and 3.5, 1300 4.5 and 4.8, 2000 6.1 and 5.5.  In the last factor of two below the limit
  // it depends on how the units fill the warps.
  constexpr int kRows = kUnitRows<DT, PV>;
  Walk w = plan_walk(c, c.q_heads, c.k_heads, items, kRows, cap, grid);
  if (w.n_units >= 2 * cap * kWarps) return launch_forward_vec<DT, DTC, PV, 1, kRows>(a, w, grid, stream);
  grid = 0;
  w = plan_walk(c, c.q_heads, c.k_heads, items, 1, cap, grid);
  return launch_forward_vec<DT, DTC, PV, 1, 1>(a, w, grid, stream);
}

template <int DT, int DTC>
cudaError_t launch_forward(const ForwardArgs& a, cudaStream_t stream) {
  HeadRows rows[4] = {a.in[0], a.in[1], a.out[0], a.out[1]};
  bool done = false;
  cudaError_t e = cudaSuccess;
  switch (vector_elements(a.c, rows, 4, Elem<DT>::kBytes, Elem<DTC>::kBytes)) {
    case 8:
      if constexpr (DT != kDtF32) e = launch_forward_pv<DT, DTC, 8>(a, stream, &done);
      break;
    case 4: e = launch_forward_pv<DT, DTC, 4>(a, stream, &done); break;
    case 2: e = launch_forward_pv<DT, DTC, 2>(a, stream, &done); break;
    default: break;
  }
  if (done) return e;
  const int64_t n_rows = a.c.n_tokens * (a.c.q_heads + a.c.k_heads);
  int64_t grid = (n_rows + kWarps - 1) / kWarps;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  if (grid > cap) grid = cap;
  forward_any_kernel<DT, DTC><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

int max_workers() { return sm_count() * 4 * kWarps; }

template <int DT, int DTC, int PV, int NI, int R>
cudaError_t launch_backward_vec(BackwardArgs& a, int items, int ctas_per_sm, cudaStream_t stream) {
  const Common& c = a.c;
  auto kern = c.interleaved ? backward_kernel<DT, DTC, PV, NI, R, true> : backward_kernel<DT, DTC, PV, NI, R, false>;
  const int64_t cap = static_cast<int64_t>(sm_count()) * ctas_per_sm;
  int64_t grid = 0, k_grid = 0;
  plan_walk(c, c.q_heads, 0, items, R, cap, grid);
  plan_walk(c, c.k_heads, 0, items, R, cap, k_grid);
  if (k_grid > grid) grid = k_grid;
  const Walk q = plan_walk(c, c.q_heads, 0, items, R, cap, grid), k = plan_walk(c, c.k_heads, 0, items, R, cap, grid);
  a.workers = static_cast<int>(grid);
  kern<<<static_cast<unsigned>(grid), kThreads, static_cast<size_t>(kWarps) * c.dim * 4, stream>>>(a, q, k);
  return cudaGetLastError();
}

template <int DT, int DTC, int PV>
cudaError_t launch_backward_pv(BackwardArgs& a, cudaStream_t stream, bool* done) {
  const int items = row_items(a.c, PV);
  *done = items <= 64;
  if (!*done) return cudaSuccess;
  if (items > 32) return launch_backward_vec<DT, DTC, PV, 2, 1>(a, items, 1, stream);
  return launch_backward_vec<DT, DTC, PV, 1, kUnitRows<DT, PV>>(a, items, 2, stream);
}

template <int DT, int DTC>
cudaError_t launch_backward(BackwardArgs& a, float* dq_weight, float* dk_weight, cudaStream_t stream) {
  HeadRows rows[6] = {a.grad[0], a.grad[1], a.x[0], a.x[1], a.dx[0], a.dx[1]};
  bool done = false;
  cudaError_t e = cudaSuccess;
  switch (vector_elements(a.c, rows, 6, Elem<DT>::kBytes, Elem<DTC>::kBytes)) {
    case 8:
      if constexpr (DT != kDtF32) e = launch_backward_pv<DT, DTC, 8>(a, stream, &done);
      break;
    case 4: e = launch_backward_pv<DT, DTC, 4>(a, stream, &done); break;
    case 2: e = launch_backward_pv<DT, DTC, 2>(a, stream, &done); break;
    default: break;
  }
  if (!done) {
    const int64_t n_rows = a.c.n_tokens * (a.c.q_heads > a.c.k_heads ? a.c.q_heads : a.c.k_heads);
    int64_t grid = (n_rows + kWarps - 1) / kWarps;
    if (grid * kWarps > max_workers()) grid = max_workers() / kWarps;
    a.workers = static_cast<int>(grid) * kWarps;
    backward_any_kernel<DT, DTC><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
    e = cudaGetLastError();
  }
  return e != cudaSuccess ? e : launch_sum_partials(a.partials, a.workers, 2 * a.c.dim, dq_weight, a.c.dim, dk_weight, stream);
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
