// The scaled lookup and the gradient of the embedding table.
//
// Gradient: out[v] = scale * sum of grad[i] over the tokens i with ids[i] == v.  The tokens are sorted by id
// (stable radix sort of (id, position) pairs), so each table row owns a contiguous run of the sorted list and
// its sum has a fixed order: no floating-point atomics, equal inputs give equal bits.  Then
//   - chunk_sums_kernel adds up every aligned chunk of 64 sorted tokens that belongs to one id: text is skewed
//     (the hottest id of 65536 tokens has thousands) and this is what spreads a long run over the GPU;
//   - row_sums_kernel writes the table rows: a warp per (row, tile of columns), and for rows with long runs a CTA,
//     which adds the chunk sums and the ends that do not fill a chunk.
#include "launch.h"

namespace cb200 {

namespace {

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// VEC consecutive elements <-> floats; VEC is the 16-byte vector's element count or 1 (any alignment).
template <int DT, int VEC>
__device__ __forceinline__ void load_floats(const void* base, int64_t elem, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = load_elem<DT>(base, elem);
  } else {
    static_assert(VEC == Elem<DT>::kPerVec, "one 16-byte vector");
    vec_to_floats<DT>(ldg_stream(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + elem * Elem<DT>::kBytes)), f);
  }
}
// As load_floats, for memory that this launch also writes (no read-only path).
template <int DT, int VEC>
__device__ __forceinline__ void load_floats_plain(const void* base, int64_t elem, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = load_elem<DT>(base, elem);
  } else {
    constexpr int kPV = Elem<DT>::kPerVec;
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + elem * Elem<DT>::kBytes);
#pragma unroll
    for (int k = 0; k < VEC / kPV; ++k) {
      float t[kPV];
      vec_to_floats<DT>(p[k], t);
#pragma unroll
      for (int e = 0; e < kPV; ++e) f[k * kPV + e] = t[e];
    }
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_floats(void* base, int64_t elem, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    store_elem<DT>(base, elem, f[0]);
  } else {
    constexpr int kPV = Elem<DT>::kPerVec;
    uint4* p = reinterpret_cast<uint4*>(static_cast<unsigned char*>(base) + elem * Elem<DT>::kBytes);
#pragma unroll
    for (int k = 0; k < VEC / kPV; ++k) {
      float t[kPV];
#pragma unroll
      for (int e = 0; e < kPV; ++e) t[e] = f[k * kPV + e];
      stg_stream(p + k, floats_to_vec<DT>(t));
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Scaled lookup: a warp per (token, tile of columns)
// ---------------------------------------------------------------------------------------------
template <int DT, int VEC>
__global__ void __launch_bounds__(256) scaled_lookup_kernel(const ScaledLookupArgs a, int units, int tiles) {
  const int lane = threadIdx.x & 31;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int64_t n_items = a.n_ids * tiles;
  for (int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < n_items; item += n_warps) {
    const int64_t i = item / tiles;
    const int u = static_cast<int>(item - i * tiles) * 32 + lane;
    const uint64_t id = read_id(a.ids, a.id_dtype, i);
    if (id >= static_cast<uint64_t>(a.vocab)) {
      if (u == 0) report_status(a.status, CB200_STATUS_INVALID_INDEX, i, static_cast<int64_t>(id), a.vocab);
      continue;
    }
    if (u >= units) continue;
    float f[VEC];
    load_floats<DT, VEC>(a.table, static_cast<int64_t>(id) * a.hidden + static_cast<int64_t>(u) * VEC, f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = __fmul_rn(f[e], a.scale);
    store_floats<DT, VEC>(a.out, i * a.hidden + static_cast<int64_t>(u) * VEC, f);
  }
}

template <int DT, int VEC>
cudaError_t launch_scaled_lookup_t(const ScaledLookupArgs& a, cudaStream_t stream) {
  const int units = a.hidden / VEC, tiles = (units + 31) / 32;
  int64_t grid = (a.n_ids * tiles + 7) / 8;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 32;
  if (grid > cap) grid = cap;
  scaled_lookup_kernel<DT, VEC><<<static_cast<unsigned>(grid), 256, 0, stream>>>(a, units, tiles);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_scaled_lookup_dt(const ScaledLookupArgs& a, cudaStream_t stream) {
  constexpr int kPV = Elem<DT>::kPerVec;
  if (a.hidden % kPV == 0 && aligned_to(a.table, 16) && aligned_to(a.out, 16)) return launch_scaled_lookup_t<DT, kPV>(a, stream);
  return launch_scaled_lookup_t<DT, 1>(a, stream);
}

// ---------------------------------------------------------------------------------------------
// Stable radix sort of (id, position), digits of at most 9 bits, two launches per digit: counts per CTA, then
// every CTA derives where its keys of each digit go from all the counts and moves them.  A CTA takes a
// contiguous span of keys in tiles of 4096.  Tokens that contribute nothing (bad ids, padding) get the key
// `vocab` and end up behind all rows.
// ---------------------------------------------------------------------------------------------
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 16;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kSortMaxBits = 9;
constexpr int kSortMaxBins = 1 << kSortMaxBits;
constexpr int kSortMaxCtas = 512;

struct SortArgs {
  const void* ids;           // first pass: the caller's ids
  const uint32_t* keys_in;   // later passes
  const uint32_t* values_in;
  uint32_t* keys_out;
  uint32_t* values_out;
  uint32_t* counts;          // [ctas][bins]
  int2* runs;                // first pass, fresh gradient: cleared here
  int64_t n, vocab, padding_id;
  int id_dtype;
  cb200_status* status;
  int64_t span;              // keys per CTA, a multiple of kSortTile
  int shift, bins;
  int first;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t i, bool report) {
  if (!a.first) return a.keys_in[i];
  const uint64_t id = read_id(a.ids, a.id_dtype, i);
  if (id >= static_cast<uint64_t>(a.vocab)) {
    if (report) report_status(a.status, CB200_STATUS_INVALID_INDEX, i, static_cast<int64_t>(id), a.vocab);
    return static_cast<uint32_t>(a.vocab);
  }
  return static_cast<int64_t>(id) == a.padding_id ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t hist[kSortMaxBins];
  for (int d = threadIdx.x; d < a.bins; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * a.span;
  const int64_t end = begin + a.span < a.n ? begin + a.span : a.n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads)
    atomicAdd(&hist[(sort_key(a, i, true) >> a.shift) & (a.bins - 1)], 1u);
  if (a.runs != nullptr) {
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x; v < a.vocab;
         v += static_cast<int64_t>(gridDim.x) * kSortThreads)
      a.runs[v] = make_int2(0, 0);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.bins; d += kSortThreads) a.counts[static_cast<int64_t>(blockIdx.x) * a.bins + d] = hist[d];
}

__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const SortArgs a) {
  __shared__ uint32_t base[kSortMaxBins];
  __shared__ uint32_t scan[kSortMaxBins];
  __shared__ uint32_t count[kSortWarps][kSortMaxBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // first slot of this CTA's keys of digit d: all smaller digits, and this digit in the CTAs before
  for (int d = threadIdx.x; d < a.bins; d += kSortThreads) {
    uint32_t total = 0, before = 0;
    for (unsigned t = 0; t < gridDim.x; ++t) {
      const uint32_t c = a.counts[static_cast<int64_t>(t) * a.bins + d];
      if (t < blockIdx.x) before += c;
      total += c;
    }
    base[d] = before;
    scan[d] = total;
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t carry = 0;
    for (int d0 = 0; d0 < a.bins; d0 += 32) {
      const uint32_t own = d0 + lane < a.bins ? scan[d0 + lane] : 0u;
      uint32_t v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += up;
      }
      if (d0 + lane < a.bins) base[d0 + lane] += carry + v - own;
      carry += __shfl_sync(0xFFFFFFFFu, v, 31);
    }
  }

  const int64_t begin = blockIdx.x * a.span;
  const int64_t end = begin + a.span < a.n ? begin + a.span : a.n;
  for (int64_t tile = begin; tile < end; tile += kSortTile) {
    for (int d = threadIdx.x; d < kSortWarps * kSortMaxBins; d += kSortThreads) (&count[0][0])[d] = 0;
    __syncthreads();
    uint32_t key[kSortItems], rank[kSortItems];
    const int64_t mine = tile + warp * (32 * kSortItems) + lane;
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const int64_t i = mine + j * 32;
      key[j] = i < end ? sort_key(a, i, false) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const bool live = mine + j * 32 < end;
      const uint32_t digit = live ? (key[j] >> a.shift) & (a.bins - 1) : kSortMaxBins;
      const unsigned peers = __match_any_sync(0xFFFFFFFFu, digit);
      const unsigned below = peers & ((1u << lane) - 1u);
      rank[j] = live ? count[warp][digit] + __popc(below) : 0u;
      __syncwarp();
      if (live && below == 0) count[warp][digit] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.bins; d += kSortThreads) {
      uint32_t at = base[d];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w][d];
        count[w][d] = at;
        at += c;
      }
      base[d] = at;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const int64_t i = mine + j * 32;
      if (i >= end) continue;
      const uint32_t at = count[warp][(key[j] >> a.shift) & (a.bins - 1)] + rank[j];
      a.keys_out[at] = key[j];
      a.values_out[at] = a.first ? static_cast<uint32_t>(i) : a.values_in[i];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// Sums over the sorted tokens
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 64;        // sorted tokens per chunk sum
constexpr int kLongRun = 2 * kChunk;  // runs of at least this many tokens contain a whole chunk and are added by a CTA

struct SumArgs {
  const void* grad;
  int64_t grad_stride;
  const uint32_t* keys;    // sorted
  const uint32_t* tokens;  // their positions
  int2* runs;              // [vocab] first and one-past-last sorted index of a row's tokens
  float* chunk_sums;       // [n / kChunk][hidden]
  void* out;
  int64_t n, vocab;
  int hidden;
  float scale;
  int accumulate;
  int units, tiles;        // VEC-element units per row; tiles of 32 * VPL units
};

// acc += grad rows tokens[s], tokens[s + step], ... below e, in that order; the lane's units are u0 + 32 k.
template <int DT, int VEC, int VPL>
__device__ __forceinline__ void add_tokens(const SumArgs& a, int u0, int64_t s, int64_t e, int64_t step,
                                           float (&acc)[VPL][VEC]) {
  for (int64_t j = s; j < e; j += step) {
    const int64_t row = static_cast<int64_t>(a.tokens[j]) * a.grad_stride;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int u = u0 + 32 * k;
      if (u >= a.units) continue;
      float f[VEC];
      load_floats<DT, VEC>(a.grad, row + static_cast<int64_t>(u) * VEC, f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[k][i] += f[i];
    }
  }
}

template <int DTO, int VEC, int VPL>
__device__ __forceinline__ void write_row(const SumArgs& a, int64_t row, int u0, float (&acc)[VPL][VEC]) {
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int u = u0 + 32 * k;
    if (u >= a.units) continue;
    const int64_t at = row * a.hidden + static_cast<int64_t>(u) * VEC;
    float f[VEC];
    if (a.accumulate) {
      load_floats_plain<DTO, VEC>(a.out, at, f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = __fmaf_rn(a.scale, acc[k][i], f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = __fmul_rn(a.scale, acc[k][i]);
    }
    store_floats<DTO, VEC>(a.out, at, f);
  }
}

// Marks where the run of every id begins and ends, and adds up the chunks that one id fills.
template <int DT, int VEC, int VPL>
__global__ void __launch_bounds__(256) chunk_sums_kernel(const SumArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = me; i < a.n; i += threads) {
    const uint32_t key = a.keys[i];
    if (key >= a.vocab) continue;
    if (i == 0 || a.keys[i - 1] != key) a.runs[key].x = static_cast<int>(i);
    if (i + 1 == a.n || a.keys[i + 1] != key) a.runs[key].y = static_cast<int>(i + 1);
  }
  const int64_t n_items = a.n / kChunk * a.tiles;
  for (int64_t item = me >> 5; item < n_items; item += threads >> 5) {
    const int64_t c = item / a.tiles;
    const uint32_t key = a.keys[c * kChunk];
    if (key >= a.vocab || a.keys[c * kChunk + kChunk - 1] != key) continue;
    const int u0 = static_cast<int>(item - c * a.tiles) * 32 * VPL + lane;
    float acc[VPL][VEC] = {};
    add_tokens<DT, VEC, VPL>(a, u0, c * kChunk, (c + 1) * kChunk, 1, acc);
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int u = u0 + 32 * k;
      if (u >= a.units) continue;
      float* p = a.chunk_sums + c * a.hidden + static_cast<int64_t>(u) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = acc[k][i];
    }
  }
}

// Blocks [0, long_blocks): a CTA per (chunk, tile); it acts where the chunk is the first to begin inside a long
// run.  The other blocks: a warp per (row, tile) -- rows are the table's, or with `accumulate` the sorted
// positions at which a run begins.
template <int DT, int DTO, int VEC, int VPL>
__global__ void __launch_bounds__(256) row_sums_kernel(const SumArgs a, unsigned long_blocks) {
  __shared__ float part[8][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < long_blocks) {
    const int64_t n_long = a.n / kChunk * a.tiles;
    for (int64_t item = blockIdx.x; item < n_long; item += long_blocks) {
      const int64_t c = item / a.tiles;
      const uint32_t key = a.keys[c * kChunk];
      if (key >= a.vocab) continue;
      const int2 run = a.runs[key];
      if (run.y - run.x < kLongRun || (run.x + kChunk - 1) / kChunk != c) continue;
      const int u0 = static_cast<int>(item - c * a.tiles) * 32 * VPL + lane;
      const int64_t last = run.y / kChunk;  // chunks [c, last) are whole
      float acc[VPL][VEC] = {};
      add_tokens<DT, VEC, VPL>(a, u0, run.x + warp, c * kChunk, 8, acc);
      for (int64_t p = c + warp; p < last; p += 8) {
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
          const int u = u0 + 32 * k;
          if (u >= a.units) continue;
          const float* q = a.chunk_sums + p * a.hidden + static_cast<int64_t>(u) * VEC;
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[k][i] += q[i];
        }
      }
      add_tokens<DT, VEC, VPL>(a, u0, last * kChunk + warp, run.y, 8, acc);
      // the warps' parts, one unit per lane at a time
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[warp][i * 32 + lane] = acc[k][i];
        __syncthreads();
        if (warp == 0) {
          for (int w = 1; w < 8; ++w)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[k][i] += part[w][i * 32 + lane];
        }
      }
      if (warp == 0) write_row<DTO, VEC, VPL>(a, key, u0, acc);
    }
    return;
  }
  const int64_t n_warps = static_cast<int64_t>(gridDim.x - long_blocks) * 8;
  const int64_t n_items = (a.accumulate ? a.n : a.vocab) * a.tiles;
  for (int64_t item = static_cast<int64_t>(blockIdx.x - long_blocks) * 8 + warp; item < n_items; item += n_warps) {
    const int64_t at = item / a.tiles;
    const int u0 = static_cast<int>(item - at * a.tiles) * 32 * VPL + lane;
    int64_t row = at;
    if (a.accumulate) {
      row = a.keys[at];
      if (row >= a.vocab || (at > 0 && a.keys[at - 1] == row)) continue;
    }
    const int2 run = a.runs[row];
    if (run.y - run.x >= kLongRun) continue;
    float acc[VPL][VEC] = {};
    add_tokens<DT, VEC, VPL>(a, u0, run.x, run.y, 1, acc);
    write_row<DTO, VEC, VPL>(a, row, u0, acc);
  }
}

int64_t round16(int64_t bytes) { return (bytes + 15) & ~int64_t(15); }

struct Workspace {
  uint32_t *keys[2], *values[2], *counts;
  int2* runs;
  float* chunk_sums;
  int64_t bytes;
};

Workspace lay_out(void* base, int64_t vocab, int hidden, int64_t n) {
  Workspace w{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    unsigned char* p = static_cast<unsigned char*>(base) + at;
    at += round16(bytes);
    return p;
  };
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = reinterpret_cast<uint32_t*>(take(n * 4));
    w.values[i] = reinterpret_cast<uint32_t*>(take(n * 4));
  }
  w.counts = reinterpret_cast<uint32_t*>(take(int64_t(kSortMaxCtas) * kSortMaxBins * 4));
  w.runs = reinterpret_cast<int2*>(take(vocab * 8));
  w.chunk_sums = reinterpret_cast<float*>(take(n / kChunk * hidden * 4));
  w.bytes = at;
  return w;
}

// Sorts (id, position) into w.keys[0] / w.values[0] or [1]; returns which.
cudaError_t sort_tokens(const TableGradArgs& a, const Workspace& w, int* where, cudaStream_t stream) {
  int bits = 1;
  while ((int64_t(1) << bits) <= a.vocab) ++bits;  // keys go up to vocab
  const int passes = (bits + kSortMaxBits - 1) / kSortMaxBits;
  const int width = (bits + passes - 1) / passes;
  int64_t ctas = (a.n_ids + kSortTile - 1) / kSortTile;
  if (ctas > kSortMaxCtas) ctas = kSortMaxCtas;
  SortArgs s{};
  s.ids = a.ids;
  s.counts = w.counts;
  s.n = a.n_ids;
  s.vocab = a.vocab;
  s.padding_id = a.padding_id;
  s.id_dtype = a.id_dtype;
  s.status = a.status;
  s.bins = 1 << width;
  const int64_t tiles = (a.n_ids + kSortTile - 1) / kSortTile;
  s.span = (tiles + ctas - 1) / ctas * kSortTile;
  const unsigned grid = static_cast<unsigned>((a.n_ids + s.span - 1) / s.span);
  for (int p = 0; p < passes; ++p) {
    s.first = p == 0;
    s.runs = p == 0 && !a.accumulate ? w.runs : nullptr;
    s.keys_in = w.keys[(p + 1) & 1];
    s.values_in = w.values[(p + 1) & 1];
    s.keys_out = w.keys[p & 1];
    s.values_out = w.values[p & 1];
    s.shift = p * width;
    sort_count_kernel<<<grid, kSortThreads, 0, stream>>>(s);
    sort_move_kernel<<<grid, kSortThreads, 0, stream>>>(s);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  *where = (passes - 1) & 1;
  return cudaSuccess;
}

template <int DT, int DTO, int VEC, int VPL>
cudaError_t launch_sums(const TableGradArgs& a, const Workspace& w, int where, cudaStream_t stream) {
  SumArgs s{};
  s.grad = a.grad;
  s.grad_stride = a.grad_stride;
  s.keys = w.keys[where];
  s.tokens = w.values[where];
  s.runs = w.runs;
  s.chunk_sums = w.chunk_sums;
  s.out = a.out;
  s.n = a.n_ids;
  s.vocab = a.vocab;
  s.hidden = a.hidden;
  s.scale = a.scale;
  s.accumulate = a.accumulate;
  s.units = a.hidden / VEC;
  s.tiles = (s.units + 32 * VPL - 1) / (32 * VPL);
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  const int64_t chunk_items = a.n_ids / kChunk * s.tiles;
  int64_t grid = (chunk_items > a.n_ids / 32 ? chunk_items : a.n_ids / 32) / 8 + 1;
  if (grid > cap) grid = cap;
  chunk_sums_kernel<DT, VEC, VPL><<<static_cast<unsigned>(grid), 256, 0, stream>>>(s);
  const int64_t items = (a.accumulate ? a.n_ids : a.vocab) * s.tiles;
  grid = (items + 7) / 8;
  if (grid > cap) grid = cap;
  const int64_t long_blocks = chunk_items < 4 * cap ? chunk_items : 4 * cap;
  row_sums_kernel<DT, DTO, VEC, VPL>
      <<<static_cast<unsigned>(long_blocks + grid), 256, 0, stream>>>(s, static_cast<unsigned>(long_blocks));
  return cudaGetLastError();
}

template <int DT, int DTO>
cudaError_t launch_table_grad_t(const TableGradArgs& a, void* workspace, cudaStream_t stream) {
  const Workspace w = lay_out(workspace, a.vocab, a.hidden, a.n_ids);
  int where = 0;
  const cudaError_t e = sort_tokens(a, w, &where, stream);
  if (e != cudaSuccess || a.vocab == 0) return e;
  constexpr int kPV = Elem<DT>::kPerVec;
  if (a.hidden % kPV == 0 && a.grad_stride % kPV == 0 && aligned_to(a.grad, 16) && aligned_to(a.out, 16))
    return launch_sums<DT, DTO, kPV, 1>(a, w, where, stream);
  return launch_sums<DT, DTO, 1, 1>(a, w, where, stream);
}

}  // namespace

cudaError_t launch_embedding_scaled(int dtype, const ScaledLookupArgs& a, cudaStream_t stream) {
  if (a.n_ids == 0 || a.hidden == 0) return cudaSuccess;
  switch (dtype) {
    case kDtF32: return launch_scaled_lookup_dt<kDtF32>(a, stream);
    case kDtF16: return launch_scaled_lookup_dt<kDtF16>(a, stream);
    default: return launch_scaled_lookup_dt<kDtBF16>(a, stream);
  }
}

int64_t table_grad_workspace(int64_t vocab, int hidden, int64_t n_ids) { return lay_out(nullptr, vocab, hidden, n_ids).bytes; }

cudaError_t launch_table_grad(int dtype, int out_dtype, const TableGradArgs& a, void* workspace, cudaStream_t stream) {
  if (a.hidden == 0) return cudaSuccess;
  if (a.n_ids == 0) {
    if (a.accumulate || a.vocab == 0) return cudaSuccess;
    return cudaMemsetAsync(a.out, 0, static_cast<size_t>(a.vocab) * a.hidden * (out_dtype == kDtF32 ? 4 : 2), stream);
  }
  if (dtype == kDtF32) return launch_table_grad_t<kDtF32, kDtF32>(a, workspace, stream);
  if (dtype == kDtF16)
    return out_dtype == kDtF32 ? launch_table_grad_t<kDtF16, kDtF32>(a, workspace, stream)
                               : launch_table_grad_t<kDtF16, kDtF16>(a, workspace, stream);
  return out_dtype == kDtF32 ? launch_table_grad_t<kDtBF16, kDtF32>(a, workspace, stream)
                             : launch_table_grad_t<kDtBF16, kDtBF16>(a, workspace, stream);
}

}  // namespace cb200
