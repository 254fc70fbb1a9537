// The scaled lookup and the gradient of the embedding table.
//
// Gradient: out[v] = scale * sum of grad[i] over the tokens i with ids[i] == v.  The tokens are sorted by id
// (stable radix sort of (id, position) pairs), so each table row owns a contiguous run of the sorted list and
// its sum has a fixed order: no floating-point atomics, equal inputs give equal bits.  Then
//   - chunk_sums_kernel adds up every aligned chunk of 32 sorted tokens that belongs to one id: text is skewed
//     (the hottest id of 65536 tokens has thousands) and this is what spreads a long run over the GPU;
//   - row_sums_kernel writes the table rows.  Work is cut by tokens, not by rows, since a few rows of a text's table
//     have most of its tokens: a warp adds the runs that begin at a few neighbouring sorted positions, a CTA a
//     long run (the chunk sums and the ends that do not fill a chunk).
// The rows without tokens are filled with zeros beside the sort, whose few CTAs leave the memory idle.
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
// Rows without tokens
// ---------------------------------------------------------------------------------------------
constexpr int kZeroRows = 8;  // rows per warp and visit; divides 32

struct ZeroFill {
  unsigned char* out;  // the table's gradient
  int64_t row_bytes;
  int64_t begin, end;  // rows that this launch looks after
  int vectors;         // whether rows are whole, aligned 16-byte vectors
};

// A warp writes zeros to the rows v0 + k of the set bits k of `rows`.
__device__ __forceinline__ void fill_rows(const ZeroFill& z, int64_t v0, unsigned rows) {
  const int lane = threadIdx.x & 31;
  for (; rows != 0; rows &= rows - 1) {
    unsigned char* row = z.out + (v0 + __ffs(rows) - 1) * z.row_bytes;
    if (z.vectors) {
#pragma unroll 4
      for (int64_t i = lane; i < z.row_bytes / 16; i += 32) stg_stream(reinterpret_cast<uint4*>(row) + i, make_uint4(0, 0, 0, 0));
    } else {  // elements of 2 or 4 bytes
      for (int64_t i = lane; i < z.row_bytes / 2; i += 32) reinterpret_cast<uint16_t*>(row)[i] = 0;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Stable radix sort of (id, position), digits of at most 9 bits.  Tokens that contribute nothing (bad ids, padding)
// get the key `vocab` and end up behind all rows.
//   up to 4096 tokens: one CTA does every digit in shared memory;
//   more: one launch counts the first digit per CTA, then one launch per digit moves the keys: every CTA derives
//   from all the counts where its keys of each digit go, and counts the next digit for the CTA that will read them.
// A CTA takes a contiguous span of keys in tiles of 2048.
// ---------------------------------------------------------------------------------------------
constexpr int kSortItems = 4;
constexpr int kSortThreads = 512;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kSmallThreads = 1024;
constexpr int kSmallMax = kSmallThreads * kSortItems;
constexpr int kSortMaxBits = 9;
constexpr int kSortMaxBins = 1 << kSortMaxBits;
constexpr int kSortMaxCtas = 512;

struct SortArgs {
  const void* ids;           // first digit: the caller's ids
  const uint32_t* keys_in;   // later digits
  const uint32_t* values_in;
  uint32_t* keys_out;
  uint32_t* values_out;
  uint32_t* counts;          // [ctas][bins] of this digit
  uint32_t* next_counts;     // of the next one; NULL at the last
  uint32_t* long_runs;       // their number is cleared by the sort's first launch
  unsigned char* present;    // fresh gradient: [vocab] zeros, set to 1 by the count launch where an id points
  ZeroFill zero;             // what the launch's blocks behind the sorting ones fill
  unsigned sort_blocks;
  int64_t n, vocab, padding_id;
  int id_dtype;
  cb200_status* status;
  int64_t span;              // keys per CTA, a multiple of kSortTile
  int shift, width, passes;  // digit position and bits; digits in all
  int first;
};

__device__ __forceinline__ uint32_t key_of_id(const SortArgs& a, int64_t i, bool report) {
  const uint64_t id = read_id(a.ids, a.id_dtype, i);
  if (id >= static_cast<uint64_t>(a.vocab)) {
    if (report) report_status(a.status, CB200_STATUS_INVALID_INDEX, i, static_cast<int64_t>(id), a.vocab);
    return static_cast<uint32_t>(a.vocab);
  }
  return static_cast<int64_t>(id) == a.padding_id ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

// Exclusive sum over the CTA's threads; `totals` holds one word per warp.
__device__ __forceinline__ uint32_t exclusive_scan(uint32_t own, uint32_t* totals) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t v = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += up;
  }
  if (lane == 31) totals[warp] = v;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warps; ++w) before += w < warp ? totals[w] : 0u;
  return before + v - own;
}

// Ranks of a warp's keys among the warp's keys of the same digit, in the order of the keys (item j of lane l is key
// 32 j + l); count[digit] ends as their number.  The lanes with an equal digit are found by one ballot per bit: the
// match instruction takes a time that grows with the number of different digits.
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[kSortItems], const bool (&live)[kSortItems],
                                           uint32_t (&rank)[kSortItems], uint16_t* count, int width) {
  const int lane = threadIdx.x & 31;
  unsigned peers[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    peers[j] = __ballot_sync(0xFFFFFFFFu, live[j]);
    for (int bit = 0; bit < width; ++bit) {
      const bool set = (digit[j] >> bit) & 1u;
      const unsigned with = __ballot_sync(0xFFFFFFFFu, set);
      peers[j] &= set ? with : ~with;
    }
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const unsigned below = peers[j] & ((1u << lane) - 1u);
    rank[j] = live[j] ? count[digit[j]] + __popc(below) : 0u;
    __syncwarp();
    if (live[j] && below == 0) count[digit[j]] = static_cast<uint16_t>(count[digit[j]] + __popc(peers[j]));
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t hist[kSortMaxBins];
  const int bins = 1 << a.width;
  if (threadIdx.x < bins) hist[threadIdx.x] = 0;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) a.long_runs[0] = 0;
  const int64_t begin = blockIdx.x * a.span;
  const int64_t end = begin + a.span < a.n ? begin + a.span : a.n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
    const uint32_t key = key_of_id(a, i, true);
    atomicAdd(&hist[key & (bins - 1)], 1u);
    if (a.present != nullptr && key < a.vocab) a.present[key] = 1;
  }
  __syncthreads();
  if (threadIdx.x < bins) {
    a.counts[static_cast<int64_t>(blockIdx.x) * bins + threadIdx.x] = hist[threadIdx.x];
    if (a.next_counts != nullptr) a.next_counts[static_cast<int64_t>(blockIdx.x) * bins + threadIdx.x] = 0;
  }
}

// Blocks [0, sort_blocks) move the keys of one digit; the others fill rows without tokens meanwhile, which the sort
// leaves the memory free for.
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const SortArgs a) {
  if (blockIdx.x >= a.sort_blocks) {
    const int64_t warps = static_cast<int64_t>(gridDim.x - a.sort_blocks) * (kSortThreads / 32);
    for (int64_t v0 = a.zero.begin + (static_cast<int64_t>(blockIdx.x - a.sort_blocks) * (kSortThreads / 32) + (threadIdx.x >> 5)) * kZeroRows;
         v0 < a.zero.end; v0 += warps * kZeroRows) {
      const int64_t v = v0 + (threadIdx.x & 31);
      const bool empty = (threadIdx.x & 31) < kZeroRows && v < a.zero.end && a.present[v] == 0;
      fill_rows(a.zero, v0, __ballot_sync(0xFFFFFFFFu, empty));
    }
    return;
  }
  __shared__ uint32_t base[kSortMaxBins];
  __shared__ uint32_t totals[kSortThreads / 32];
  __shared__ uint16_t count[kSortThreads / 32][kSortMaxBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << a.width;

  // first slot of this CTA's keys of digit d: all smaller digits, and this digit in the CTAs before
  uint32_t total = 0, before = 0;
  if (threadIdx.x < bins) {
#pragma unroll 16
    for (unsigned t = 0; t < a.sort_blocks; ++t) {
      const uint32_t c = a.counts[static_cast<int64_t>(t) * bins + threadIdx.x];
      before += t < blockIdx.x ? c : 0u;
      total += c;
    }
  }
  before += exclusive_scan(total, totals);
  base[threadIdx.x] = before;

  const int64_t begin = blockIdx.x * a.span;
  const int64_t end = begin + a.span < a.n ? begin + a.span : a.n;
  for (int64_t tile = begin; tile < end; tile += kSortTile) {
    uint32_t* zero = reinterpret_cast<uint32_t*>(&count[0][0]);
#pragma unroll
    for (int k = 0; k < kSortThreads / 32 * kSortMaxBins / 2 / kSortThreads; ++k) zero[k * kSortThreads + threadIdx.x] = 0;
    uint32_t key[kSortItems], value[kSortItems], digit[kSortItems], rank[kSortItems];
    bool live[kSortItems];
    const int64_t mine = tile + warp * (32 * kSortItems) + lane;
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const int64_t i = mine + j * 32;
      live[j] = i < end;
      key[j] = !live[j] ? 0u : a.first ? key_of_id(a, i, false) : a.keys_in[i];
      value[j] = !live[j] ? 0u : a.first ? static_cast<uint32_t>(i) : a.values_in[i];
      digit[j] = (key[j] >> a.shift) & (bins - 1);
    }
    __syncthreads();
    warp_ranks(digit, live, rank, count[warp], a.width);
    __syncthreads();
    {
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < kSortThreads / 32; ++w) {
        const uint32_t c = count[w][threadIdx.x];
        count[w][threadIdx.x] = static_cast<uint16_t>(sum);
        sum += c;
      }
      total = sum;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      if (!live[j]) continue;
      const uint32_t at = base[digit[j]] + count[warp][digit[j]] + rank[j];
      a.keys_out[at] = key[j];
      a.values_out[at] = value[j];
      if (a.next_counts != nullptr)
        atomicAdd(&a.next_counts[at / a.span * bins + ((key[j] >> (a.shift + a.width)) & (bins - 1))], 1u);
    }
    __syncthreads();
    base[threadIdx.x] += total;
  }
}

// Block 0 sorts up to kSmallMax tokens.  The others fill the rows without tokens: each takes an equal share of the
// table's rows, marks in shared memory which of them the ids name, and writes zeros to the rest.
constexpr int kMarkWords = 4096;  // rows marked at a time: 32 per word
constexpr int kSmallSmem = (2 * kSmallMax + kSortMaxBins + kSmallThreads / 32) * 4 + kSmallThreads / 32 * kSortMaxBins * 2;
static_assert(kMarkWords * 4 <= kSmallSmem, "the marks fit");

__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(const SortArgs a) {
  extern __shared__ uint32_t pairs[];  // [keys | values][kSmallMax], then what the digits need
  if (blockIdx.x > 0) {
    const int64_t shares = gridDim.x - 1, share = blockIdx.x - 1;
    const int64_t begin = a.vocab * share / shares, end = a.vocab * (share + 1) / shares;
    for (int64_t from = begin; from < end; from += kMarkWords * 32) {
      const int64_t to = from + kMarkWords * 32 < end ? from + kMarkWords * 32 : end;
      const int words = static_cast<int>((to - from + 31) / 32);
      for (int w = threadIdx.x; w < words; w += kSmallThreads) pairs[w] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < a.n; i += kSmallThreads) {
        const int64_t key = key_of_id(a, i, false);
        if (key >= from && key < to) atomicOr(&pairs[(key - from) >> 5], 1u << ((key - from) & 31));
      }
      __syncthreads();
      const int rows = static_cast<int>(to - from);
      for (int r = (threadIdx.x >> 5) * kZeroRows; r < rows; r += kSmallThreads / 32 * kZeroRows) {
        const unsigned inside = rows - r < kZeroRows ? (1u << (rows - r)) - 1u : (1u << kZeroRows) - 1u;
        fill_rows(a.zero, from + r, ~(pairs[r >> 5] >> (r & 31)) & inside);
      }
      __syncthreads();
    }
    return;
  }
  uint32_t* base = pairs + 2 * kSmallMax;       // [kSortMaxBins]
  uint32_t* totals = base + kSortMaxBins;       // [warps]
  uint16_t(*count)[kSortMaxBins] = reinterpret_cast<uint16_t(*)[kSortMaxBins]>(totals + kSmallThreads / 32);  // [warps]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << a.width, n = static_cast<int>(a.n);
  if (threadIdx.x == 0) a.long_runs[0] = 0;
  const int mine = warp * (32 * kSortItems) + lane;
  uint32_t key[kSortItems], value[kSortItems], digit[kSortItems], rank[kSortItems];
  bool live[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = mine + j * 32;
    live[j] = i < n;
    key[j] = live[j] ? key_of_id(a, i, true) : 0u;
    value[j] = i;
  }
  for (int p = 0; p < a.passes; ++p) {
    uint32_t* zero = reinterpret_cast<uint32_t*>(&count[0][0]);
#pragma unroll
    for (int k = 0; k < kSmallThreads / 32 * kSortMaxBins / 2 / kSmallThreads; ++k) zero[k * kSmallThreads + threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) digit[j] = (key[j] >> (p * a.width)) & (bins - 1);
    warp_ranks(digit, live, rank, count[warp], a.width);
    __syncthreads();
    uint32_t sum = 0;
    if (threadIdx.x < bins) {
#pragma unroll
      for (int w = 0; w < kSmallThreads / 32; ++w) {
        const uint32_t c = count[w][threadIdx.x];
        count[w][threadIdx.x] = static_cast<uint16_t>(sum);
        sum += c;
      }
    }
    const uint32_t first = exclusive_scan(sum, totals);
    if (threadIdx.x < kSortMaxBins) base[threadIdx.x] = first;
    __syncthreads();
    const bool last = p + 1 == a.passes;
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      if (!live[j]) continue;
      const uint32_t at = base[digit[j]] + count[warp][digit[j]] + rank[j];
      (last ? a.keys_out : pairs)[at] = key[j];
      (last ? a.values_out : pairs + kSmallMax)[at] = value[j];
    }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      if (!live[j]) continue;
      key[j] = pairs[mine + j * 32];
      value[j] = pairs[kSmallMax + mine + j * 32];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Sums over the sorted tokens
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 32;            // sorted tokens per chunk sum
constexpr int kLongRun = 2 * kChunk;  // runs of at least this many tokens contain a whole chunk and are added by a CTA
constexpr int kMaxGroup = 16;         // sorted positions per warp and visit, at most

struct SumArgs {
  const void* grad;
  int64_t grad_stride;
  const uint32_t* keys;    // sorted
  const uint32_t* tokens;  // their positions
  int2* runs;              // [vocab] first and one-past-last sorted index of a row's tokens
  float* chunk_sums;       // [n / kChunk][hidden]
  uint32_t* long_runs;     // [0]: their number, then the ids that have one, in no particular order
  void* out;
  int64_t n, vocab;
  int hidden;
  float scale;
  int units;               // VEC-element units per row
  int chunk_tiles, tiles;  // tiles of units per row: of 32 for chunks and long runs, of 32 * kRowVecs for the others
  int group;               // sorted positions per warp and visit
  unsigned long_blocks;    // of row_sums_kernel, for the long runs
};
#ifndef RV
#define RV 1
#endif
#ifndef RB
#define RB 4
#endif
constexpr int kRowVecs = RV;    // units per lane of a row tile
constexpr int kRowBatch = RB;   // tokens whose loads are in flight together
constexpr int kChunkBatch = 8;

// One VEC-element unit as it lies in memory.
template <int DT, int VEC>
struct Unit {
  uint4 v;
};
template <int DT>
struct Unit<DT, 1> {
  float v;
};
template <int DT, int VEC>
__device__ __forceinline__ Unit<DT, VEC> load_unit(const void* base, int64_t elem) {
  Unit<DT, VEC> u;
  if constexpr (VEC == 1) u.v = load_elem<DT>(base, elem);
  else u.v = ldg_stream(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + elem * Elem<DT>::kBytes));
  return u;
}
template <int DT, int VEC>
__device__ __forceinline__ void add_unit(const Unit<DT, VEC>& u, float (&acc)[VEC]) {
  if constexpr (VEC == 1) {
    acc[0] += u.v;
  } else {
    float f[VEC];
    vec_to_floats<DT>(u.v, f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += f[i];
  }
}

// acc += grad rows of the tokens s, s + step, ... below e, in that order, for unit u of the row.
template <int DT, int VEC>
__device__ __forceinline__ void add_tokens(const SumArgs& a, int u, int64_t s, int64_t e, int64_t step, float (&acc)[VEC]) {
  for (; s < e; s += step * kChunkBatch) {
    Unit<DT, VEC> q[kChunkBatch];
    const int64_t left = (e - s + step - 1) / step;
    uint32_t token[kChunkBatch];
#pragma unroll
    for (int k = 0; k < kChunkBatch; ++k) token[k] = a.tokens[k < left ? s + k * step : s];
#pragma unroll
    for (int k = 0; k < kChunkBatch; ++k)
      if (k < left) q[k] = load_unit<DT, VEC>(a.grad, static_cast<int64_t>(token[k]) * a.grad_stride + static_cast<int64_t>(u) * VEC);
#pragma unroll
    for (int k = 0; k < kChunkBatch; ++k)
      if (k < left) add_unit<DT, VEC>(q[k], acc);
  }
}

// Unit u of a table row from its sum; `old` is what it holds, read only with ACC.
template <int DTO, int VEC, bool ACC>
__device__ __forceinline__ void write_unit(const SumArgs& a, int64_t row, int u, const float (&acc)[VEC], const float (&old)[VEC]) {
  float f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = ACC ? __fmaf_rn(a.scale, acc[i], old[i]) : __fmul_rn(a.scale, acc[i]);
  store_floats<DTO, VEC>(a.out, row * a.hidden + static_cast<int64_t>(u) * VEC, f);
}

// Marks where the run of every id begins and ends, and adds up the chunks that one id fills.
template <int DT, int VEC>
__global__ void __launch_bounds__(256) chunk_sums_kernel(const SumArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = me; i < a.n; i += threads) {
    const uint32_t key = a.keys[i];
    if (key >= a.vocab) continue;
    if (i == 0 || a.keys[i - 1] != key) {
      a.runs[key].x = static_cast<int>(i);
      if (i + kLongRun <= a.n && a.keys[i + kLongRun - 1] == key) a.long_runs[1 + atomicAdd(a.long_runs, 1u)] = key;
    }
    if (i + 1 == a.n || a.keys[i + 1] != key) a.runs[key].y = static_cast<int>(i + 1);
  }
  const int64_t n_items = a.n / kChunk * a.chunk_tiles;
  for (int64_t item = me >> 5; item < n_items; item += threads >> 5) {
    const int64_t c = item / a.chunk_tiles;
    const uint32_t key = a.keys[c * kChunk];
    if (key >= a.vocab || a.keys[c * kChunk + kChunk - 1] != key) continue;
    const int u = static_cast<int>(item - c * a.chunk_tiles) * 32 + lane;
    if (u >= a.units) continue;
    float acc[VEC] = {};
    add_tokens<DT, VEC>(a, u, c * kChunk, (c + 1) * kChunk, 1, acc);
    store_floats<kDtF32, VEC>(a.chunk_sums, c * a.hidden + static_cast<int64_t>(u) * VEC, acc);
  }
}

// A long run, by a CTA per tile of 32 units: its whole chunks and the tokens before and behind them, each warp every
// eighth, then the warps' parts in order.
template <int DT, int DTO, int VEC, bool ACC>
__device__ __noinline__ void add_long_run(const SumArgs& a, uint32_t key, int tile, float (*part)[32 * VEC]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int2 run = a.runs[key];
  const int u = tile * 32 + lane;
  const int64_t first = (run.x + kChunk - 1) / kChunk, last = run.y / kChunk;  // chunks [first, last) are whole
  float acc[VEC] = {};
  if (u < a.units) {
    add_tokens<DT, VEC>(a, u, run.x + warp, first * kChunk, 8, acc);
    for (int64_t p = first + warp; p < last; p += 8 * 4) {
      float f[4][VEC];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p + 8 * k < last)
          load_floats_plain<kDtF32, VEC>(a.chunk_sums, (p + 8 * k) * a.hidden + static_cast<int64_t>(u) * VEC, f[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p + 8 * k < last)
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += f[k][i];
    }
    add_tokens<DT, VEC>(a, u, last * kChunk + warp, run.y, 8, acc);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[warp][i * 32 + lane] = acc[i];
  __syncthreads();
  if (warp == 0 && u < a.units) {
    for (int w = 1; w < 8; ++w)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += part[w][i * 32 + lane];
    float old[VEC];
    if constexpr (ACC) load_floats_plain<DTO, VEC>(a.out, static_cast<int64_t>(key) * a.hidden + static_cast<int64_t>(u) * VEC, old);
    write_unit<DTO, VEC, ACC>(a, key, u, acc, old);
  }
  __syncthreads();
}

// Blocks [0, long_blocks): the long runs.  The others: a warp takes `group` sorted positions and a tile of columns
// and adds the runs that begin there -- one contiguous stretch of the sorted list (but for long runs), gone through
// in batches whose loads are in flight together, whatever the runs' lengths.
#ifndef TB
#define TB 4
#endif
#ifndef RMB
#define RMB 3
#endif
template <int DT, int DTO, int VEC, bool ACC>
__global__ void __launch_bounds__(256, RMB) row_sums_kernel(const SumArgs a) {
  __shared__ float part[8][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < a.long_blocks) {
    const int64_t n_items = static_cast<int64_t>(a.long_runs[0]) * a.chunk_tiles;
    for (int64_t item = blockIdx.x; item < n_items; item += a.long_blocks)
      add_long_run<DT, DTO, VEC, ACC>(a, a.long_runs[1 + item / a.chunk_tiles], static_cast<int>(item % a.chunk_tiles), part);
    return;
  }
  const int64_t n_items = (a.n + a.group - 1) / a.group * a.tiles;
  const int64_t n_warps = static_cast<int64_t>(gridDim.x - a.long_blocks) * 8;
  for (int64_t item = static_cast<int64_t>(blockIdx.x - a.long_blocks) * 8 + warp; item < n_items; item += n_warps) {
    const int64_t group = item / a.tiles;
    const int u0 = static_cast<int>(item - group * a.tiles) * (32 * kRowVecs) + lane;
    // lane l < group: the row, first sorted index and number of tokens of the run that begins at position l
    const int64_t mine = group * a.group + lane;
    uint32_t row = 0;
    int begin = 0, count = 0;
    if (lane < a.group && mine < a.n) {
      row = a.keys[mine];
      if (row < a.vocab && (mine == 0 || a.keys[mine - 1] != row)) {
        begin = static_cast<int>(mine);
        count = a.runs[row].y - begin;
        if (count >= kLongRun) count = 0;
      }
    }
    int before = count;  // tokens of the runs up to and with this lane's, then without
#pragma unroll
    for (int o = 1; o < kMaxGroup; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += up;
    }
    const int n_tokens = __shfl_sync(0xFFFFFFFFu, before, kMaxGroup - 1);
    before -= count;
    float acc[kRowVecs][VEC] = {};
    for (int w = 0; w < n_tokens; w += 32) {
      // lane l: token w + l of the stretch, and whose run it is in (the last one that starts at or before it)
      int of = 0;
#pragma unroll
      for (int o = kMaxGroup / 2; o > 0; o >>= 1) {
        const int start = __shfl_sync(0xFFFFFFFFu, before, of + o);
        if (start <= w + lane) of += o;
      }
      const int starts = __shfl_sync(0xFFFFFFFFu, before, of);
      const int from = __shfl_sync(0xFFFFFFFFu, begin, of) + (w + lane - starts);
      const uint32_t token = w + lane < n_tokens ? a.tokens[from] : 0u;
      const uint32_t of_row = __shfl_sync(0xFFFFFFFFu, row, of);
      // the tokens that are their run's last
      const unsigned ends = __ballot_sync(0xFFFFFFFFu, w + lane + 1 == starts + __shfl_sync(0xFFFFFFFFu, count, of));
      const int here = n_tokens - w < 32 ? n_tokens - w : 32;
      for (int t0 = 0; t0 < here; t0 += kRowBatch) {
        Unit<DT, VEC> q[kRowBatch][kRowVecs];
        float old[kRowBatch][kRowVecs][VEC];
#pragma unroll
        for (int t = 0; t < kRowBatch; ++t) {
          const int64_t at = static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, token, (t0 + t) & 31)) * a.grad_stride;
          const int64_t to = static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, of_row, (t0 + t) & 31)) * a.hidden;
#pragma unroll
          for (int k = 0; k < kRowVecs; ++k) {
            if (t0 + t >= here || u0 + 32 * k >= a.units) continue;
            q[t][k] = load_unit<DT, VEC>(a.grad, at + static_cast<int64_t>(u0 + 32 * k) * VEC);
            if constexpr (ACC)
              if ((ends >> (t0 + t)) & 1u) load_floats_plain<DTO, VEC>(a.out, to + static_cast<int64_t>(u0 + 32 * k) * VEC, old[t][k]);
          }
        }
#pragma unroll
        for (int t = 0; t < kRowBatch; ++t) {
          const uint32_t to = __shfl_sync(0xFFFFFFFFu, of_row, (t0 + t) & 31);
          if (t0 + t >= here) continue;
#pragma unroll
          for (int k = 0; k < kRowVecs; ++k) {
            if (u0 + 32 * k >= a.units) continue;
            add_unit<DT, VEC>(q[t][k], acc[k]);
            if ((ends >> (t0 + t)) & 1u) {
              write_unit<DTO, VEC, ACC>(a, to, u0 + 32 * k, acc[k], old[t][k]);
#pragma unroll
              for (int i = 0; i < VEC; ++i) acc[k][i] = 0.0f;
            }
          }
        }
      }
    }
  }
}

int64_t round16(int64_t bytes) { return (bytes + 15) & ~int64_t(15); }

struct Workspace {
  uint32_t *keys[2], *values[2], *counts[2];
  int2* runs;
  uint32_t* long_runs;
  unsigned char* present;
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
    w.counts[i] = reinterpret_cast<uint32_t*>(take(int64_t(kSortMaxCtas) * kSortMaxBins * 4));
  }
  w.runs = reinterpret_cast<int2*>(take(vocab * 8));
  w.long_runs = reinterpret_cast<uint32_t*>(take((1 + n / kLongRun) * 4));
  w.present = take(vocab);
  w.chunk_sums = reinterpret_cast<float*>(take(n / kChunk * hidden * 4));
  w.bytes = at;
  return w;
}

// Sorts (id, position) into w.keys[where] / w.values[where]; without `accumulate` also fills the rows without tokens.
cudaError_t sort_tokens(const TableGradArgs& a, const Workspace& w, int out_bytes, int* where, cudaStream_t stream) {
  int bits = 1;
  while ((int64_t(1) << bits) <= a.vocab) ++bits;  // keys go up to vocab
  SortArgs s{};
  s.ids = a.ids;
  s.n = a.n_ids;
  s.vocab = a.vocab;
  s.padding_id = a.padding_id;
  s.id_dtype = a.id_dtype;
  s.status = a.status;
  s.passes = (bits + kSortMaxBits - 1) / kSortMaxBits;
  s.width = (bits + s.passes - 1) / s.passes;
  s.long_runs = w.long_runs;
  s.zero.out = static_cast<unsigned char*>(a.out);
  s.zero.row_bytes = static_cast<int64_t>(a.hidden) * out_bytes;
  s.zero.vectors = s.zero.row_bytes % 16 == 0 && aligned_to(a.out, 16);
  const bool zero = !a.accumulate && a.vocab > 0;
  const int64_t sms = sm_count();
  *where = 0;
  if (a.n_ids <= kSmallMax) {
    const cudaError_t e = kernel_launch_config(reinterpret_cast<const void*>(sort_small_kernel), kSmallThreads, kSmallSmem, -1, nullptr);
    if (e != cudaSuccess) return e;
    s.keys_out = w.keys[0];
    s.values_out = w.values[0];
    const int64_t shares = !zero ? 0 : a.vocab < 2 * sms - 1 ? a.vocab : 2 * sms - 1;
    sort_small_kernel<<<static_cast<unsigned>(1 + shares), kSmallThreads, kSmallSmem, stream>>>(s);
    return cudaGetLastError();
  }
  const int64_t tiles = (a.n_ids + kSortTile - 1) / kSortTile;
  const int64_t ctas = tiles < kSortMaxCtas ? tiles : kSortMaxCtas;
  s.span = (tiles + ctas - 1) / ctas * kSortTile;
  s.sort_blocks = static_cast<unsigned>((a.n_ids + s.span - 1) / s.span);
  if (zero) {
    s.present = w.present;
    const cudaError_t e = cudaMemsetAsync(w.present, 0, static_cast<size_t>(a.vocab), stream);
    if (e != cudaSuccess) return e;
  }
  for (int p = 0; p < s.passes; ++p) {
    s.first = p == 0;
    s.keys_in = w.keys[(p + 1) & 1];
    s.values_in = w.values[(p + 1) & 1];
    s.keys_out = w.keys[p & 1];
    s.values_out = w.values[p & 1];
    s.counts = w.counts[p & 1];
    s.next_counts = p + 1 < s.passes ? w.counts[(p + 1) & 1] : nullptr;
    s.shift = p * s.width;
    if (p == 0) {
      sort_count_kernel<<<s.sort_blocks, kSortThreads, 0, stream>>>(s);
    } else if (s.next_counts != nullptr) {  // cleared by the count launch for the second digit only
      const cudaError_t e = cudaMemsetAsync(s.next_counts, 0, static_cast<size_t>(s.sort_blocks) * 4 << s.width, stream);
      if (e != cudaSuccess) return e;
    }
    // each digit's launch fills its share of the rows
    s.zero.begin = a.vocab * p / s.passes;
    s.zero.end = a.vocab * (p + 1) / s.passes;
    const int64_t wanted = (s.zero.end - s.zero.begin + kZeroRows * kSortThreads / 32 - 1) / (kZeroRows * kSortThreads / 32);
    const int64_t fillers = !zero ? 0 : wanted < 3 * sms ? wanted : 3 * sms;
    sort_move_kernel<<<static_cast<unsigned>(s.sort_blocks + fillers), kSortThreads, 0, stream>>>(s);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  *where = (s.passes - 1) & 1;
  return cudaSuccess;
}

template <int DT, int DTO, int VEC, bool ACC>
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
  s.units = a.hidden / VEC;
  s.long_runs = w.long_runs;
  s.chunk_tiles = (s.units + 31) / 32;
  s.tiles = (s.units + 32 * kRowVecs - 1) / (32 * kRowVecs);
  const int64_t sms = sm_count();
  const int64_t chunk_items = a.n_ids / kChunk * s.chunk_tiles;
  int64_t grid = (chunk_items > a.n_ids / 32 ? chunk_items : a.n_ids / 32) / 8 + 1;
  if (grid > sms * 6) grid = sms * 6;
  chunk_sums_kernel<DT, VEC><<<static_cast<unsigned>(grid), 256, 0, stream>>>(s);
  // fewer positions per warp where there would be too few warps to fill the GPU
  s.group = kMaxGroup;
  while (s.group > 1 && (a.n_ids + s.group - 1) / s.group * s.tiles < sms * 8 * RMB * 4) s.group /= 2;
  const int64_t items = (a.n_ids + s.group - 1) / s.group * s.tiles;
  const int64_t max_long = a.n_ids / kLongRun * s.chunk_tiles;
  s.long_blocks = static_cast<unsigned>(max_long < sms ? max_long : sms);
  const int64_t token_blocks = (items + 7) / 8 < sms * TB ? (items + 7) / 8 : sms * TB;
  row_sums_kernel<DT, DTO, VEC, ACC><<<static_cast<unsigned>(s.long_blocks + token_blocks), 256, 0, stream>>>(s);
  return cudaGetLastError();
}

template <int DT, int DTO, int VEC>
cudaError_t launch_sums(const TableGradArgs& a, const Workspace& w, int where, cudaStream_t stream) {
  return a.accumulate ? launch_sums<DT, DTO, VEC, true>(a, w, where, stream) : launch_sums<DT, DTO, VEC, false>(a, w, where, stream);
}

template <int DT, int DTO>
cudaError_t launch_table_grad_t(const TableGradArgs& a, void* workspace, cudaStream_t stream) {
  const Workspace w = lay_out(workspace, a.vocab, a.hidden, a.n_ids);
  int where = 0;
  const cudaError_t e = sort_tokens(a, w, Elem<DTO>::kBytes, &where, stream);
  if (e != cudaSuccess || a.vocab == 0) return e;
  constexpr int kPV = Elem<DT>::kPerVec;
  if (a.hidden % kPV == 0 && a.grad_stride % kPV == 0 && aligned_to(a.grad, 16) && aligned_to(a.out, 16))
    return launch_sums<DT, DTO, kPV>(a, w, where, stream);
  return launch_sums<DT, DTO, 1>(a, w, where, stream);
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
