// The scaled lookup and the gradient of the embedding table.
//
// Gradient: out[v] = scale * sum of grad[i] over the tokens i with ids[i] == v.  The tokens are sorted by id
// (stable, as (id, position) pairs), so each table row owns a contiguous run of the sorted list and its sum has a
// fixed order: no floating-point atomics, and equal inputs of equal alignment and strides give equal bits (alignment decides
// the width of the tiles, and the number of tiles whether a warp or a CTA adds a long run of up to 511 tokens).  Then
//   - chunk_sums_kernel adds up every aligned chunk of 32 sorted tokens that belongs to one id: text is skewed
//     (the hottest id of 65536 tokens has thousands) and this is what spreads a long run over the GPU;
//   - row_stream_kernel adds the runs.  A CTA per SM begins with the long ones (64 tokens and more: the ends that do not
//     fill a chunk, then their chunk sums), whose chains of dependent loads the other CTAs' traffic hides.  For the others
//     work is cut by tokens, not by rows, since a few rows of a text's table have most of its tokens: a warp takes the
//     runs that begin at a few neighbouring sorted positions.
// The rows without tokens are filled with zeros by further blocks of the launches that leave the memory idle: the radix
// sort's, or with few tokens the chunk sums' or the row sums'.
//
// Measured (B200): 65536 Zipf-distributed tokens, 128256 x 4096 bf16 (537 MB of gradients in, 1051 MB out): 295 us, 5.4 TB/s
// (the long runs in a launch of their own: 312); 4096 tokens added to a 32000 x 4096 f32 table (160 MB): 43 us; 46 tokens,
// 81761 x 2504 f32 (819 MB of zeros): 114 us.  Rows that are not whole, aligned 16-byte vectors go by elements: 16384 skewed tokens, 30000 x 4097
// bf16 182 us (4096 columns: 93), the lookup of 16384 such rows 67 us (44), of 2731 f32 columns 60 us.  Below some 8000 tokens the time is the latency of the three to four launches.
#include "launch.h"

namespace cb200 {

namespace {

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

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
// f = the unit's elements times `scale`, each rounded once in f32.
template <int DT, int VEC>
__device__ __forceinline__ void scale_unit(const Unit<DT, VEC>& u, float scale, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = u.v;
  else vec_to_floats<DT>(u.v, f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = __fmul_rn(f[i], scale);
}
// VEC consecutive elements <-> floats; VEC is the 16-byte vector's element count of one of the types, or 1 (any alignment).
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
// Scaled lookup: a warp per (token, tile of 32 U units), its loads in flight together.  Four units per lane whatever the
// number of rows: with one, which spreads few rows over more warps, 1 to 16 rows take the same time within 0.1 us, 592 rows of
// 4096 bf16 columns 3.7 us on the device instead of 3.3, 8192 rows 20.7 instead of 18.0.
// ---------------------------------------------------------------------------------------------
constexpr int kLookupUnits = 4;
template <int DT, int VEC>
__global__ void __launch_bounds__(256) scaled_lookup_kernel(const ScaledLookupArgs a, int units, int tiles) {
  constexpr int U = kLookupUnits;
  const int lane = threadIdx.x & 31;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int64_t n_items = a.n_ids * tiles;
  for (int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < n_items; item += n_warps) {
    const int64_t i = item / tiles;
    const int u0 = static_cast<int>(item - i * tiles) * (32 * U) + lane;
    const uint64_t id = read_id(a.ids, a.id_dtype, i);
    if (id >= static_cast<uint64_t>(a.vocab)) {
      if (u0 == 0) report_status(a.status, CB200_STATUS_INVALID_INDEX, i, static_cast<int64_t>(id), a.vocab);
      continue;
    }
    Unit<DT, VEC> q[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (u0 + 32 * k < units)
        q[k] = load_unit<DT, VEC>(a.table, static_cast<int64_t>(id) * a.hidden + static_cast<int64_t>(u0 + 32 * k) * VEC);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (u0 + 32 * k >= units) continue;
      float f[VEC];
      scale_unit<DT, VEC>(q[k], a.scale, f);
      store_floats<DT, VEC>(a.out, i * a.hidden + static_cast<int64_t>(u0 + 32 * k) * VEC, f);
    }
  }
}

template <int DT, int VEC>
cudaError_t launch_scaled_lookup_t(const ScaledLookupArgs& a, cudaStream_t stream) {
  const int units = a.hidden / VEC, tiles = (units + 32 * kLookupUnits - 1) / (32 * kLookupUnits);
  int64_t grid = (a.n_ids * tiles + 7) / 8;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  if (grid > cap) grid = cap;
  scaled_lookup_kernel<DT, VEC><<<static_cast<unsigned>(grid), 256, 0, stream>>>(a, units, tiles);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_scaled_lookup_dt(const ScaledLookupArgs& a, cudaStream_t stream) {
  constexpr int kPV = Elem<DT>::kPerVec;
  if (a.hidden % kPV != 0 || !aligned_to(a.table, 16) || !aligned_to(a.out, 16)) return launch_scaled_lookup_t<DT, 1>(a, stream);
  return launch_scaled_lookup_t<DT, kPV>(a, stream);
}

// The caller's ids.
struct Ids {
  const void* ids;
  int64_t n, vocab, padding_id;
  int id_dtype;
  cb200_status* status;
};

// Sorting key of token i: its id, or `vocab` for one that contributes nothing.
__device__ __forceinline__ uint32_t key_of_id(const Ids& a, int64_t i, bool report) {
  const uint64_t id = read_id(a.ids, a.id_dtype, i);
  if (id >= static_cast<uint64_t>(a.vocab)) {
    if (report) report_status(a.status, CB200_STATUS_INVALID_INDEX, i, static_cast<int64_t>(id), a.vocab);
    return static_cast<uint32_t>(a.vocab);
  }
  return static_cast<int64_t>(id) == a.padding_id ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

// ---------------------------------------------------------------------------------------------
// Rows without tokens.  A block fills a few neighbouring rows and ends: blocks that follow one another through memory
// write at 7.4 TB/s, resident ones that stride over the table at 6.0 (1 GB, rows of 8 KB).
// ---------------------------------------------------------------------------------------------
constexpr int kFillBytes = 64 * 1024;  // per block, but at least a row (16 KB: 60 us more for 0.9 GB, the launches of the blocks)

struct ZeroFill {
  unsigned char* out;      // the table's gradient
  int64_t row_bytes;
  int vectors;             // whether rows are whole, aligned 16-byte vectors
  unsigned char* present;  // [vocab] whether an id points at the row
  int64_t begin, end;      // rows that this launch looks after
  int rows;                // per block
  unsigned blocks;         // the launch's last blocks, which do
};

__device__ __forceinline__ void fill_rows(const ZeroFill& z, unsigned block) {
  const int64_t first = z.begin + static_cast<int64_t>(block) * z.rows;
  const int rows = static_cast<int>(z.end - first < z.rows ? z.end - first : z.rows);
  unsigned char* base = z.out + first * z.row_bytes;
  if (z.vectors) {
    const int64_t per_row = z.row_bytes / 16;
    if (rows == 1) {
      if (z.present[first] != 0) return;
      for (int64_t i = threadIdx.x; i < per_row; i += blockDim.x) stg_stream(reinterpret_cast<uint4*>(base) + i, make_uint4(0, 0, 0, 0));
      return;
    }
    const unsigned row_vectors = static_cast<unsigned>(per_row);  // several rows are at most kFillBytes
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < rows * row_vectors; i += blockDim.x)
      if (z.present[first + i / row_vectors] == 0) stg_stream(reinterpret_cast<uint4*>(base) + i, make_uint4(0, 0, 0, 0));
    return;
  }
  // a warp per row: vectors where it is aligned, elements of two bytes before and behind
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
    if (z.present[first + r] != 0) continue;
    uint16_t* from = reinterpret_cast<uint16_t*>(base + r * z.row_bytes);
    uint16_t* to = reinterpret_cast<uint16_t*>(base + (r + 1) * z.row_bytes);
    uint16_t* middle = reinterpret_cast<uint16_t*>((reinterpret_cast<uintptr_t>(from) + 15) & ~uintptr_t(15));
    uint16_t* behind = reinterpret_cast<uint16_t*>(reinterpret_cast<uintptr_t>(to) & ~uintptr_t(15));
    if (middle >= behind) middle = behind = to;  // shorter than two vectors: element by element
    for (uint16_t* p = from + lane; p < middle; p += 32) *p = 0;
    for (uint16_t* p = middle + 8 * lane; p < behind; p += 8 * 32) stg_stream(reinterpret_cast<uint4*>(p), make_uint4(0, 0, 0, 0));
    for (uint16_t* p = behind + lane; p < to; p += 32) *p = 0;
  }
}

// ---------------------------------------------------------------------------------------------
// Stable sort of (id, position).  Tokens that contribute nothing (bad ids, padding) get the key `vocab` and end up behind
// all rows.
//   up to 8192 tokens: one launch; a token's place is the number of tokens that sort before it, counted over all of
//   them by a CTA per 32 tokens (67 M comparisons at most, a few microseconds on the whole GPU);
//   more: radix sort, digits of at most 9 bits.  One launch counts the first digit per CTA, then one launch per digit
//   moves the keys: every CTA derives from all the counts where its keys of each digit go, and counts the next digit
//   for the CTA that will read them.  A CTA takes a contiguous span of keys in tiles of 2048.
// ---------------------------------------------------------------------------------------------
struct Counters {
  unsigned long long next_item;  // items of the row sums that warps took beyond their first
  uint32_t n_long;               // long runs listed
};

constexpr int kSortItems = 4;
constexpr int kSortThreads = 512;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kRankThreads = 256;
constexpr int kRankWarps = kRankThreads / 32;
constexpr int kRankMax = 8192;  // 2000 rows of 512 bf16 columns: 1024 skewed tokens 20.1 us (radix 27.6), 6000 39.8 (41.4), 8192 44.6 (43.3)
constexpr int kSortMaxBits = 9;
constexpr int kSortMaxBins = 1 << kSortMaxBits;
constexpr int kSortMaxCtas = 512;

struct SortArgs {
  Ids tokens;                // first digit: the keys come from here
  const uint32_t* keys_in;   // later digits
  const uint32_t* values_in;
  uint32_t* keys_out;
  uint32_t* values_out;
  uint32_t* counts;          // [ctas][bins] of this digit
  uint32_t* next_counts;     // of the next one; NULL at the last
  Counters* counters;        // cleared by the sort's first launch
  ZeroFill zero;
  unsigned sort_blocks;      // the first blocks; the zero-filling ones follow
  int64_t n;
  int64_t span;              // keys per CTA, a multiple of kSortTile
  int shift, width;          // digit position and bits
  int first;
};

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
  follow_previous();
  __shared__ uint32_t hist[kSortMaxBins];
  __shared__ uint32_t marked[kSortThreads];  // some id of each residue that was marked already, or none
  const int bins = 1 << a.width;
  if (threadIdx.x < bins) hist[threadIdx.x] = 0;
  marked[threadIdx.x] = 0xFFFFFFFFu;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.counters = Counters{};
  const int64_t begin = blockIdx.x * a.span;
  const int64_t end = begin + a.span < a.n ? begin + a.span : a.n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
    const uint32_t key = key_of_id(a.tokens, i, true);
    atomicAdd(&hist[key & (bins - 1)], 1u);
    // thousands of stores to a hot id's byte would queue up in one place
    if (a.zero.present != nullptr && key < a.tokens.vocab && marked[key % kSortThreads] != key) {
      marked[key % kSortThreads] = key;
      a.zero.present[key] = 1;
    }
  }
  __syncthreads();
  if (threadIdx.x < bins) {
    a.counts[static_cast<int64_t>(blockIdx.x) * bins + threadIdx.x] = hist[threadIdx.x];
    if (a.next_counts != nullptr) a.next_counts[static_cast<int64_t>(blockIdx.x) * bins + threadIdx.x] = 0;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const SortArgs a) {
  follow_previous();
  __shared__ uint32_t base[kSortMaxBins];
  __shared__ uint32_t totals[kSortThreads / 32];
  __shared__ uint16_t count[kSortThreads / 32][kSortMaxBins];
  if (blockIdx.x >= a.sort_blocks) return fill_rows(a.zero, blockIdx.x - a.sort_blocks);
  const unsigned block = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << a.width;

  // first slot of this CTA's keys of digit d: all smaller digits, and this digit in the CTAs before
  uint32_t total = 0, before = 0;
  if (threadIdx.x < bins) {
#pragma unroll 16
    for (unsigned t = 0; t < a.sort_blocks; ++t) {
      const uint32_t c = a.counts[static_cast<int64_t>(t) * bins + threadIdx.x];
      before += t < block ? c : 0u;
      total += c;
    }
  }
  before += exclusive_scan(total, totals);
  base[threadIdx.x] = before;

  const int64_t begin = block * a.span;
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
      key[j] = !live[j] ? 0u : a.first ? key_of_id(a.tokens, i, false) : a.keys_in[i];
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

// A block places 32 tokens.
__global__ void __launch_bounds__(kRankThreads) sort_small_kernel(const SortArgs a) {
  follow_previous();
  extern __shared__ __align__(16) uint32_t words[];
  __shared__ uint32_t part[kRankWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = static_cast<int>(a.n);
  const int first = static_cast<int>(blockIdx.x) * 32;  // this block's tokens
  if (first == 0 && threadIdx.x == 0) *a.counters = Counters{};
  const int padded = (n + 31) / 32 * 32;
#pragma unroll 8
  for (int i = threadIdx.x; i < padded; i += kRankThreads) words[i] = i < n ? key_of_id(a.tokens, i, false) : 0xFFFFFFFFu;
  if (threadIdx.x < 32 && first + threadIdx.x < n) {
    const uint32_t own = key_of_id(a.tokens, first + threadIdx.x, true);
    if (a.zero.present != nullptr && own < a.tokens.vocab) a.zero.present[own] = 1;
  }
  __syncthreads();
  // lane: one token; warp: every eighth group of four others.  A token before it sorts before it with an equal key.
  const uint32_t key = words[first + lane];
  uint32_t before = 0;
  const uint4* fours = reinterpret_cast<const uint4*>(words);
#pragma unroll 4
  for (int j = warp; j < first / 4; j += kRankWarps) {
    const uint4 k = fours[j];
    before += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
  }
#pragma unroll 4
  for (int j = first / 4 + 8 + warp; j < padded / 4; j += kRankWarps) {
    const uint4 k = fours[j];
    before += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
  }
  if (warp == 0)
    for (int l = 0; l < 32; ++l) before += l < lane ? words[first + l] <= key : words[first + l] < key;
  part[warp][lane] = before;
  __syncthreads();
  if (warp == 0 && first + lane < n) {
    for (int w = 1; w < kRankWarps; ++w) before += part[w][lane];
    a.keys_out[before] = key;
    a.values_out[before] = static_cast<uint32_t>(first + lane);
  }
}

// ---------------------------------------------------------------------------------------------
// Sums over the sorted tokens
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 32;            // sorted tokens per chunk sum
constexpr int kLongRun = 2 * kChunk;  // runs of at least this many tokens contain a whole chunk and are added apart from the others
constexpr int kMaxGroup = 16;         // sorted positions per warp and visit, at most: with kLongRun - 1 behind them fewer than 96

struct SumArgs {
  const void* grad;
  int64_t grad_stride;
  const uint32_t* keys;    // sorted
  const uint32_t* tokens;  // their positions
  float* chunk_sums;       // [n / kChunk][hidden]
  Counters* counters;
  uint2* long_runs;        // {one past its last sorted index, id} of each, in no particular order
  uint32_t* begins;        // [vocab] where the long runs begin; nothing for other ids
  void* out;
  int64_t n, vocab;
  int hidden;
  float scale;
  int units;               // VEC-element units per row
  int tiles;               // tiles of 32 units per row
  int group;               // sorted positions per warp and visit
  unsigned long_blocks;    // the launch's first blocks, which begin with the long runs
  int share;               // how the items of the row sums are shared out
  ZeroFill zero;
};
constexpr int kChunkBatch = 8;
constexpr int kTokenBatch = 8;
// Up to so many tokens a CTA adds even the longest run, token by token (at most 128 additions per warp, then the eight warps).
// The launch for the chunks keeps the additions in a row few and the longest run short; 4096 skewed tokens of 1000 columns
// over 2000 rows take 36.9 us with it and 38.4 without, 3001 32.6 and 31.9, 1024 25.4 and 21.3, 256 21.1 and 17.6.
constexpr int kDirectMax = 1024;

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

// Unit u of a table row from its sum; `old` is what it holds, read only with ACC.
template <int DTO, int VEC, bool ACC>
__device__ __forceinline__ void write_unit(const SumArgs& a, int64_t row, int u, const float (&acc)[VEC], const float (&old)[VEC]) {
  float f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = ACC ? __fmaf_rn(a.scale, acc[i], old[i]) : __fmul_rn(a.scale, acc[i]);
  store_floats<DTO, VEC>(a.out, row * a.hidden + static_cast<int64_t>(u) * VEC, f);
}

// Lists the long runs and adds up the chunks that one id fills: a warp per (chunk, tile of 32 C units), eight tokens' loads
// in flight.  Bound by memory: 288 MB of the skewed 65536 tokens of 4096 bf16 columns in 54 us.
template <int DT, int VEC, int C>
__global__ void __launch_bounds__(256) chunk_sums_kernel(const __grid_constant__ SumArgs a) {
  follow_previous();
  const unsigned blocks = gridDim.x - a.zero.blocks;
  if (blockIdx.x >= blocks) return fill_rows(a.zero, blockIdx.x - blocks);
  const int lane = threadIdx.x & 31;
  const int64_t threads = static_cast<int64_t>(blocks) * blockDim.x;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = me; i + kLongRun <= a.n; i += threads) {
    const uint32_t key = a.keys[i];
    if (key >= a.vocab || a.keys[i + kLongRun - 1] != key) continue;
    if (i == 0 || a.keys[i - 1] != key) a.begins[key] = static_cast<uint32_t>(i);
    const int64_t behind = i + kLongRun;  // of the 64 positions from i on
    if (behind == a.n || a.keys[behind] != key) a.long_runs[atomicAdd(&a.counters->n_long, 1u)] = make_uint2(static_cast<uint32_t>(behind), key);
  }
  const int tiles = (a.units + 32 * C - 1) / (32 * C);
  const int64_t n_items = a.n / kChunk * tiles;
  for (int64_t item = me >> 5; item < n_items; item += threads >> 5) {
    const int64_t c = item / tiles;
    const uint32_t key = a.keys[c * kChunk + lane], token = a.tokens[c * kChunk + lane];
    if (key >= a.vocab || !__all_sync(0xFFFFFFFFu, key == __shfl_sync(0xFFFFFFFFu, key, 0))) continue;
    const int u0 = static_cast<int>(item - c * tiles) * (32 * C) + lane;
    float acc[C][VEC] = {};
#pragma unroll
    for (int t0 = 0; t0 < kChunk; t0 += kChunkBatch) {
      Unit<DT, VEC> q[kChunkBatch][C];
#pragma unroll
      for (int t = 0; t < kChunkBatch; ++t) {
        const int64_t at = static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, token, t0 + t)) * a.grad_stride;
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (u0 + 32 * j < a.units) q[t][j] = load_unit<DT, VEC>(a.grad, at + static_cast<int64_t>(u0 + 32 * j) * VEC);
      }
#pragma unroll
      for (int t = 0; t < kChunkBatch; ++t)
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (u0 + 32 * j < a.units) add_unit<DT, VEC>(q[t][j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (u0 + 32 * j < a.units) store_floats<kDtF32, VEC>(a.chunk_sums, c * a.hidden + static_cast<int64_t>(u0 + 32 * j) * VEC, acc[j]);
  }
}

// One past the last sorted index of the run that holds index `at`: the keys behind it are searched 32 ways at a time.
__device__ __forceinline__ int64_t run_end(const SumArgs& a, int64_t at) {
  const uint32_t key = a.keys[at];
  const int lane = threadIdx.x & 31;
  int64_t lo = at, hi = a.n;  // keys[lo] == key; hi: behind the run, or the end
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t probe = lo + (lane + 1) * step;
    const unsigned in = __ballot_sync(0xFFFFFFFFu, probe < hi && a.keys[probe < hi ? probe : at] == key);
    const int inside = __popc(in);  // the probes are in order: the first `inside` of them are in the run
    if (lo + (inside + 1) * step < hi) hi = lo + (inside + 1) * step;
    lo += inside * step;
  }
  return hi;
}

// acc += every step-th piece of a long run [begin, end) from `piece` on, for the unit u of its row: the tokens before and
// behind the whole chunks (all tokens where there are no chunk sums), then the chunk sums.  The pieces come into `ring`, the
// lane's slots of shared memory, kPieces - 1 ahead.
constexpr int kPieces = 8;
template <int VEC>
struct PieceRing {
  static constexpr int kWords = VEC > 1 ? VEC / 4 : 0;  // 16-byte words per lane and slot: VEC floats of a chunk sum
};

template <int DT, int VEC>
__device__ __forceinline__ void add_pieces(const SumArgs& a, int64_t begin, int64_t end, int u, int64_t piece, int step,
                                           uint4* ring, float (&acc)[VEC]) {
  const int lane = threadIdx.x & 31;
  int64_t first = a.chunk_sums == nullptr ? 0 : (begin + kChunk - 1) / kChunk, last = a.chunk_sums == nullptr ? 0 : end / kChunk;
  if (first >= last) first = last = 0;
  const int64_t head = first < last ? first * kChunk - begin : end - begin, loose = first < last ? head + end - last * kChunk : head;
  const int64_t pieces = loose + last - first, count = piece < pieces ? (pieces - piece + step - 1) / step : 0;
  const bool here = u < a.units;
  uint32_t ahead = 0;  // lane l: position of the token that is piece number i - i % 32 + l of this warp
  auto positions = [&](int64_t i) {
    const int64_t e = piece + (i + lane) * step;
    ahead = e < loose ? a.tokens[e < head ? begin + e : last * kChunk + (e - head)] : 0u;
  };
  if constexpr (VEC == 1) {
    for (int64_t i = 0; i < count; ++i) {
      if (i % 32 == 0) positions(i);
      const int64_t e = piece + i * step;
      const int64_t token = __shfl_sync(0xFFFFFFFFu, ahead, static_cast<int>(i % 32));
      if (here) acc[0] += e < loose ? load_elem<DT>(a.grad, token * a.grad_stride + u) : a.chunk_sums[(first + e - loose) * a.hidden + u];
    }
  } else {
    constexpr int kWords = PieceRing<VEC>::kWords;
    for (int64_t i = 0; i < count + kPieces - 1; ++i) {
      if (i < count) {
        if (i % 32 == 0) positions(i);
        const int64_t e = piece + i * step;
        const int64_t token = __shfl_sync(0xFFFFFFFFu, ahead, static_cast<int>(i % 32));
        uint4* slot = ring + static_cast<int>(i % kPieces) * (kWords * 32);
        if (here && e < loose) {
          cp_async16(slot, static_cast<const unsigned char*>(a.grad) + (token * a.grad_stride + static_cast<int64_t>(u) * VEC) * Elem<DT>::kBytes);
        } else if (here) {
          const float* sums = a.chunk_sums + (first + e - loose) * a.hidden + static_cast<int64_t>(u) * VEC;
#pragma unroll
          for (int w = 0; w < kWords; ++w) cp_async16(slot + w * 32, sums + 4 * w);
        }
      }
      cp_async_commit();
      const int64_t done = i - (kPieces - 1);
      if (done < 0) continue;
      asm volatile("cp.async.wait_group %0;" ::"n"(kPieces - 1) : "memory");
      const uint4* slot = ring + static_cast<int>(done % kPieces) * (kWords * 32);
      if (here && piece + done * step < loose) {
        Unit<DT, VEC> q;
        q.v = slot[0];
        add_unit<DT, VEC>(q, acc);
      } else if (here) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const uint4 v = slot[w * 32];
          acc[4 * w] += __uint_as_float(v.x);
          acc[4 * w + 1] += __uint_as_float(v.y);
          acc[4 * w + 2] += __uint_as_float(v.z);
          acc[4 * w + 3] += __uint_as_float(v.w);
        }
      }
    }
    cp_async_wait_all();
  }
}

template <int DTO, int VEC, bool ACC>
__device__ __forceinline__ void finish_run(const SumArgs& a, uint32_t key, int u, const float (&acc)[VEC]) {
  if (u >= a.units) return;
  float old[VEC] = {};
  if constexpr (ACC) load_floats_plain<DTO, VEC>(a.out, static_cast<int64_t>(key) * a.hidden + static_cast<int64_t>(u) * VEC, old);
  write_unit<DTO, VEC, ACC>(a, key, u, acc, old);
}

// The long runs, by the launch's first long_blocks CTAs.  Bound by the latency of dependent loads (list, positions, rows).
// With chunk sums and many of them: eight (run, tile) items per CTA at a time, a warp for each run of fewer
// than kWarpRun tokens; the others take a CTA each, every warp every eighth piece, then the warps' sums in order.  The eight
// lie far apart in the list, so that the tiles of a hot run go to different CTAs (65536 tokens over 1000 rows of
// 8192: 343 us with neighbours, 284 so).  "Many" is beyond 12 items per CTA: below, one warp's chain of loads is what is
// waited for (2000 tokens over 10 rows of 64 columns: 27.8 us by warps, 18.5 by CTAs), above, the CTAs' barriers (40000 over
// 300 rows of 4096: 129 by warps, 160 by CTAs).  kWarpRun: 65536 tokens over 200 rows of 4096 151 us with 512, 175 with 256;
// no difference in text's skew.
constexpr int kWarpRun = 512;
template <int VEC>
constexpr size_t kLongShared = size_t(8) * 32 * VEC * 4 + size_t(8) * kPieces * PieceRing<VEC>::kWords * 32 * 16;
template <int DT, int DTO, int VEC, bool ACC>
__device__ __forceinline__ void long_runs(const SumArgs& a, unsigned char* shared) {
  const int blocks = a.long_blocks, block = static_cast<int>(blockIdx.x);
  float(*part)[32 * VEC] = reinterpret_cast<float(*)[32 * VEC]>(shared);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* ring = reinterpret_cast<uint4*>(shared + 8 * 32 * VEC * 4) + warp * (kPieces * PieceRing<VEC>::kWords * 32) + lane;
  auto by_cta = [&](int64_t begin, int64_t end, uint32_t key, int tile) {
    const int u = tile * 32 + lane;
    float acc[VEC] = {};
    add_pieces<DT, VEC>(a, begin, end, u, warp, 8, ring, acc);
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[warp][i * 32 + lane] = acc[i];
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < 8; ++w)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += part[w][i * 32 + lane];
      finish_run<DTO, VEC, ACC>(a, key, u, acc);
    }
    __syncthreads();
  };
  if (a.chunk_sums != nullptr) {
    const int64_t n_items = static_cast<int64_t>(a.counters->n_long) * a.tiles;
    const bool together = n_items > 12 * static_cast<int64_t>(blocks);
    const int64_t batches = together ? (n_items + 7) / 8 : n_items;  // batch b: the items b, b + batches, ...
    for (int64_t batch = block; batch < batches; batch += blocks) {
      if (together) {
        const int64_t mine = batch + warp * batches;
        bool big = false;
        if (mine < n_items) {
          const uint2 run = a.long_runs[mine / a.tiles];
          const int64_t begin = a.begins[run.y];
          big = run.x - begin >= kWarpRun;
          if (!big) {
            const int u = static_cast<int>(mine % a.tiles) * 32 + lane;
            float acc[VEC] = {};
            add_pieces<DT, VEC>(a, begin, run.x, u, 0, 1, ring, acc);
            finish_run<DTO, VEC, ACC>(a, run.y, u, acc);
          }
        }
        if (!__syncthreads_or(big)) continue;
      }
      for (int64_t item = batch; item < n_items; item += batches) {
        const uint2 run = a.long_runs[item / a.tiles];
        const int64_t begin = a.begins[run.y];
        if (!together || run.x - begin >= kWarpRun) by_cta(begin, run.x, run.y, static_cast<int>(item % a.tiles));
      }
    }
    return;
  }
  // no list: a long run holds a multiple of kLongRun, and the block of the first one takes it
  const int64_t n_items = (a.n + kLongRun - 1) / kLongRun * a.tiles;
  for (int64_t item = block; item < n_items; item += blocks) {
    const int64_t at = item / a.tiles * kLongRun;
    const uint32_t key = a.keys[at];
    if (key >= a.vocab || (at > 0 && a.keys[at - kLongRun] == key)) continue;
    int64_t begin = at;  // back to where the run begins, at most 63 positions
    for (int k = 0; k < 2; ++k) {
      const int64_t p = at - 1 - 32 * k - lane;
      const unsigned other = ~__ballot_sync(0xFFFFFFFFu, p >= 0 && a.keys[p >= 0 ? p : 0] == key);
      begin = at - 32 * k - (other ? __ffs(other) - 1 : 32);
      if (other) break;
    }
    if (begin + kLongRun <= a.n && a.keys[begin + kLongRun - 1] == key) by_cta(begin, run_end(a, begin), key, static_cast<int>(item % a.tiles));
  }
}

// The runs that begin in a group of sorted positions show in the keys of the positions themselves and of the 63 behind
// them: a window of 96 keys, three per lane.
struct Window {
  uint32_t key[3], token[3];
  uint32_t last;  // the key before the window
  __device__ __forceinline__ void load(const SumArgs& a, int64_t at) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int64_t i = at + 32 * k + lane;
      key[k] = i < a.n ? a.keys[i] : static_cast<uint32_t>(a.vocab);
      token[k] = i < a.n ? a.tokens[i] : 0u;
    }
    last = at > 0 && at < a.n ? a.keys[at - 1] : 0xFFFFFFFFu;
  }
  __device__ __forceinline__ uint32_t key_at(int p) const {
    return __shfl_sync(0xFFFFFFFFu, p < 32 ? key[0] : p < 64 ? key[1] : key[2], p & 31);
  }
  __device__ __forceinline__ uint32_t token_at(int p) const {
    return __shfl_sync(0xFFFFFFFFu, p < 32 ? token[0] : p < 64 ? token[1] : token[2], p & 31);
  }
};

// The tokens of those runs: positions [from, to) of the window, without a long run, which can only be the last one;
// bit p of heads: a run (or what is no row) begins at position p.
struct Stretch {
  unsigned heads[3];
  int from, to;
  __device__ __forceinline__ void find(const SumArgs& a, const Window& w) {
    const int lane = threadIdx.x & 31;
    uint32_t last = w.last;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, w.key[k], 1);
      heads[k] = __ballot_sync(0xFFFFFFFFu, w.key[k] != (lane == 0 ? last : up));
      last = __shfl_sync(0xFFFFFFFFu, w.key[k], 31);
    }
    from = to = 0;
    const unsigned mine = heads[0] & ((1u << a.group) - 1u) & __ballot_sync(0xFFFFFFFFu, w.key[0] < a.vocab);
    if (mine == 0) return;
    from = __ffs(mine) - 1;
    const int final = 31 - __clz(mine);
    const unsigned behind = heads[0] & ~((2u << final) - 1u);
    const int end = behind ? __ffs(behind) - 1 : heads[1] ? 32 + __ffs(heads[1]) - 1 : heads[2] ? 64 + __ffs(heads[2]) - 1 : 96;
    to = end - final < kLongRun ? end : final;
  }
  __device__ __forceinline__ bool last_of_run(int p) const {
    const int next = p + 1;
    return next == to || (((next < 32 ? heads[0] : next < 64 ? heads[1] : heads[2]) >> (next & 31)) & 1u);
  }
};

// The blocks of row_stream_kernel and its like: the ones that sum and the zero-filling ones take turns, as far as there are
// both, so that they share the SMs.  Whether this is a zero-filling one; `block` becomes its index among its kind.
__device__ __forceinline__ bool take_turns(const SumArgs& a, unsigned& block) {
  if (block < a.long_blocks) return false;
  const unsigned sums = gridDim.x - a.long_blocks - a.zero.blocks, both = sums < a.zero.blocks ? sums : a.zero.blocks;
  bool fill;
  block -= a.long_blocks;
  if (block < 2 * both) {
    fill = block & 1u;
    block >>= 1;
  } else {
    fill = both == sums;
    block -= both;
  }
  return fill;
}

// The items of a warp of the row sums.  The first is its own.  With `share` each then takes the next that nobody has,
// since runs differ in length and the blocks that began with the long runs come late (these take their first one so as
// well); without, it takes every so-manieth and those blocks none: few tokens make small items, and thousands of warps
// that count in one place at the same time wait for one another.
struct Items {
  unsigned long long claimed = 0;  // lane 0: the item after the current one, asked for an item ahead
  int64_t fixed, n_items;          // items that are somebody's own, all items
  __device__ __forceinline__ void claim(const SumArgs& a) {
    if ((threadIdx.x & 31) == 0 && fixed < n_items) claimed = atomicAdd(&a.counters->next_item, 1ull);
  }
  __device__ __forceinline__ int64_t next(const SumArgs& a, int64_t item) {
    if (!a.share) return item + fixed;
    item = fixed + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, claimed, 0));
    claim(a);
    return item;
  }
  __device__ __forceinline__ int64_t first(const SumArgs& a, int64_t n, unsigned block) {
    n_items = n;
    fixed = static_cast<int64_t>(gridDim.x - a.long_blocks - a.zero.blocks) * 8;
    if (a.share) claim(a);
    if (blockIdx.x < a.long_blocks) return a.share ? next(a, 0) : n;
    return static_cast<int64_t>(block) * 8 + (threadIdx.x >> 5);
  }
};

template <bool ACC, int V>
struct Ring {
  static constexpr int kDepth = (ACC ? 8 : 16) / V;
};
// zero.blocks of the blocks: rows without tokens.  In the others a warp takes `group` sorted positions and a tile of 32 V
// vectors and adds the runs that begin there, then the next such item: one stream of tokens, whatever the runs' lengths
// and the items' borders.  Each lane brings its V vectors of the next 15 / V tokens (7 / V with ACC) into its own slots of
// shared memory by asynchronous copies and reads back only what it copied itself, so nothing but the copies' own
// completion is waited for.  With ACC the warp also brings what the table holds, for a run's last token.
template <int DT, int DTO, bool ACC, int V>
__global__ void __launch_bounds__(256, ACC ? 2 : 3) row_stream_kernel(const __grid_constant__ SumArgs a) {
  follow_previous();
  constexpr int VEC = Elem<DT>::kPerVec, kOld = ACC ? VEC * Elem<DTO>::kBytes / 16 : 0, kSlot = V * (1 + kOld);  // 16-byte words
  extern __shared__ __align__(16) unsigned char shared[];
  unsigned block = blockIdx.x;
  if (take_turns(a, block)) return fill_rows(a.zero, block);
  if (blockIdx.x < a.long_blocks) {
    long_runs<DT, DTO, VEC, ACC>(a, shared);
    __syncthreads();  // the shared memory changes its use
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* ring = reinterpret_cast<uint4*>(shared) + warp * (Ring<ACC, V>::kDepth * kSlot * 32) + lane;  // [slot][word][lane]
  const int row_tiles = (a.units + 32 * V - 1) / (32 * V);
  const int64_t n_items = (a.n + a.group - 1) / a.group * row_tiles;

  Items items;
  int64_t item = items.first(a, n_items, block);  // the next one to be opened; its window is on the way
  Window ahead, now;
  Stretch s;
  s.from = s.to = 0;
  int p = 0, tile = 0;
  ahead.load(a, item < n_items ? item / row_tiles * a.group : a.n);
  uint32_t slot_row = 0, slot_end = 0, slot_tile = 0;  // lane k: of the token in slot k
  unsigned issued = 0, done = 0;

  auto issue = [&]() {
    while (p == s.to && item < n_items) {
      now = ahead;
      tile = static_cast<int>(item % row_tiles);
      item = items.next(a, item);
      ahead.load(a, item < n_items ? item / row_tiles * a.group : a.n);
      s.find(a, now);
      p = s.from;
    }
    if (p < s.to) {
      const uint32_t row = now.key_at(p), token = now.token_at(p);
      const bool end = s.last_of_run(p);
      const int slot = issued % Ring<ACC, V>::kDepth, u0 = tile * (32 * V) + lane;
      uint4* to = ring + slot * kSlot * 32;
      const unsigned char* from = static_cast<const unsigned char*>(a.grad) + (static_cast<int64_t>(token) * a.grad_stride + static_cast<int64_t>(u0) * VEC) * Elem<DT>::kBytes;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (u0 + 32 * k < a.units) cp_async16(to + k * 32, from + k * 512);
      if (ACC && end) {  // 16-byte words in the order of memory, not of the lanes that will use them
        const int u = tile * (32 * V);
        const unsigned char* old = static_cast<const unsigned char*>(a.out) + (static_cast<int64_t>(row) * a.hidden + static_cast<int64_t>(u) * VEC) * Elem<DTO>::kBytes;
#pragma unroll
        for (int k = 0; k < V * kOld; ++k)
          if (32 * k + lane < (a.units - u) * kOld) cp_async16(to + (V + k) * 32, old + (32 * k + lane) * 16);
      }
      if (lane == slot) {
        slot_row = row;
        slot_end = end;
        slot_tile = tile;
      }
      ++issued;
      ++p;
    }
    cp_async_commit();
  };

  float acc[V][VEC] = {};
#pragma unroll 1
  for (int k = 0; k < Ring<ACC, V>::kDepth - 1; ++k) issue();
  for (;;) {
    issue();
    if (done == issued) break;
    asm volatile("cp.async.wait_group %0;" ::"n"(Ring<ACC, V>::kDepth - 1) : "memory");
    const int slot = done % Ring<ACC, V>::kDepth;
    const uint32_t row = __shfl_sync(0xFFFFFFFFu, slot_row, slot), end = __shfl_sync(0xFFFFFFFFu, slot_end, slot);
    const int u0 = __shfl_sync(0xFFFFFFFFu, slot_tile, slot) * (32 * V) + lane;
    ++done;
    const uint4* from = ring + slot * kSlot * 32;
    if constexpr (ACC) __syncwarp();  // the other lanes' copies of what the table holds
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (u0 + 32 * k >= a.units) continue;
      Unit<DT, VEC> q;
      q.v = from[k * 32];
      add_unit<DT, VEC>(q, acc[k]);
      if (end) {
        float old[VEC] = {};
        if constexpr (ACC) {
          constexpr int kPV = Elem<DTO>::kPerVec;
#pragma unroll
          for (int o = 0; o < kOld; ++o) {
            float t[kPV];
            vec_to_floats<DTO>(from[(V + k * kOld) * 32 - lane + kOld * lane + o], t);
#pragma unroll
            for (int i = 0; i < kPV; ++i) old[o * kPV + i] = t[i];
          }
        }
        write_unit<DTO, VEC, ACC>(a, row, u0 + 32 * k, acc[k], old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[k][i] = 0.0f;
      }
    }
    if constexpr (ACC) __syncwarp();  // the slot's next copies are not the reading lanes' own
  }
}

// The same for rows that are not whole, aligned vectors: kAny elements per lane, a few tokens' loads in flight together.
constexpr int kAny = 4;
template <int DT, int DTO, bool ACC>
__global__ void __launch_bounds__(256, 3) row_sums_any_kernel(const __grid_constant__ SumArgs a) {
  follow_previous();
  extern __shared__ __align__(16) unsigned char shared[];
  unsigned block = blockIdx.x;
  if (take_turns(a, block)) return fill_rows(a.zero, block);
  if (blockIdx.x < a.long_blocks) long_runs<DT, DTO, 1, ACC>(a, shared);
  const int lane = threadIdx.x & 31;
  const int row_tiles = (a.units + 32 * kAny - 1) / (32 * kAny);
  const int64_t n_items = (a.n + a.group - 1) / a.group * row_tiles;
  Items items;
  for (int64_t item = items.first(a, n_items, block); item < n_items; item = items.next(a, item)) {
    const int64_t group = item / row_tiles;
    const int u0 = static_cast<int>(item - group * row_tiles) * (32 * kAny) + lane;
    Window w;
    Stretch s;
    w.load(a, group * a.group);
    s.find(a, w);
    float acc[kAny][1] = {};
    for (int t0 = s.from; t0 < s.to; t0 += kTokenBatch) {
      Unit<DT, 1> q[kTokenBatch][kAny];
#pragma unroll
      for (int t = 0; t < kTokenBatch; ++t) {
        const int64_t at = static_cast<int64_t>(w.token_at(t0 + t < s.to ? t0 + t : t0)) * a.grad_stride;
#pragma unroll
        for (int j = 0; j < kAny; ++j)
          if (u0 + 32 * j < a.units) q[t][j] = load_unit<DT, 1>(a.grad, at + u0 + 32 * j);
      }
#pragma unroll
      for (int t = 0; t < kTokenBatch; ++t) {
        if (t0 + t >= s.to) break;
        const int64_t row = w.key_at(t0 + t);
        const bool end = s.last_of_run(t0 + t);
#pragma unroll
        for (int j = 0; j < kAny; ++j) {
          if (u0 + 32 * j >= a.units) continue;
          add_unit<DT, 1>(q[t][j], acc[j]);
          if (!end) continue;
          float old[1] = {};
          if constexpr (ACC) load_floats_plain<DTO, 1>(a.out, row * a.hidden + u0 + 32 * j, old);
          write_unit<DTO, 1, ACC>(a, row, u0 + 32 * j, acc[j], old);
          acc[j][0] = 0.0f;
        }
      }
    }
  }
}

int64_t round16(int64_t bytes) { return (bytes + 15) & ~int64_t(15); }

struct Workspace {
  uint32_t *keys[2], *values[2], *counts[2];
  Counters* counters;
  uint2* long_runs;
  uint32_t* begins;
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
    w.counts[i] = reinterpret_cast<uint32_t*>(take(n > kRankMax ? int64_t(kSortMaxCtas) * kSortMaxBins * 4 : 0));
  }
  w.counters = reinterpret_cast<Counters*>(take(sizeof(Counters)));
  w.long_runs = reinterpret_cast<uint2*>(take(n / kLongRun * 8));
  w.begins = reinterpret_cast<uint32_t*>(take(vocab * 4));
  w.present = take(vocab);
  w.chunk_sums = reinterpret_cast<float*>(take(n > kDirectMax ? n / kChunk * hidden * 4 : 0));
  w.bytes = at;
  return w;
}

// The next `rows` of the rows that are not looked after yet.
ZeroFill share_of(ZeroFill& rest, int64_t rows) {
  ZeroFill z = rest;
  if (rest.end - rest.begin < rows) rows = rest.end - rest.begin;
  z.end = z.begin + rows;
  rest.begin = z.end;
  // whole blocks of neighbouring rows; a grid has room for 2^31 of them
  z.rows = static_cast<int>(z.row_bytes < kFillBytes ? kFillBytes / z.row_bytes : 1);
  z.blocks = static_cast<unsigned>((rows + z.rows - 1) / z.rows);
  return z;
}

// Sorts (id, position) into w.keys[where] / w.values[where].  `rest`: the rows in which zeros are still to be looked for
// (none with `accumulate`).
cudaError_t sort_tokens(const TableGradArgs& a, const Workspace& w, int* where, ZeroFill& rest, cudaStream_t stream) {
  int bits = 1;
  while ((int64_t(1) << bits) <= a.vocab) ++bits;  // keys go up to vocab
  SortArgs s{};
  s.tokens = Ids{a.ids, a.n_ids, a.vocab, a.padding_id, a.id_dtype, a.status};
  s.n = a.n_ids;
  s.counters = w.counters;
  if (rest.end > 0) {
    const cudaError_t e = cudaMemsetAsync(w.present, 0, static_cast<size_t>(a.vocab), stream);
    if (e != cudaSuccess) return e;
    s.zero.present = w.present;
  }
  *where = 0;
  if (a.n_ids <= kRankMax) {
    s.keys_out = w.keys[0];
    s.values_out = w.values[0];
    sort_small_kernel<<<static_cast<unsigned>((a.n_ids + 31) / 32), kRankThreads, kRankMax * 4, stream>>>(s);
    return cudaGetLastError();
  }
  const int passes = (bits + kSortMaxBits - 1) / kSortMaxBits;
  s.width = (bits + passes - 1) / passes;
  const int64_t tiles = (a.n_ids + kSortTile - 1) / kSortTile;
  const int64_t ctas = tiles < kSortMaxCtas ? tiles : kSortMaxCtas;
  s.span = (tiles + ctas - 1) / ctas * kSortTile;
  s.sort_blocks = static_cast<unsigned>((a.n_ids + s.span - 1) / s.span);
  for (int p = 0; p < passes; ++p) {
    s.first = p == 0;
    s.keys_in = w.keys[(p + 1) & 1];
    s.values_in = w.values[(p + 1) & 1];
    s.keys_out = w.keys[p & 1];
    s.values_out = w.values[p & 1];
    s.counts = w.counts[p & 1];
    s.next_counts = p + 1 < passes ? w.counts[(p + 1) & 1] : nullptr;
    s.shift = p * s.width;
    if (p == 0) {
      sort_count_kernel<<<s.sort_blocks, kSortThreads, 0, stream>>>(s);
    } else if (s.next_counts != nullptr) {  // cleared by the count launch for the second digit only
      const cudaError_t e = cudaMemsetAsync(s.next_counts, 0, static_cast<size_t>(s.sort_blocks) * 4 << s.width, stream);
      if (e != cudaSuccess) return e;
    }
    s.zero = share_of(rest, p + 1 < passes ? a.vocab / passes : a.vocab);
    cudaError_t e = cudaGetLastError();
    // overlaps the launch before it unless that was the clearing of the counts
    if (e == cudaSuccess) e = launch_dependent(p == 0 || s.next_counts == nullptr, sort_move_kernel, s.sort_blocks + s.zero.blocks, kSortThreads, 0, stream, s);
    if (e != cudaSuccess) return e;
  }
  *where = (passes - 1) & 1;
  return cudaSuccess;
}

template <int DT, int DTO, int VEC, bool ACC>
cudaError_t launch_sums(const TableGradArgs& a, const Workspace& w, int where, ZeroFill rest, cudaStream_t stream) {
  SumArgs s{};
  s.grad = a.grad;
  s.grad_stride = a.grad_stride;
  s.keys = w.keys[where];
  s.tokens = w.values[where];
  s.counters = w.counters;
  s.long_runs = w.long_runs;
  s.begins = w.begins;
  s.out = a.out;
  s.n = a.n_ids;
  s.vocab = a.vocab;
  s.hidden = a.hidden;
  s.scale = a.scale;
  s.units = a.hidden / VEC;
  s.tiles = (s.units + 31) / 32;
  const int64_t sms = sm_count();
  const bool chunks = a.n_ids > kDirectMax;
  const bool few = a.n_ids <= kRankMax;  // short kernels one behind the other: their launches overlap
  if (chunks) {
    s.chunk_sums = w.chunk_sums;
    constexpr int kUnits = VEC > 1 ? 1 : kAny;
    const int64_t items = a.n_ids / kChunk * ((s.units + 32 * kUnits - 1) / (32 * kUnits));
    const int64_t grid = (items + 7) / 8 < sms * 5 ? (items + 7) / 8 : sms * 5;
    s.zero = share_of(rest, (rest.end - rest.begin) / 2);
    const cudaError_t e = launch_dependent(few, chunk_sums_kernel<DT, VEC, kUnits>, static_cast<unsigned>(grid) + s.zero.blocks, 256, 0, stream, s);
    if (e != cudaSuccess) return e;
  }
  s.zero = share_of(rest, rest.end - rest.begin);
  const auto finish = [&](auto kern, int vectors, size_t smem) {
    int per_sm = 4;
    if (smem < kLongShared<VEC>) smem = kLongShared<VEC>;
    const cudaError_t e = kernel_launch_config(reinterpret_cast<const void*>(kern), 256, smem, -1, &per_sm);
    if (e != cudaSuccess) return e;
    // a few items per warp that is resident at once, so that the uneven runs even out; few tokens: few positions per item
    const int64_t tiles = (s.units + 32 * vectors - 1) / (32 * vectors);
    s.group = kMaxGroup;
    while (s.group > 1 && (a.n_ids + s.group - 1) / s.group * tiles < sms * per_sm * 8 * 4) s.group /= 2;
    const int64_t items = (a.n_ids + s.group - 1) / s.group * tiles;
    // A CTA per SM begins with the long runs, if there are any.  With two, text's skew loses (65536 tokens of 4096 columns over
    // 128256 rows 285 -> 287 us in a graph, 16384 over 32000 97 -> 99), many tokens per row gain (65536 of 8192 columns over 1000 rows,
    // uniform: 349 -> 309).
    const int64_t long_items = a.n_ids < kLongRun ? 0 : (chunks ? a.n_ids / kLongRun : (a.n_ids + kLongRun - 1) / kLongRun) * s.tiles;
    s.long_blocks = static_cast<unsigned>(long_items < sms ? long_items : sms);
    s.share = few ? 0 : 1;
    const int64_t room = sms * (per_sm > 1 ? per_sm : 2) - (s.share ? s.long_blocks : 0);
    const int64_t blocks = (items + 7) / 8 < room ? (items + 7) / 8 : room;
    return launch_dependent(few, kern, s.long_blocks + static_cast<unsigned>(blocks) + s.zero.blocks, 256, smem, stream, s);
  };
  if constexpr (VEC > 1) {
    // Two vectors per lane share what a token costs in instructions (65536 skewed tokens of 4096 columns over 128256 rows: 302 us
    // with one, 283 with two; 16384 uniform ones over 2000 rows 72 and 66); one keeps more warps busy where there are not four
    // such items for each (1024 skewed tokens over 2000 rows: 26.1 and 29.2; 1776, about the limit, 35.8 and 37.7, but uniform
    // 26.5 and 24.8).  Four make the items so large that the last ones are waited for: 115 us instead of 104 for 16384 tokens.
    constexpr size_t kSmem = size_t(8) * (ACC ? 8 : 16) * 32 * (16 + (ACC ? VEC * Elem<DTO>::kBytes : 0));
    if (s.units > 32 && a.n_ids * ((s.units + 63) / 64) >= sms * 24 * 4) return finish(row_stream_kernel<DT, DTO, ACC, 2>, 2, kSmem);
    return finish(row_stream_kernel<DT, DTO, ACC, 1>, 1, kSmem);
  } else {
    return finish(row_sums_any_kernel<DT, DTO, ACC>, kAny, 0);
  }
}

template <int DT, int DTO, int VEC>
cudaError_t launch_sums(const TableGradArgs& a, const Workspace& w, int where, const ZeroFill& rest, cudaStream_t stream) {
  return a.accumulate ? launch_sums<DT, DTO, VEC, true>(a, w, where, rest, stream)
                      : launch_sums<DT, DTO, VEC, false>(a, w, where, rest, stream);
}

template <int DT, int DTO>
cudaError_t launch_table_grad_t(const TableGradArgs& a, void* workspace, cudaStream_t stream) {
  const Workspace w = lay_out(workspace, a.vocab, a.hidden, a.n_ids);
  ZeroFill rest{};
  rest.out = static_cast<unsigned char*>(a.out);
  rest.row_bytes = static_cast<int64_t>(a.hidden) * Elem<DTO>::kBytes;
  rest.vectors = rest.row_bytes % 16 == 0 && aligned_to(a.out, 16);
  rest.present = w.present;
  rest.end = a.accumulate ? 0 : a.vocab;
  int where = 0;
  const cudaError_t e = sort_tokens(a, w, &where, rest, stream);
  if (e != cudaSuccess || a.vocab == 0) return e;
  constexpr int kPV = Elem<DT>::kPerVec;
  if (a.hidden % kPV == 0 && a.grad_stride % kPV == 0 && aligned_to(a.grad, 16) && aligned_to(a.out, 16))
    return launch_sums<DT, DTO, kPV>(a, w, where, rest, stream);
  return launch_sums<DT, DTO, 1>(a, w, where, rest, stream);
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
