// Host-side launcher declarations shared by the .cu files and the C ABI layer.
#pragma once

#include "common.cuh"

namespace cb200 {

// launch_cache.cu: per-device values and per-kernel attributes, set up once and cached.
// device_sm_count: SMs of the current device.  kernel_launch_config: raises `func`'s dynamic
// shared-memory limit to the architectural maximum (once), applies the shared-memory carve-out
// preference when it changes (pass -1 to leave it alone) and returns how many CTAs of `threads`
// threads and `smem` dynamic bytes fit on an SM (pass NULL to skip the query).
cudaError_t device_sm_count(int* out);
cudaError_t kernel_launch_config(const void* func, int threads, size_t smem, int carveout_percent,
                                 int* ctas_per_sm);

// The wait parameters every launcher copies into its kernel's arguments (launch_cache.cu).
WaitTuning wait_tuning();
void set_wait_tuning(WaitTuning t);

// Launches a kernel that begins with follow_previous() behind the kernel launched last on `stream`, which is one of the
// same call and does so too: with `overlap` its launch overlaps that kernel's end, which saves about 1.5 us.  Not behind a
// kernel that keeps the memory busy with loads into registers for long: shared memory of the waiting CTAs takes L1 from
// them (table gradient of 65536 tokens over 1000 rows of 8192 columns: 350 us without, 377 with).
template <typename... P, typename... A>
cudaError_t launch_dependent(bool overlap, void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                             const A&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
  c.attrs = &attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kern, args...);
}

// SMs of the current device for grid sizing; if the query fails the launch that follows reports
// the error, and 148 (B200) stands in meanwhile.
inline int sm_count() {
  int n = 148;
  return device_sm_count(&n) == cudaSuccess ? n : 148;
}

constexpr int kOpRmsNorm = 0;
constexpr int kOpLayerNorm = 1;

// Arguments of the lane-per-row and any-shape norm kernels.
struct LaneRowArgs {
  const void* x;      // [rows, n], or the dense table [vocab, n] when ids != nullptr
  const void* res;    // optional residual (dense source only)
  const void* alpha;  // weight [n]
  const void* beta;   // bias [n] (layer norm)
  void* y;
  void* sum_out;      // optional: h = x + res, or the gathered rows
  const void* ids;
  int id_dtype;
  int64_t vocab;
  cb200_status* status;
  int64_t rows;
  int n;
  float eps;
  int bulk;   // gather source: stage rows with the bulk-copy engine
  int V;      // filled by the launcher: 16-byte vectors per row
  int pitch;  // filled by the launcher: shared-memory row pitch in bytes
  int R;      // filled by the launcher: rows per CTA
  int classic;  // keep to the whole-row kernel where the streaming one would apply (cross-checks)
  WaitTuning wt;  // filled by the launcher
};

struct RmsRowRegArgs;
struct QRmsArgs;

bool rms_rowreg_supported(int dtype, int cols);
bool qrms_rowreg_supported(int dtype, int cols);
cudaError_t launch_rms_rowreg(int dtype, const RmsRowRegArgs& a, cudaStream_t stream);
cudaError_t launch_qrms_rowreg(int qtype, int dtype, const QRmsArgs& a, cudaStream_t stream);
// lookup + RMS norm for the K-quant super-block formats (kqrms.cu)
bool kqrms_supported(int qtype, int dtype, int cols);
cudaError_t launch_kqrms(int qtype, int dtype, const QRmsArgs& a, cudaStream_t stream);

bool norm_lanerow_supported(int dtype, int cols);
cudaError_t launch_norm_lanerow(int dtype, int op, const LaneRowArgs& a, cudaStream_t stream);
cudaError_t launch_norm_generic(int dtype, int op, const LaneRowArgs& a, cudaStream_t stream);

// candle's composite norm (norm_slow.cu); bias may be NULL
cudaError_t launch_norm_slow(int dtype, const void* x, const void* weight, const void* bias, void* y, int64_t rows,
                             int n, float eps, int remove_mean, cudaStream_t stream);

// softmax over the last dimension and rotary embeddings (neighbours.cu).  rope variants: 0 rope_i
// (interleaved pairs, src [b, h, t, d]), 1 rope (half-split pairs, [b, h, t, d]), 2 rope_thd ([b, t, h, d]).
cudaError_t launch_softmax_last_dim(int dtype, const void* x, void* y, int64_t rows, int n, cudaStream_t stream);
cudaError_t launch_rope(int variant, int dtype, const void* src, const void* cos_, const void* sin_, void* dst, int64_t b,
                        int h, int t, int d, cudaStream_t stream);

// Row gathers (embedding.cu)
struct GatherArgs {
  const unsigned char* src;  // [left, src_dim, row_bytes]
  const void* ids;
  unsigned char* out;        // [left, n_ids, row_bytes]
  int64_t left, src_dim, n_ids;
  int64_t row_bytes;
  int id_dtype;
  cb200_status* status;
  WaitTuning wt;  // filled by the launcher
};
cudaError_t launch_gather_rows(const GatherArgs& a, cudaStream_t stream);

struct QGatherArgs {
  const unsigned char* qtable;
  const void* ids;
  void* out;
  int id_dtype;
  int64_t vocab, vocab_begin, vocab_end;
  cb200_status* status;
  int64_t rows;
  int n;          // elements per row (multiple of 32)
  int row_bytes;  // bytes per quantised row
  int bulk;
  WaitTuning wt;  // filled by the launcher
};
cudaError_t launch_qgather(int qtype, int out_dtype, const QGatherArgs& a, cudaStream_t stream);
cudaError_t launch_qroute_rows(const unsigned char* qtable, const void* ids, int id_dtype, int64_t vocab,
                               int64_t vocab_begin, int64_t vocab_end, cb200_status* status, int64_t rows, int row_bytes,
                               void* const* dsts, int n_dsts, const int64_t* row_bounds, cudaStream_t stream);
cudaError_t launch_dequantize_flat(int qtype, int out_dtype, const void* blocks, void* out, int64_t n_vec,
                                   cudaStream_t stream);  // n_vec: groups of 8 elements

// Scaled lookup and the table's gradient (embedding_train.cu)
struct ScaledLookupArgs {
  const void* table;  // [vocab, hidden]
  const void* ids;
  void* out;          // [n_ids, hidden]
  int64_t vocab, n_ids;
  int hidden;
  float scale;
  int id_dtype;
  cb200_status* status;
};
cudaError_t launch_embedding_scaled(int dtype, const ScaledLookupArgs& a, cudaStream_t stream);

struct TableGradArgs {
  const void* grad;  // [n_ids, hidden], rows grad_stride elements apart
  int64_t grad_stride;
  const void* ids;
  void* out;  // [vocab, hidden]
  int64_t vocab, n_ids, padding_id;
  int hidden;
  float scale;
  int id_dtype;
  int accumulate;
  cb200_status* status;
};
int64_t table_grad_workspace(int64_t vocab, int hidden, int64_t n_ids);
cudaError_t launch_table_grad(int dtype, int out_dtype, const TableGradArgs& a, void* workspace, cudaStream_t stream);

// Gradient of the RMS norm (rms_backward.cu)
struct RmsBackwardArgs {
  const void* grad;
  const void* x;
  const void* alpha;
  const void* grad_sum;  // optional
  void* dx;
  float* dalpha;
  int64_t rows;
  int n;
  float eps;
};
int64_t rms_backward_workspace(int64_t rows, int n);
cudaError_t launch_rms_backward(int dtype, const RmsBackwardArgs& a, void* workspace, cudaStream_t stream);
// Sum over p of partials[p * cols + c] in a fixed order, to out[c] for c < split, out2[c - split] behind (rms_backward.cu)
cudaError_t launch_sum_partials(const float* partials, int n_partials, int cols, float* out, int split, float* out2,
                                cudaStream_t stream);

// Head norms with the rotation in the same pass (head_norm.cu)
cudaError_t launch_qk_norm_rope(const cb200_heads& q, const cb200_heads& k, const cb200_heads& q_out,
                                const cb200_heads& k_out, const cb200_qk_args& a, cb200_status* status,
                                cudaStream_t stream);
int64_t qk_backward_workspace(int dim);
cudaError_t launch_qk_norm_rope_backward(const cb200_heads& grad_q, const cb200_heads& grad_k, const cb200_heads& q,
                                         const cb200_heads& k, const cb200_heads& dq, const cb200_heads& dk,
                                         float* dq_weight, float* dk_weight, const cb200_qk_args& a, void* workspace,
                                         cb200_status* status, cudaStream_t stream);

}  // namespace cb200
