// The C++ mirror of the training and serving operators on a GPU: f32 inputs from files of the test, outputs back to files.
//   training_gpu <dir> <vocab> <hidden> <tokens> <q heads> <k heads> <dim>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "candle_b200.hpp"

using namespace candle_b200;

static std::string dir;

static void* allocate(int64_t bytes) {
  void* d = nullptr;
  if (cudaMalloc(&d, bytes ? bytes : 16) != cudaSuccess) std::exit(3);
  return d;
}
static Tensor read(const char* name, Shape dims, DType dtype = DType::F32) {
  FILE* f = std::fopen((dir + "/" + name).c_str(), "rb");
  Tensor t{nullptr, dims, dtype, true};
  std::vector<char> b(t.elem_count() * 4);
  if (!f || std::fread(b.data(), 1, b.size(), f) != b.size()) std::exit(2);
  std::fclose(f);
  t.data = allocate(static_cast<int64_t>(b.size()));
  if (cudaMemcpy(t.data, b.data(), b.size(), cudaMemcpyHostToDevice) != cudaSuccess) std::exit(3);
  return t;
}
static Tensor fresh(Shape dims) {
  Tensor t{nullptr, dims, DType::F32, true};
  t.data = allocate(t.elem_count() * 4);
  return t;
}
static void write(const char* name, const Tensor& t) {
  std::vector<char> b(t.elem_count() * 4);
  if (cudaMemcpy(b.data(), t.data, b.size(), cudaMemcpyDeviceToHost) != cudaSuccess) std::exit(4);
  FILE* f = std::fopen((dir + "/" + name).c_str(), "wb");
  if (!f || std::fwrite(b.data(), 1, b.size(), f) != b.size()) std::exit(2);
  std::fclose(f);
}
static ops::Workspace workspace(int64_t bytes) { return {allocate(bytes), bytes}; }

int main(int argc, char** argv) {
  if (argc != 8) return 2;
  dir = argv[1];
  const int64_t vocab = std::atoll(argv[2]), hidden = std::atoll(argv[3]), n = std::atoll(argv[4]);
  const int hq = std::atoi(argv[5]), hk = std::atoi(argv[6]), d = std::atoi(argv[7]);
  cudaStream_t stream;
  if (cudaStreamCreate(&stream) != cudaSuccess) return 3;
  try {
    cb200_status* status = static_cast<cb200_status*>(allocate(sizeof(cb200_status)));
    cudaMemset(status, 0, sizeof(cb200_status));
    const Tensor table = read("table", {vocab, hidden}), ids = read("ids", {2, n / 2}, DType::U32), alpha = read("alpha", {hidden});
    const Tensor grad = read("grad", {2, n / 2, hidden}), extra = read("extra", {2, n / 2, hidden});
    Tensor y = fresh({2, n / 2, hidden}), dtable = fresh({vocab, hidden}), sum = read("sum", {vocab, hidden});
    ops::embedding_scaled(table, ids, 3.0f, y, status, stream);
    const ops::Workspace tw = workspace(ops::embedding_backward_workspace(vocab, hidden, n));
    ops::embedding_backward(grad, ids, dtable, tw, status, stream, 3.0f);
    ops::embedding_backward(grad, ids, sum, tw, status, stream, 3.0f, true, 1);
    Tensor dx = fresh(y.dims), dalpha = fresh({hidden});
    const ops::Workspace nw = workspace(ops::rms_norm_backward_workspace(n, hidden));
    ops::rms_norm_backward(grad, y, alpha, 1e-5f, dx, dalpha, nw, stream, &extra);

    const Tensor q = read("q", {n, hq, d}), k = read("k", {n, hk, d}), gq = read("gq", q.dims), gk = read("gk", k.dims);
    const Tensor wq = read("wq", {d}), wk = read("wk", {d}), cosines = read("cos", {n, d / 2}), sines = read("sin", {n, d / 2});
    Tensor oq = fresh(q.dims), ok = fresh(k.dims), dq = fresh(q.dims), dk = fresh(k.dims), dwq = fresh({d}), dwk = fresh({d});
    const auto heads = [&](const Tensor& t, int count) { return cb200_heads{const_cast<void*>(static_cast<const void*>(t.data)), 0, int64_t(count) * d, d, count, 0}; };
    const cb200_qk_args a{wq.data, wk.data, cosines.data, sines.data, nullptr, 1, n, n, d, d, 1e-5f, 1, CB200_DTYPE_F32, CB200_DTYPE_F32, CB200_ID_I64, 0};
    ops::qk_norm_rope(heads(q, hq), heads(k, hk), heads(oq, hq), heads(ok, hk), a, status, stream);
    const ops::Workspace qw = workspace(ops::qk_norm_rope_backward_workspace(d));
    ops::qk_norm_rope_backward(heads(gq, hq), heads(gk, hk), heads(q, hq), heads(k, hk), heads(dq, hq), heads(dk, hk), dwq, dwk, a, qw, status, stream);
    if (cudaStreamSynchronize(stream) != cudaSuccess) return 4;
    cb200_status seen;
    if (cudaMemcpy(&seen, status, sizeof(seen), cudaMemcpyDeviceToHost) != cudaSuccess || seen.code != 0) return 5;
    write("out.y", y), write("out.dtable", dtable), write("out.sum", sum), write("out.dx", dx), write("out.dalpha", dalpha);
    write("out.oq", oq), write("out.ok", ok), write("out.dq", dq), write("out.dk", dk), write("out.dwq", dwq), write("out.dwk", dwk);
  } catch (const Error& e) {
    std::printf("%s\n", e.what());
    return 1;
  }
  try {  // 2^32 + 8 columns are not 8
    ops::rms_norm_backward_workspace(4, (int64_t(1) << 32) + 8);
    return 6;
  } catch (const Error& e) {
    if (std::string(e.what()).find("4294967304 columns") == std::string::npos) return 7;
  }
  return 0;
}
