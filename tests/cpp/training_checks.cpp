// The host side of the training and serving operators in candle_b200.hpp: argument errors, decided without a device.
#include <cstdio>
#include <functional>

#include "candle_b200.hpp"

using namespace candle_b200;

static int failed = 0;
static void refuses(const char* what, const char* part, const std::function<void()>& f) {
  try {
    f();
  } catch (const Error& e) {
    if (std::string(e.what()).find(part) != std::string::npos) {
      std::printf("ok %s\n", what);
      return;
    }
    std::printf("FAILED %s: %s\n", what, e.what());
    ++failed;
    return;
  }
  std::printf("FAILED %s: no error\n", what);
  ++failed;
}

int main() {
  void* p = reinterpret_cast<void*>(256);  // never dereferenced
  Tensor table{p, {10, 8}, DType::BF16}, ids{p, {2, 3}, DType::U32}, out{p, {2, 3, 8}, DType::BF16}, wrong{p, {6, 8}, DType::BF16};
  refuses("lookup into a wrong shape", "destination", [&] { ops::embedding_scaled(table, ids, 2.0f, wrong, nullptr, nullptr); });
  Tensor float_ids{p, {2, 3}, DType::F32};
  refuses("float ids", "ids", [&] { ops::embedding_scaled(table, float_ids, 2.0f, out, nullptr, nullptr); });

  Tensor dtable{p, {10, 8}, DType::F32}, half{p, {10, 8}, DType::F16}, grad{p, {2, 3, 8}, DType::BF16};
  ops::Workspace ws{p, ops::embedding_backward_workspace(10, 8, 6)}, small{p, ws.bytes - 1};
  refuses("gradient of another shape", "shape mismatch", [&] { ops::embedding_backward(wrong, ids, dtable, ws, nullptr, nullptr); });
  refuses("f16 result of a bf16 gradient", "destination", [&] { ops::embedding_backward(grad, ids, half, ws, nullptr, nullptr); });
  refuses("small workspace", "workspace", [&] { ops::embedding_backward(grad, ids, dtable, small, nullptr, nullptr); });

  Tensor x{p, {4, 8}, DType::F16}, alpha{p, {8}, DType::F16}, dalpha{p, {8}, DType::F32}, dx{p, {4, 8}, DType::F16}, g32{p, {4, 8}, DType::F32};
  ops::Workspace nw{p, ops::rms_norm_backward_workspace(4, 8)};
  refuses("gradient of another type", "rms-norm-backward", [&] { ops::rms_norm_backward(g32, x, alpha, 1e-5f, dx, dalpha, nw, nullptr); });
  refuses("dalpha in f16", "destination", [&] { ops::rms_norm_backward(x, x, alpha, 1e-5f, dx, alpha, nw, nullptr); });

  cb200_heads h{p, 64, 32, 16, 2, 0}, overlapping{p, 64, 32, 8, 2, 0};
  cb200_qk_args a{p, p, p, p, nullptr, 3, 2, 2, 16, 16, 1e-5f, 0, CB200_DTYPE_BF16, CB200_DTYPE_F32, CB200_ID_I64, 0};
  refuses("overlapping rows of the output", "overlap", [&] { ops::qk_norm_rope(h, h, overlapping, h, a, nullptr, nullptr); });
  a.rotary = 15;
  refuses("odd rotation", "rotated columns", [&] { ops::qk_norm_rope(h, h, h, h, a, nullptr, nullptr); });
  a.rotary = 16;
  Tensor dw{p, {16}, DType::F32}, dw16{p, {16}, DType::BF16};
  ops::Workspace qw{p, ops::qk_norm_rope_backward_workspace(16)}, none{};
  refuses("weight gradient in bf16", "destination", [&] { ops::qk_norm_rope_backward(h, h, h, h, h, h, dw, dw16, a, qw, nullptr, nullptr); });
  refuses("no workspace", "workspace", [&] { ops::qk_norm_rope_backward(h, h, h, h, h, h, dw, dw, a, none, nullptr, nullptr); });
  return failed;
}
