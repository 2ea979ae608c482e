// Launchers of the token operators: RMS norm with residual and 8-bit output, the 8-bit linear product,
// rotary positions, window attention and its step on a rolling cache.
#pragma once

#include "common.hpp"

namespace mnn {
namespace k {

// A row of values that a kernel reads or writes, f32 or bf16 (or e4m3 where stated).
struct RmsNormArgs {
  const void* x = nullptr;
  const void* r = nullptr;     // residual, may be null
  void* sum = nullptr;         // x + r, may be null; may be x or r
  mnn_dtype in = MNN_F32;      // of x, r and sum
  const float* w = nullptr;    // [F]; null: no norm, the rows of x are only rounded to 8 bits
  void* y = nullptr;
  mnn_dtype out = MNN_F32;     // f32, bf16 or e4m3
  float* scales = nullptr;     // [rows], with e4m3
  int64_t rows = 0;
  int F = 0;
  int64_t ldy = 0;             // elements from one row of y to the next; those behind F become 0
  float eps = 0.f;
};
void rmsnorm(const LaunchCtx& c, const RmsNormArgs& a);

struct LinearE4m3Args {
  const uint8_t* x = nullptr;  // [M][ldx], ldx = K or, up to kLinearFew rows, in_features
  const float* xs = nullptr;   // [M]
  const uint8_t* w = nullptr;  // [N][K]
  const float* ws = nullptr;   // [N]
  const float* bias = nullptr; // [N] or null
  const void* r = nullptr;     // [M][N] of the output's type, or null; may be y
  void* y = nullptr;           // [M][N]
  mnn_dtype out = MNN_F32;     // f32 or bf16
  int64_t M = 0;
  int N = 0, K = 0, ldx = 0;   // K: a multiple of 128, the weights' zeros behind in_features included
  int act = 0;
  float alpha = 0.01f;
};
constexpr int kLinearFew = 32;
void linear_e4m3(const LaunchCtx& c, const LinearE4m3Args& a);
// rows of `n` bytes copied to rows of `ld` >= n, the rest zero
void pad_rows_u8(const LaunchCtx& c, const uint8_t* x, int64_t rows, int n, uint8_t* y, int ld);

struct RotaryArgs {
  const void* x[2] = {nullptr, nullptr};  // q and k
  void* y[2] = {nullptr, nullptr};
  int heads[2] = {0, 0};
  mnn_dtype type = MNN_F32;
  const int* pos = nullptr;               // [S][axes] or [B * S][axes]
  bool shared = true;                     // positions shared by the batch
  int64_t B = 0, S = 0;
  int hd = 0, axes = 0, interleaved = 0;
  int dims[4] = {0, 0, 0, 0};
  int pairs = 0;                          // sum of dims / 2
  const double* rate = nullptr;           // [pairs], turns per position
};
void rotary(const LaunchCtx& c, const RotaryArgs& a);

struct WindowArgs {
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  void* o = nullptr;
  mnn_dtype type = MNN_F32;
  const int* lengths = nullptr;  // [B] or null
  int B = 0, S = 0, H = 0, KV = 0, hd = 0;
  int left = 0, right = 0, sinks = 0;
  float scale = 1.f;
};
void window_attention(const LaunchCtx& c, const WindowArgs& a);

struct WindowStepArgs {
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  void* kc = nullptr;
  void* vc = nullptr;
  void* o = nullptr;
  mnn_dtype type = MNN_F32;
  const int* pos = nullptr;    // [B]
  const int* steps = nullptr;  // [B] or null
  int B = 0, T = 0, C = 0, H = 0, KV = 0, hd = 0;
  int left = 0, sinks = 0;
  float scale = 1.f;
};
// floats of workspace that a call needs (0: none), the same on every call of the same sizes
int64_t window_step_part_floats(const LaunchCtx& c, const WindowStepArgs& a);
void window_step(const LaunchCtx& c, const WindowStepArgs& a, float* part);

}  // namespace k
}  // namespace mnn
