// Host-side declarations of the gated feed-forward block, the trainable norms and dropout (raw pointers + stream; no
// torch headers).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace afb {

// Gated feed-forward block over T rows: g = x Wg^T, u = x Wu^T (w13 = [Wg; Wu], [2F, H]), h = act(g) u,
// y = h W2^T (+ residual), W2 [N, F]. H, F and N are multiples of 8; every row stride is a multiple of 8 elements
// and every base 16-byte aligned.
struct FfnShape {
  int64_t T = 0;
  int H = 0, F = 0, N = 0;
  int act = 0;   // 0 silu, 1 tanh-GELU, 2 erf-GELU
  int fp16 = 0;  // element type of x, weights and results: 0 bf16, 1 fp16
};
// fp32 elements of scratch the calls below need (one buffer per call in flight)
size_t ffn_fwd_scratch(const FfnShape& s, int num_sms);
size_t ffn_bwd_scratch(const FfnShape& s, int num_sms);
int64_t ffn_h_rows(const FfnShape& s);  // rows of the buffer for h: T, or 2T where a second term is kept
// h [ffn_h_rows, F], h itself in the first T rows; gu [T rounded up to 32, 2F] fp32 (u act'(g) and act(g) in the
// kernels' own order, for the backward pass), 32-byte aligned, or null; y [T, N]
int ffn_fwd(const FfnShape& s, const void* x, int64_t ldx, const void* w13, const void* w2, const void* residual,
            int64_t ldr, void* h, float* gu, void* y, float* scratch, int num_sms, uint32_t* status,
            cudaStream_t stream);
// dgu [T, 2F] (element type) is written when dx or dw13 is asked for; dx / dw13 / dw2 may be null
int ffn_bwd(const FfnShape& s, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w13,
            const void* w2, const void* h, const float* gu, void* dgu, void* dx, void* dw13, void* dw2, float* scratch,
            int num_sms, uint32_t* status, cudaStream_t stream);

// Norms with trainable weights over rows of `width` (1 .. NORM_MAX_WIDTH), fp32 statistics.
constexpr int NORM_MAX_WIDTH = 16384;
enum ElemType { ELEM_BF16 = 0, ELEM_FP16 = 1, ELEM_FP32 = 2 };
struct NormArgs {
  int64_t rows = 0;
  int width = 0;
  int rms = 0;    // 0: (x - mean) rstd w + b; 1: x rstd (1 + w)
  int dtype = 0;  // ElemType of x, y, dy, dx
  int wtype = 0;  // ElemType of w, b, dw, db: ELEM_FP32 or dtype
  float eps = 0.f;
  const void* x = nullptr;
  int64_t ldx = 0;
  const void* w = nullptr;
  const void* b = nullptr;      // optional, not with rms
  void* y = nullptr;            // [rows, width]
  float* mean = nullptr;        // [rows], written / read unless rms; null: not kept
  float* rstd = nullptr;        // [rows]; null: not kept
  const void* dy = nullptr;     // backward: [rows, width]
  void* dx = nullptr;           // or null
  void* dw = nullptr;           // or null
  void* db = nullptr;           // or null
  float* partial = nullptr;     // with dw or db: `partials` rows of 2 x width floats
  int partials = 0;             // norm_bwd_partials()
  uint32_t* status = nullptr;   // kernel status word
};
int norm_bwd_partials(const NormArgs& a, int num_sms);  // rows of `partial` the backward pass writes; 0: it cannot run
int norm_fwd(const NormArgs& a, int num_sms, cudaStream_t stream);
int norm_bwd(const NormArgs& a, int num_sms, cudaStream_t stream);

// y = x * scale where kept, else 0 (+ residual), over n contiguous elements; element i is kept when its 16 bits of
// Philox4x32-10(key = seed, counter = offset + i / 8) are below `threshold` (0 .. 65536), scale = 65536 / threshold.
// `rng` (optional, int64 [2] on the device): its seed and offset are added to the call's.
int dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, uint32_t threshold, uint64_t seed,
            uint64_t offset, const int64_t* rng, int num_sms, cudaStream_t stream);

}  // namespace afb
