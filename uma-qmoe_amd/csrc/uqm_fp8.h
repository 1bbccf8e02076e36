// Matrices in 8-bit floats (e4m3, largest value 448) with FP32 scales, and the
// operators around their products (uqm_fp8_rows.hip, uqm_fp8_linear.hip).
//
// A group is 128 neighbouring columns of one row (activations) or of 128 rows
// (weights), the last one of a row or of the rows possibly shorter. Its scale is
//   d = 1                        if every |v| is 0,
//       max(max|v| / 448, 2^-126) otherwise,
// and a code is e4m3(v * r), r = 1 / d rounded to FP32, to nearest even. That is v / d
// but for two FP32 roundings: where v / d is the middle between two codes up to
// 2^-23 of itself, the code may be the other one, as near as the one of the
// division (1 of 2000 codes of normal BF16 values; d itself is a rounded number, and
// against v / d in 64 bits the product is off no more often than an FP32 division).
// The lower limit of d keeps r finite.
// A group that holds a NaN or an infinity has a scale that is one, too (the
// maximum is taken over the bits, which keeps a NaN), and its codes are NaN or 0:
// every product of the row comes out as NaN.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace uqm {

constexpr int kFp8Group = 128;  // columns of a scale group; rows too, of a weight

// What a row operator writes (NULL: not wanted): rows [rows, cols] in BF16, the
// e4m3 codes [rows, cols] and their scales [rows, ceil(cols / 128)].
struct RowOutputs {
  uint16_t* bf16;
  uint8_t* codes;
  float* scales;
};

// s = bf16(x + r) -> sum (r NULL: s = x, nothing written); n = s * rsqrt(mean(s^2) + eps);
// BF16 output bf16(w * n), codes of the same w * n. weight NULL: ones. sum may be x or r.
hipError_t launch_add_rmsnorm(const uint16_t* x, const uint16_t* r, int64_t rows, int64_t cols, const uint16_t* weight,
                              float eps, uint16_t* sum, const RowOutputs& out, hipStream_t stream);
// y = silu(g) * u of rows [g (cols) | u (cols)].
hipError_t launch_silu_mul(const uint16_t* gate_up, int64_t rows, int64_t cols, const RowOutputs& out,
                           hipStream_t stream);
// Codes and scales of x [rows, cols] in blocks of block_rows (1 or 128) x 128.
hipError_t launch_fp8_quantize(const uint16_t* x, int64_t rows, int64_t cols, int block_rows, uint8_t* codes,
                               float* scales, hipStream_t stream);

// out[t, n] = bf16(bias[n] + sum over blocks b of 128 columns of
//                  xs[t, b] ws[n / 128, b] sum over k in b of x[t, k] w[n, k])
constexpr int64_t kFp8MaxK = int64_t{1} << 25;  // 64 rows below 2^31 bytes
struct Fp8LinearArgs {
  const uint8_t* x;       // codes [T, K]
  const float* xs;        // scales [T, ceil(K / 128)]
  const uint8_t* w;       // codes [N, K]
  const float* ws;        // scales [ceil(N / 128), ceil(K / 128)]
  const uint16_t* bias;   // bf16 [N] or NULL
  uint16_t* out;          // bf16 [T, N]
  int64_t T, N, K;        // K a multiple of 16 below kFp8MaxK
};
// Whether a launch has room for the outputs (2^31 of one token are the first without).
bool fp8_linear_fits(const Fp8LinearArgs& a);
// Rows and tokens of a workgroup, and its waves, that the call takes (zeros if it does not fit).
struct Fp8LinearPlan {
  int rows, tokens, waves;
};
Fp8LinearPlan plan_fp8_linear(const Fp8LinearArgs& a, int cus);
hipError_t launch_fp8_linear(const Fp8LinearArgs& a, int cus, hipStream_t stream);

}  // namespace uqm
