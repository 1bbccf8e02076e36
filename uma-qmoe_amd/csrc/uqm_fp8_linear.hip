// Product of matrices in 8-bit floats with a scale per group (definition in
// uqm_fp8.h). One v_mfma_f32_16x16x128_f8f6f4 takes exactly the 128 columns of a
// scale group, so a block's sum comes out of one instruction unscaled and
//   acc += (xs[t, b] * ws[n / 128, b]) * sum
// is folded in FP32: a 16-row tile of the weight lies in one row block, a lane of
// the result holds one token, so the factor is one value per lane and tile.
//
// The weight is the A operand (rows of D: 4 * (lane / 16) + i), tokens the B
// operand (columns of D: lane % 16). Both take the lane's row lane % 16 and the
// 16-byte pieces lane / 16 and lane / 16 + 4 of a group's 128 bytes; which
// columns an instruction puts at which of its 128 steps does not matter as long
// as both operands agree.
//
// Rounding: the matrix cores add 8-bit products in eights (8 neighbouring bytes
// of the operands), aligned to the largest sum of exponents E among the eight and
// cut towards zero below 2^(E - 13); the sums of eights are FP32. (Measured; all
// forms of the instruction do it, also the ones of half the rate.) That is 2^9
// times finer than the codes' own steps, and the scaled sums here are FP32.
#include "uqm_device.h"
#include "uqm_fp8.h"

namespace uqm {
namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4_t mfma_fp8(const uint4& a0, const uint4& a1, const uint4& b0, const uint4& b1) {
  const i32x8_t a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const i32x8_t b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;

// 16 weight rows x 16 * NT tokens per workgroup, the column blocks dealt out to
// its waves, whose sums are added in wave order.
template <int NT>
__global__ __launch_bounds__(kThreads) void fp8_rows_kernel(Fp8LinearArgs a) {
  __shared__ f32x4_t part[kWaves][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q = lane >> 4, r = lane & 15;
  const int64_t blocks_n = (a.N + 15) / 16;
  const int64_t n0 = blockIdx.x % blocks_n * 16, t0 = blockIdx.x / blocks_n * (16 * NT);
  const int64_t KB = (a.K + kFp8Group - 1) / kFp8Group;
  const uint8_t* w = a.w + min(n0 + r, a.N - 1) * a.K;
  const float* ws = a.ws + n0 / kFp8Group * KB;
  const uint8_t* x[NT];
  const float* xs[NT];
  f32x4_t acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t t = min(t0 + 16 * i + r, a.T - 1);  // (rows behind the last repeat it)
    x[i] = a.x + t * a.K;
    xs[i] = a.xs + t * KB;
    acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t b = wave; b < KB; b += kWaves) {
    const int64_t k0 = b * kFp8Group + 16 * q, k1 = k0 + 64;
    const bool in0 = k0 < a.K, in1 = k1 < a.K;  // (K is a multiple of 16)
    const uint4 w0 = in0 ? ldg16(w + k0) : zero, w1 = in1 ? ldg16(w + k1) : zero;
    const float s = ws[b];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const f32x4_t d = mfma_fp8(w0, w1, in0 ? ldg16(x[i] + k0) : zero, in1 ? ldg16(x[i] + k1) : zero);
      const float f = s * xs[i][b];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(f, d[e], acc[i][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int o = threadIdx.x; o < NT * 64; o += kThreads) {
    const int i = o >> 6, l = o & 63;
    f32x4_t v = part[0][i][l];
#pragma unroll
    for (int g = 1; g < kWaves; ++g) v += part[g][i][l];
    const int64_t t = t0 + 16 * i + (l & 15), n = n0 + 4 * (l >> 4);
    if (t >= a.T) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N)
        a.out[t * a.N + n + e] = f32_to_bf16(v[e] + (a.bias != nullptr ? bf16_to_f32(a.bias[n + e]) : 0.f));
  }
}

}  // namespace

hipError_t launch_fp8_linear(const Fp8LinearArgs& a, int cus, hipStream_t stream) {
  (void)cus;
  if (a.T <= 0) return hipSuccess;
  const int nt = a.T <= 16 ? 1 : 4;
  const int64_t grid = (a.N + 15) / 16 * ((a.T + 16 * nt - 1) / (16 * nt));
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  auto* k = nt == 1 ? fp8_rows_kernel<1> : fp8_rows_kernel<4>;
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace uqm
