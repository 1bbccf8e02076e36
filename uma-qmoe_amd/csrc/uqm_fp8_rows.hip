// Row operators with an 8-bit output: residual addition + RMSNorm, gated SiLU,
// and the quantisation itself (definitions in uqm_fp8.h).
//
// All of them are bound by memory (3 to 9 bytes per element against some twenty
// instructions): norm of 4095 x 2048 with a residual and both outputs 13.5 us, 5.6
// TB/s; blocks of 11264 x 2048 12.2 us, 5.7; gate of 4095 x 5632 21.6 us, 5.4. A lane
// holds 8 neighbouring columns (one 16-byte load, an 8-byte store of codes), so 16
// lanes hold a group and its maximum is four exchanges within a row of the wave;
// each input is read once and kept in registers between the maximum and the codes.
// A row's results depend on that row alone, to the bit (of blocks of 128 rows: on
// that block).
#include "uqm_device.h"
#include "uqm_fp8.h"

#include <algorithm>
#include <initializer_list>

namespace uqm {
namespace {

constexpr int kThreads = 256;
constexpr float kFp8Max = 448.0f;

// 16 and 8 bytes at any alignment of their elements: one access each (the memory
// takes them at twice the cost or less; one per element was 3 to 4 times slower: 4000
// rows of 5475 with both outputs 118.6 us, so 36.9).
typedef uint32_t loose16_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t loose8_t __attribute__((ext_vector_type(2), aligned(1)));

// Columns c .. c+7 of a row as FP32, zeros from `cols` on. VEC: rows of a multiple
// of 8 columns, aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* row, int64_t c, int64_t cols, float (&v)[8]) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (c < cols) {
      const uint4 q = ldg16(row + c);
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
  } else if (c + 8 <= cols) {
    const loose16_t q = *reinterpret_cast<const loose16_t*>(row + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = q[j];
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (c + j < cols) w[j / 2] |= static_cast<uint32_t>(row[c + j]) << (16 * (j & 1));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = bf16lo(w[j]);
    v[2 * j + 1] = bf16hi(w[j]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store8_bf16(uint16_t* row, int64_t c, int64_t cols, const float (&v)[8]) {
  const uint32_t w[4] = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7])};
  if constexpr (VEC) {
    if (c < cols) *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (c + 8 <= cols) {
    *reinterpret_cast<loose16_t*>(row + c) = loose16_t{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (c + j < cols) row[c + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
  }
}

// Four values as e4m3 bytes, to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// (inv = 1 / d: one division a group; the codes are defined by the product with it)
template <bool VEC>
__device__ __forceinline__ void store8_fp8(uint8_t* row, int64_t c, int64_t cols, const float (&v)[8], float inv) {
  const uint32_t lo = pack_fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  const uint32_t hi = pack_fp8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  if constexpr (VEC) {
    if (c < cols) *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
  } else if (c + 8 <= cols) {
    *reinterpret_cast<loose8_t*>(row + c) = loose8_t{lo, hi};
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (c + j < cols) row[c + j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

// Bits of max|v|: as unsigned numbers magnitudes order like the floats, and a
// NaN above every other value, which fmaxf would drop.
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return m;
}
template <int O>
__device__ __forceinline__ uint32_t max_step(uint32_t m) {
  return max(m, __float_as_uint(xor_partner<O>(__uint_as_float(m))));
}
// Maximum over the 16 lanes of a group.
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = max_step<8>(m);
  m = max_step<4>(m);
  m = max_step<2>(m);
  return max_step<1>(m);
}
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const float d = __uint_as_float(bits) / kFp8Max;
  return bits == 0u ? 1.0f : (d < 0x1p-126f ? 0x1p-126f : d);
}

// Codes and scale of the group that this lane's 8 columns belong to.
template <bool VEC>
__device__ __forceinline__ void write_fp8(const RowOutputs& out, int64_t row, int64_t c, int64_t cols,
                                          int64_t all_cols, const float (&v)[8]) {
  const float d = scale_of(group_max(magnitude8(v)));
  store8_fp8<VEC>(out.codes + row * all_cols, c, cols, v, 1.0f / d);
  if ((threadIdx.x & 15u) == 0 && c < cols)
    out.scales[row * ((all_cols + kFp8Group - 1) / kFp8Group) + c / kFp8Group] = d;
}

// Sum over the workgroup of 4 waves.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

// LANES lanes per row: 16 for rows of a group, 64 (a wave, no barrier) up to 512
// columns, a workgroup beyond. Rows beyond 8 * kThreads * PASSES columns are read
// again in the second part (PASSES 0), each thread its own columns: the sum from
// where it wrote it.
template <int LANES, int PASSES, bool VEC>
__global__ __launch_bounds__(kThreads) void add_rmsnorm_kernel(const uint16_t* x, const uint16_t* r, int64_t rows,
                                                               int64_t all_cols, const uint16_t* __restrict__ weight,
                                                               float eps, uint16_t* sum, RowOutputs out) {
  __shared__ float part[kThreads / 64];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  // (lanes behind the last row stay, with no columns: a wave's exchanges take them all)
  const int64_t cols = row < rows ? all_cols : 0;
  const int64_t at = row * all_cols;
  const int64_t first = 8 * (threadIdx.x % LANES);  // this thread's columns of pass p: first + 8 * LANES * p
  auto load = [&](int64_t c, float (&s)[8]) {  // s = bf16(x + r), kept in `sum`
    load8<VEC>(x + at, c, cols, s);
    if (r != nullptr) {
      float t[8];
      load8<VEC>(r + at, c, cols, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = round_bf16(s[j] + t[j]);
      store8_bf16<VEC>(sum + at, c, cols, s);
    }
  };
  auto finish = [&](int64_t c, const float (&s)[8], float rstd) {
    float w[8], y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 1.0f;
    if (weight != nullptr) load8<VEC>(weight, c, cols, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = w[j] * (s[j] * rstd);
    if (out.bf16 != nullptr) store8_bf16<VEC>(out.bf16 + at, c, cols, y);
    if (out.codes != nullptr) write_fp8<VEC>(out, row, c, cols, all_cols, y);
  };
  float ss = 0.f;
  auto add = [&](const float (&s)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(s[j], s[j], ss);
  };
  auto rstd = [&]() {
    if constexpr (LANES == 16) {
      ss += xor_partner<8>(ss);
      ss += xor_partner<4>(ss);
      ss += xor_partner<2>(ss);
      ss += xor_partner<1>(ss);
    } else {
      ss = LANES == 64 ? wave_sum(ss) : block_sum(ss, part);
    }
    return rsqrtf(ss / static_cast<float>(all_cols) + eps);
  };
  if constexpr (PASSES > 0) {
    float v[PASSES][8];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) load(first + 8 * LANES * p, v[p]);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) add(v[p]);
    const float f = rstd();
#pragma unroll
    for (int p = 0; p < PASSES; ++p) finish(first + 8 * LANES * p, v[p], f);
  } else {
    static_assert(LANES == kThreads, "a workgroup per row");
    // (rounds in whole workgroups, so that a group's 16 lanes stay together)
    const int64_t rounds = (cols + 8 * kThreads - 1) / (8 * kThreads);
    float s[8];
    for (int64_t p = 0; p < rounds; ++p) {
      load(first + 8 * kThreads * p, s);
      add(s);
    }
    const float f = rstd();
    for (int64_t p = 0; p < rounds; ++p) {
      load8<VEC>((r != nullptr ? sum : x) + at, first + 8 * kThreads * p, cols, s);
      finish(first + 8 * kThreads * p, s, f);
    }
  }
}

// Position of this thread's 8 columns when rows of `chunks` groups of 8 columns
// (a multiple of 16) are dealt out over workgroups: several rows to a workgroup
// when they are short, several workgroups to a row when they are long.
struct Place {
  int64_t row, c;
};
__device__ __forceinline__ Place place(int64_t chunks) {
  if (chunks >= kThreads) {
    const int64_t per_row = (chunks + kThreads - 1) / kThreads;
    return {blockIdx.x / per_row, 8 * ((blockIdx.x % per_row) * kThreads + threadIdx.x)};
  }
  const int n = static_cast<int>(chunks), rows = kThreads / n;
  const int r = static_cast<int>(threadIdx.x) / n;
  // (threads behind the last whole row of the workgroup take none)
  return {r < rows ? static_cast<int64_t>(blockIdx.x) * rows + r : INT64_MAX, 8 * (static_cast<int>(threadIdx.x) % n)};
}
int64_t place_grid(int64_t rows, int64_t chunks) {
  if (chunks >= kThreads) return rows * ((chunks + kThreads - 1) / kThreads);
  const int64_t per = kThreads / chunks;
  return (rows + per - 1) / per;
}
__host__ __device__ int64_t chunks_of(int64_t cols) { return (cols + kFp8Group - 1) / kFp8Group * (kFp8Group / 8); }

// g / (1 + exp(-g)): the reciprocal with one Newton step, as near as the division
// at half its instructions. It flushes subnormal results to 0, so gates below
// -87.3 (1 + exp(-g) from 2^126 on) divide, and only they: a wave holds parts of
// several rows, and a row's result must not depend on its neighbours'.
__device__ __forceinline__ void silu8(float (&g)[8]) {
  float d[8], most = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    d[j] = 1.0f + __expf(-g[j]);
    most = fmaxf(most, d[j]);
  }
  auto by_reciprocal = [&](int j) {
    const float r = __builtin_amdgcn_rcpf(d[j]);
    return g[j] * fmaf(fmaf(-d[j], r, 1.0f), r, r);
  };
  if (__builtin_expect(__any(most > 0x1p126f), 0)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = d[j] > 0x1p126f ? g[j] / d[j] : by_reciprocal(j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = by_reciprocal(j);
  }
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void silu_mul_kernel(const uint16_t* __restrict__ x, int64_t rows, int64_t cols,
                                                            RowOutputs out) {
  const Place at = place(chunks_of(cols));
  if (at.row >= rows) return;  // (the 16 lanes of a group leave together)
  const uint16_t* g_row = x + at.row * 2 * cols;
  float g[8], u[8];
  load8<VEC>(g_row, at.c, cols, g);
  load8<VEC>(g_row + cols, at.c, cols, u);
  silu8(g);
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] *= u[j];
  if (out.bf16 != nullptr) store8_bf16<VEC>(out.bf16 + at.row * cols, at.c, cols, g);
  if (out.codes != nullptr) write_fp8<VEC>(out, at.row, at.c, cols, cols, g);
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                                 int64_t cols, RowOutputs out) {
  const Place at = place(chunks_of(cols));
  if (at.row >= rows) return;
  float v[8];
  load8<VEC>(x + at.row * cols, at.c, cols, v);
  write_fp8<VEC>(out, at.row, at.c, cols, cols, v);
}

// One workgroup per 128 x 128 block: 16 lanes a row of it, 16 rows at a time, all
// 8 turns in registers.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                                   int64_t cols, uint8_t* __restrict__ codes,
                                                                   float* __restrict__ scales) {
  __shared__ uint32_t part[kThreads / 64];
  const int64_t across = (cols + kFp8Group - 1) / kFp8Group;
  const int64_t row0 = blockIdx.x / across * kFp8Group + (threadIdx.x >> 4);
  const int64_t c = blockIdx.x % across * kFp8Group + 8 * (threadIdx.x & 15u);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    load8<VEC>(x + row * cols, row < rows ? c : cols, cols, v[i]);
    m = max(m, magnitude8(v[i]));
  }
  m = wave_max_u32(m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  const float d = scale_of(max(max(part[0], part[1]), max(part[2], part[3])));
  const float inv = 1.0f / d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    store8_fp8<VEC>(codes + row * cols, row < rows ? c : cols, cols, v[i], inv);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = d;
}

bool aligned(int64_t cols, std::initializer_list<const void*> wide, const void* codes) {
  uintptr_t bits = 0;
  for (const void* p : wide) bits |= reinterpret_cast<uintptr_t>(p);
  return cols % 8 == 0 && (bits & 15u) == 0 && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0;
}

// A launch has less than 2^32 threads, so more workgroups than these take several
// launches, each of whole rows.
constexpr int64_t kMaxGrid = 0xFFFFFFFF / kThreads;

template <typename T>
T* behind(T* p, int64_t elements) {
  return p == nullptr ? nullptr : p + elements;
}
RowOutputs behind(const RowOutputs& out, int64_t rows, int64_t cols) {
  return {behind(out.bf16, rows * cols), behind(out.codes, rows * cols),
          behind(out.scales, rows * ((cols + kFp8Group - 1) / kFp8Group))};
}
// Rows of a launch of silu_mul_kernel or quantize_rows_kernel.
int64_t place_rows(int64_t chunks) {
  return chunks >= kThreads ? kMaxGrid / ((chunks + kThreads - 1) / kThreads) : kMaxGrid * (kThreads / chunks);
}

}  // namespace

hipError_t launch_add_rmsnorm(const uint16_t* x, const uint16_t* r, int64_t rows, int64_t cols, const uint16_t* weight,
                              float eps, uint16_t* sum, const RowOutputs& out, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  const bool vec = aligned(cols, {x, r, weight, sum, out.bf16}, out.codes);
  const int64_t passes = (cols + 8 * kThreads - 1) / (8 * kThreads);
  const int lanes = cols <= kFp8Group ? 16 : cols <= 512 ? 64 : kThreads;
  auto* k = lanes == 16   ? (vec ? add_rmsnorm_kernel<16, 1, true> : add_rmsnorm_kernel<16, 1, false>)
            : lanes == 64 ? (vec ? add_rmsnorm_kernel<64, 1, true> : add_rmsnorm_kernel<64, 1, false>)
            : passes <= 1 ? (vec ? add_rmsnorm_kernel<kThreads, 1, true> : add_rmsnorm_kernel<kThreads, 1, false>)
            : passes <= 2 ? (vec ? add_rmsnorm_kernel<kThreads, 2, true> : add_rmsnorm_kernel<kThreads, 2, false>)
            : passes <= 3 ? (vec ? add_rmsnorm_kernel<kThreads, 3, true> : add_rmsnorm_kernel<kThreads, 3, false>)
            : passes <= 4 ? (vec ? add_rmsnorm_kernel<kThreads, 4, true> : add_rmsnorm_kernel<kThreads, 4, false>)
                          : (vec ? add_rmsnorm_kernel<kThreads, 0, true> : add_rmsnorm_kernel<kThreads, 0, false>);
  const int64_t per = kThreads / lanes;
  for (int64_t first = 0; first < rows; first += kMaxGrid * per) {
    const int64_t n = std::min(rows - first, kMaxGrid * per), at = first * cols;
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((n + per - 1) / per)), dim3(kThreads), 0, stream, behind(x, at),
                       behind(r, at), n, cols, weight, eps, behind(sum, at), behind(out, first, cols));
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_silu_mul(const uint16_t* gate_up, int64_t rows, int64_t cols, const RowOutputs& out,
                           hipStream_t stream) {
  auto* k = aligned(cols, {gate_up, out.bf16}, out.codes) ? silu_mul_kernel<true> : silu_mul_kernel<false>;
  const int64_t chunks = chunks_of(cols), step = place_rows(chunks);
  for (int64_t first = 0; first < rows; first += step) {
    const int64_t n = std::min(rows - first, step);
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(place_grid(n, chunks))), dim3(kThreads), 0, stream,
                       gate_up + first * 2 * cols, n, cols, behind(out, first, cols));
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_fp8_quantize(const uint16_t* x, int64_t rows, int64_t cols, int block_rows, uint8_t* codes,
                               float* scales, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  const bool vec = aligned(cols, {x}, codes);
  const bool blocks = block_rows == kFp8Group;
  const int64_t across = (cols + kFp8Group - 1) / kFp8Group;
  const int64_t chunks = chunks_of(cols), step = blocks ? kMaxGrid / across * kFp8Group : place_rows(chunks);
  if (step == 0) return hipErrorInvalidValue;  // (2^31 - 127 columns or more in blocks)
  for (int64_t first = 0; first < rows; first += step) {
    const int64_t n = std::min(rows - first, step), at = first * cols;
    const dim3 t(kThreads);
    if (blocks) {
      const dim3 g(static_cast<unsigned>((n + kFp8Group - 1) / kFp8Group * across));
      auto* k = vec ? quantize_blocks_kernel<true> : quantize_blocks_kernel<false>;
      hipLaunchKernelGGL(k, g, t, 0, stream, x + at, n, cols, codes + at, scales + first / kFp8Group * across);
    } else {
      auto* k = vec ? quantize_rows_kernel<true> : quantize_rows_kernel<false>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(place_grid(n, chunks))), t, 0, stream, x + at, n, cols,
                         behind(RowOutputs{nullptr, codes, scales}, first, cols));
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace uqm
