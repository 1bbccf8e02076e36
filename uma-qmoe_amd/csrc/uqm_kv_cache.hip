// Keys and values into a paged cache, quantised as they are written, and back
// (layout in uqm_kv.h).
//
// A row is one token's head: 8 values a lane, 8, 16 or 32 lanes a row (head sizes
// up to 64, 128, 256), so a row's maximum is three to five exchanges inside the
// wave and nothing is read twice. Neighbouring rows of a workgroup are
// neighbouring tokens of one head, which are neighbours in the cache.
#include "uqm_device.h"
#include "uqm_fp8_codes.h"
#include "uqm_kv.h"

#include <algorithm>

namespace uqm {
namespace {

constexpr int kThreads = 256;

template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t m) {
  if constexpr (LANES == 32) m = max_step<16>(m);
  if constexpr (LANES >= 16) m = max_step<8>(m);
  m = max_step<4>(m);
  m = max_step<2>(m);
  return max_step<1>(m);
}

// Place of position p of a sequence, as a row of the cache's [pages, page_size] for
// head h; -1: no page.
__device__ __forceinline__ int64_t place_of(const KvPages& c, const PageTable& t, int64_t b, int32_t p, int h) {
  const int32_t i = p >> c.page_log2;
  const int32_t page = i < t.width ? t.table[b * t.stride + i] : -1;
  if (page < 0 || page >= c.pages) return -1;
  return (((static_cast<int64_t>(page) * c.kv_heads + h) << c.page_log2) | (p & ((1 << c.page_log2) - 1)));
}

template <int LANES, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendArgs a) {
  constexpr int kRows = kThreads / LANES;
  const bool is_value = blockIdx.z != 0;
  const KvRows& in = is_value ? a.value : a.key;
  const int c = 8 * (threadIdx.x % LANES);
  const int32_t rows = a.cache.kv_heads * a.tokens;  // below 2^31
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t start = a.starts[b];
    const int32_t count = a.counts != nullptr ? min(a.counts[b], a.tokens) : a.tokens;
    // (lanes behind the last row stay for the exchanges, with no place)
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < rows; first += static_cast<int64_t>(gridDim.x) * kRows) {
      const int64_t at = first + threadIdx.x / LANES;
      const int32_t r = static_cast<int32_t>(at < rows ? at : rows - 1);
      const int32_t h = r / a.tokens, j = r - h * a.tokens;
      const int64_t p = start + j;
      int64_t place = -1;
      if (at < rows && j < count && p >= 0 && p <= INT32_MAX)
        place = place_of(a.cache, a.pages, b, static_cast<int32_t>(p), h);
      const bool mine = place >= 0 && c < a.cache.dim;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (mine) v = ldg16(in.data + b * in.batch + h * in.head + j * in.token + c);
      if constexpr (FP8) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = bf16lo(w[i]);
          f[2 * i + 1] = bf16hi(w[i]);
        }
        const float d = scale_of(row_max<LANES>(magnitude8(f)));
        const float inv = 1.0f / d;
        if (mine) {
          const uint2 codes = make_uint2(pack_fp8x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                         pack_fp8x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
          uint8_t* out = static_cast<uint8_t*>(is_value ? a.cache.value : a.cache.key);
          *reinterpret_cast<uint2*>(out + place * a.cache.dim + c) = codes;
          if (c == 0) (is_value ? a.cache.value_scales : a.cache.key_scales)[place] = d;
        }
      } else if (mine) {
        uint16_t* out = static_cast<uint16_t*>(is_value ? a.cache.value : a.cache.key);
        *reinterpret_cast<uint4*>(out + place * a.cache.dim + c) = v;
      }
    }
  }
}

template <int LANES, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvReadArgs a) {
  constexpr int kRows = kThreads / LANES;
  const bool is_value = blockIdx.z != 0;
  const int c = 8 * (threadIdx.x % LANES);
  if (c >= a.cache.dim) return;
  const int32_t rows = a.cache.kv_heads * a.length;  // below 2^31
  uint16_t* out = is_value ? a.value : a.key;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int32_t length = a.lengths[b];
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < rows; first += static_cast<int64_t>(gridDim.x) * kRows) {
      const int64_t at = first + threadIdx.x / LANES;
      if (at >= rows) break;
      const int32_t h = static_cast<int32_t>(at) / a.length, p = static_cast<int32_t>(at) - h * a.length;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      const int64_t place = p < length ? place_of(a.cache, a.pages, b, p, h) : -1;
      if (place >= 0) {
        if constexpr (FP8) {
          const uint2 q = *reinterpret_cast<const uint2*>(
              static_cast<const uint8_t*>(is_value ? a.cache.value : a.cache.key) + place * a.cache.dim + c);
          const float d = (is_value ? a.cache.value_scales : a.cache.key_scales)[place];
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, false), lo2 = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, true);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, false), hi2 = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, true);
          v = make_uint4(pack_bf16x2(lo[0] * d, lo[1] * d), pack_bf16x2(lo2[0] * d, lo2[1] * d),
                         pack_bf16x2(hi[0] * d, hi[1] * d), pack_bf16x2(hi2[0] * d, hi2[1] * d));
        } else {
          v = ldg16(static_cast<const uint16_t*>(is_value ? a.cache.value : a.cache.key) + place * a.cache.dim + c);
        }
      }
      *reinterpret_cast<uint4*>(out + ((b * a.cache.kv_heads) * static_cast<int64_t>(a.length) + at) * a.cache.dim + c) = v;
    }
  }
}

// Workgroups for `rows` rows of each of `batch` sequences, keys and values. Rows
// beyond 2^20 workgroups (and sequences beyond 65535) are taken in rounds.
dim3 grid_of(int64_t rows, int64_t batch, int lanes) {
  const int64_t per = kThreads / lanes;
  return dim3(static_cast<unsigned>(std::min<int64_t>((rows + per - 1) / per, 1 << 20)),
              static_cast<unsigned>(std::min<int64_t>(batch, 65535)), 2);
}

}  // namespace

#define UQM_KV_LAUNCH(KERNEL, GRID_ROWS)                                                              \
  do {                                                                                                \
    const bool fp8 = a.cache.key_scales != nullptr;                                                   \
    const int lanes = a.cache.dim <= 64 ? 8 : a.cache.dim <= 128 ? 16 : 32;                           \
    const dim3 grid = grid_of(GRID_ROWS, a.batch, lanes);                                             \
    if (lanes == 8) {                                                                                 \
      if (fp8) KERNEL<8, true><<<grid, kThreads, 0, stream>>>(a);                                     \
      else KERNEL<8, false><<<grid, kThreads, 0, stream>>>(a);                                        \
    } else if (lanes == 16) {                                                                         \
      if (fp8) KERNEL<16, true><<<grid, kThreads, 0, stream>>>(a);                                    \
      else KERNEL<16, false><<<grid, kThreads, 0, stream>>>(a);                                       \
    } else {                                                                                          \
      if (fp8) KERNEL<32, true><<<grid, kThreads, 0, stream>>>(a);                                    \
      else KERNEL<32, false><<<grid, kThreads, 0, stream>>>(a);                                       \
    }                                                                                                 \
    return hipGetLastError();                                                                         \
  } while (0)

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t stream) {
  UQM_KV_LAUNCH(kv_append_kernel, static_cast<int64_t>(a.cache.kv_heads) * a.tokens);
}

hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t stream) {
  UQM_KV_LAUNCH(kv_read_kernel, static_cast<int64_t>(a.cache.kv_heads) * a.length);
}

}  // namespace uqm
