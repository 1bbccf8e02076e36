// Keys and values into a paged cache, quantised as they are written, and back
// (layout in uqm_kv.h). Both are bound by memory.
//
// A row is one token's head, 16 values a lane, so 4, 8 or 16 lanes a row (head sizes
// up to 64, 128, 256) find its maximum by two to four exchanges, and nothing is read
// twice. Which 16 goes by the stores, which should be whole segments: neighbouring ones
// for 8-bit codes, two chunks of 8, half a row apart, for BF16.
// A workgroup takes a tile of neighbouring tokens of one head, which are neighbours in
// the cache (or of several heads where a call has few tokens), a thread its part of
// one key and one value.
// 8 x 16 heads of 128 in 8 bits: up to 4095 tokens appended 68 us, 4.8 TB/s (68.9 with
// two chunks a lane; 114 with 8 values a lane and keys and values apart), up to 8191
// read back 141 us, 4.9 TB/s (148 with neighbouring values; 161 with two rows a
// thread, for the occupancy).
#include "uqm_device.h"
#include "uqm_fp8_codes.h"
#include "uqm_kv.h"

#include <algorithm>

namespace uqm {
namespace {

constexpr int kThreads = 256;

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
// Bits of the largest magnitude of a row (a NaN is above every other value) of which
// this lane has the BF16 pairs of x and y.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(const uint4 x, const uint4 y) {
  const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_u16x2(m, w[i] & 0x7FFF7FFFu);
  m = max(m << 16, m & 0xFFFF0000u);
  if constexpr (LANES >= 16) m = max_step<8>(m);
  if constexpr (LANES >= 8) m = max_step<4>(m);
  m = max_step<2>(m);
  return max_step<1>(m);
}

// Place of position p of sequence b, as a row of the cache's [pages, page_size] for
// head h; -1: no page.
__device__ __forceinline__ int64_t place_of(const KvPages& c, const int32_t* table, int32_t width, int32_t p, int h) {
  const int32_t i = p >> c.page_log2;
  const int32_t page = i < width ? table[i] : -1;
  if (page < 0 || page >= c.pages) return -1;
  return (((static_cast<int64_t>(page) * c.kv_heads + h) << c.page_log2) | (p & ((1 << c.page_log2) - 1)));
}

// This thread's row: token `first` + r % 2^token_log2 of head (block of heads) + r / 2^token_log2.
template <int LANES>
struct Row {
  int64_t token;
  int head;
  __device__ __forceinline__ Row(int64_t first, int token_log2) {
    const int r = threadIdx.x / LANES;
    token = first + (r & ((1 << token_log2) - 1));
    head = blockIdx.y * (kThreads / LANES >> token_log2) + (r >> token_log2);
  }
};

// Two BF16 pairs as four codes.
__device__ __forceinline__ uint32_t codes_of(uint32_t a, uint32_t b, float inv) {
  return pack_fp8x4(bf16lo(a) * inv, bf16hi(a) * inv, bf16lo(b) * inv, bf16hi(b) * inv);
}

template <int LANES, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendArgs a, int token_log2) {
  // (16 codes next to each other, or two chunks of 8 values: whole segments are stored)
  constexpr int kNext = FP8 ? 8 : 8 * LANES;
  const int c = (FP8 ? 16 : 8) * (threadIdx.x % LANES);
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int64_t start = a.starts[b];
    const int32_t count = a.counts != nullptr ? min(a.counts[b], a.tokens) : a.tokens;
    const int32_t* table = a.pages.table + b * a.pages.stride;
    for (int64_t first = static_cast<int64_t>(blockIdx.x) << token_log2; first < count; first += static_cast<int64_t>(gridDim.x) << token_log2) {
      const Row<LANES> row(first, token_log2);
      const int64_t p = start + row.token;
      int64_t place = -1;  // (lanes without one stay for the exchanges)
      if (row.token < count && row.head < a.cache.kv_heads && p >= 0 && p <= INT32_MAX)
        place = place_of(a.cache, table, a.pages.width, static_cast<int32_t>(p), row.head);
      const bool mine[2] = {place >= 0 && c < a.cache.dim, place >= 0 && c + kNext < a.cache.dim};
      uint4 w[2][2];
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const KvRows& in = kind == 0 ? a.key : a.value;
        const uint16_t* from = in.data + b * in.batch + row.head * in.head + row.token * in.token + c;
#pragma unroll
        for (int i = 0; i < 2; ++i) w[kind][i] = mine[i] ? ldg16(from + kNext * i) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        void* out = kind == 0 ? a.cache.key : a.cache.value;
        if constexpr (FP8) {
          const uint4 x = w[kind][0], y = w[kind][1];
          const float d = scale_of(row_max<LANES>(x, y));
          const float inv = 1.0f / d;
          if (mine[0]) {
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + place * a.cache.dim + c) =
                make_uint4(codes_of(x.x, x.y, inv), codes_of(x.z, x.w, inv), codes_of(y.x, y.y, inv), codes_of(y.z, y.w, inv));
            if (c == 0) (kind == 0 ? a.cache.key_scales : a.cache.value_scales)[place] = d;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (mine[i]) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + place * a.cache.dim + c + kNext * i) = w[kind][i];
        }
      }
    }
  }
}

__device__ __forceinline__ uint32_t read_pair(uint32_t codes, bool hi, float d) {
  const auto v = hi ? __builtin_amdgcn_cvt_pk_f32_fp8(codes, true) : __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  return pack_bf16x2(v[0] * d, v[1] * d);
}

template <int LANES, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvReadArgs a, int token_log2) {
  const int c = 8 * (threadIdx.x % LANES);  // chunks at c and c + 8 * LANES
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int32_t length = min(a.lengths[b], a.length);
    const int32_t* table = a.pages.table + b * a.pages.stride;
    for (int64_t first = static_cast<int64_t>(blockIdx.x) << token_log2; first < a.length; first += static_cast<int64_t>(gridDim.x) << token_log2) {
      const Row<LANES> row(first, token_log2);
      if (row.token >= a.length || row.head >= a.cache.kv_heads) continue;
      const int64_t place = row.token < length ? place_of(a.cache, table, a.pages.width, static_cast<int32_t>(row.token), row.head) : -1;
      uint4 q[2][2];
      float d[2];
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const void* data = kind == 0 ? a.cache.key : a.cache.value;
        if constexpr (FP8) d[kind] = place >= 0 ? (kind == 0 ? a.cache.key_scales : a.cache.value_scales)[place] : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = c + 8 * LANES * i;
          q[kind][i] = make_uint4(0u, 0u, 0u, 0u);
          if (place < 0 || at >= a.cache.dim) continue;
          if constexpr (FP8) {
            const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(data) + place * a.cache.dim + at);
            q[kind][i].x = x.x, q[kind][i].y = x.y;
          } else {
            q[kind][i] = ldg16(static_cast<const uint16_t*>(data) + place * a.cache.dim + at);
          }
        }
      }
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        uint16_t* out = (kind == 0 ? a.key : a.value) + ((b * a.cache.kv_heads + row.head) * a.length + row.token) * a.cache.dim;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = c + 8 * LANES * i;
          if (at >= a.cache.dim) continue;
          const uint4 x = q[kind][i];
          *reinterpret_cast<uint4*>(out + at) = !FP8 ? x : make_uint4(read_pair(x.x, false, d[kind]), read_pair(x.x, true, d[kind]),
                                                                     read_pair(x.y, false, d[kind]), read_pair(x.y, true, d[kind]));
        }
      }
    }
  }
}

// Tiles of `tokens` tokens and `heads` heads of `rows` rows. Token tiles beyond 2^20,
// and sequences beyond 65535, are taken in rounds.
struct Tiling {
  dim3 grid;
  int token_log2;
};
Tiling tiling_of(int64_t tokens, int heads, int64_t batch, int rows) {
  Tiling t;
  t.token_log2 = 0;
  while ((1 << t.token_log2) < std::min<int64_t>(tokens, rows)) ++t.token_log2;
  const int64_t token_tiles = (tokens + (1 << t.token_log2) - 1) >> t.token_log2;
  const int per = rows >> t.token_log2;
  t.grid = dim3(static_cast<unsigned>(std::min<int64_t>(token_tiles, 1 << 20)), (heads + per - 1) / per,
                static_cast<unsigned>(std::min<int64_t>(batch, 65535)));
  return t;
}

template <int LANES>
hipError_t launch(const KvAppendArgs& a, hipStream_t stream) {
  const Tiling t = tiling_of(a.tokens, a.cache.kv_heads, a.batch, kThreads / LANES);
  if (a.cache.key_scales != nullptr) kv_append_kernel<LANES, true><<<t.grid, kThreads, 0, stream>>>(a, t.token_log2);
  else kv_append_kernel<LANES, false><<<t.grid, kThreads, 0, stream>>>(a, t.token_log2);
  return hipGetLastError();
}
template <int LANES>
hipError_t launch(const KvReadArgs& a, hipStream_t stream) {
  const Tiling t = tiling_of(a.length, a.cache.kv_heads, a.batch, kThreads / LANES);
  if (a.cache.key_scales != nullptr) kv_read_kernel<LANES, true><<<t.grid, kThreads, 0, stream>>>(a, t.token_log2);
  else kv_read_kernel<LANES, false><<<t.grid, kThreads, 0, stream>>>(a, t.token_log2);
  return hipGetLastError();
}
template <typename ARGS>
hipError_t launch_for_dim(const ARGS& a, hipStream_t stream) {
  if (a.cache.dim <= 64) return launch<4>(a, stream);
  if (a.cache.dim <= 128) return launch<8>(a, stream);
  return launch<16>(a, stream);
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t stream) { return launch_for_dim(a, stream); }
hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t stream) { return launch_for_dim(a, stream); }

}  // namespace uqm
