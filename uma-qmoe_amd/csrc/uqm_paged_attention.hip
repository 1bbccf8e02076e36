// Attention of one new token per sequence over a paged key-value cache (layout in
// uqm_kv.h):
//   s_p = scale * sum_i q_i k[p, i],   max(0, length - window) <= p < length
//   out = sum_p softmax(s)_p v[p]
// in FP32, with the running maximum and sum of the softmax, so that the cache is
// read once; zeros where no position is seen.
#include "uqm_device.h"
#include "uqm_kv.h"

namespace uqm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

template <bool FP8>
__device__ __forceinline__ void load4(const void* data, const float* scales, int64_t place, int dim, int c, float (&v)[4]) {
  if constexpr (FP8) {
    const uint32_t q = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(data) + place * dim + c);
    const float d = scales[place];
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(q, true);
    v[0] = lo[0] * d, v[1] = lo[1] * d, v[2] = hi[0] * d, v[3] = hi[1] * d;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(data) + place * dim + c);
    v[0] = bf16lo(q.x), v[1] = bf16hi(q.x), v[2] = bf16lo(q.y), v[3] = bf16hi(q.y);
  }
}

// A workgroup per sequence and query head; each wave takes every fourth position,
// a lane four of the head's dimensions.
template <bool FP8>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(PagedAttentionArgs a) {
  __shared__ float part_ml[kWaves][2];
  __shared__ float part_o[kWaves][kMaxHeadDim];
  const KvPages& kv = a.cache;
  const int wave = threadIdx.x / 64, c = 4 * (threadIdx.x % 64), head = blockIdx.x % a.heads;
  const int64_t b = blockIdx.x / a.heads;
  const int h = head / (a.heads / kv.kv_heads);
  const bool mine = c < kv.dim;
  const int64_t capacity = static_cast<int64_t>(a.pages.width) << kv.page_log2;
  const int64_t length = max(static_cast<int64_t>(0), min(static_cast<int64_t>(a.lengths[b]), capacity));
  float q[4] = {}, o[4] = {};
  if (mine) {
    const uint2 w = *reinterpret_cast<const uint2*>(a.query + (b * a.heads + head) * kv.dim + c);
    q[0] = bf16lo(w.x), q[1] = bf16hi(w.x), q[2] = bf16lo(w.y), q[3] = bf16hi(w.y);
  }
  float m = -INFINITY, l = 0.f;
  bool seen = false;
  for (int64_t p = max(static_cast<int64_t>(0), length - a.window) + wave; p < length; p += kWaves) {
    const int32_t page = a.pages.table[b * a.pages.stride + (p >> kv.page_log2)];
    if (page < 0 || page >= kv.pages) continue;
    seen = true;
    const int64_t place = (((static_cast<int64_t>(page) * kv.kv_heads + h) << kv.page_log2) | (p & ((1 << kv.page_log2) - 1)));
    float k[4] = {}, v[4] = {};
    if (mine) {
      load4<FP8>(kv.key, kv.key_scales, place, kv.dim, c, k);
      load4<FP8>(kv.value, kv.value_scales, place, kv.dim, c, v);
    }
    const float s = a.scale * wave_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]);
    const float m_new = fmaxf(m, s), from = m_new == -INFINITY ? 0.f : m_new;
    const float keep = __expf(m - from), w = __expf(s - from);
    m = m_new;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * keep + w * v[i];
  }
  if (threadIdx.x % 64 == 0) {
    if (m == -INFINITY && seen) l == 0.f ? l = NAN : m = 0.f;  // every score -inf: 0 / 0, unless another wave has a finite one
    part_ml[wave][0] = m;
    part_ml[wave][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part_o[wave][c + i] = o[i];
  __syncthreads();
  if (static_cast<int>(threadIdx.x) >= kv.dim) return;
  float most = -INFINITY;
  for (int w = 0; w < kWaves; ++w) most = fmaxf(most, part_ml[w][0]);
  float sum = 0.f, acc = 0.f;
  for (int w = 0; w < kWaves; ++w) {
    if (most != -INFINITY && part_ml[w][0] == -INFINITY) continue;
    const float f = most == -INFINITY ? 1.f : __expf(part_ml[w][0] - most);
    sum += f * part_ml[w][1];
    acc += f * part_o[w][threadIdx.x];
  }
  a.out[(b * a.heads + head) * kv.dim + threadIdx.x] = f32_to_bf16(sum == 0.f ? 0.f : acc / sum);
}

}  // namespace

size_t paged_attention_workspace(const PagedAttentionArgs&, int) { return 0; }

hipError_t launch_paged_attention(const PagedAttentionArgs& a, int, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(a.batch * a.heads);
  if (a.cache.key_scales != nullptr) paged_attention_kernel<true><<<grid, kThreads, 0, stream>>>(a);
  else paged_attention_kernel<false><<<grid, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace uqm
