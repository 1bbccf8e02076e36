// Attention of one new token per sequence over a paged key-value cache (layout in
// uqm_kv.h):
//   s_p = scale * sum_i q_i k[p, i],   max(0, length - window) <= p < length
//   out = sum_p softmax(s)_p v[p]
// in one pass over the cache with the running maximum m, sum l and output o of the
// softmax (base 2: s and m carry the factor log2 e).
//
// Bound by memory: a key and its value are read for at most 16 query heads, some
// 4 to 64 operations a byte. 64 sequences of 4001 to 8191 tokens, 16 heads of 128 in
// e4m3: 254 us, 6.5 TB/s; 32 heads on 8 over 131071 tokens in BF16 84 us, 6.4 TB/s; 32
// sequences of up to 2047, 16 heads in BF16, 48 us, 5.6 TB/s. Those are calls that begin
// from rest; without a pause the card throttles after some 3 ms, and they take 310, 91 to
// 94 and 51 to 53. Times of variants, further below, are of calls without a pause. With
// products and softmax left out the times were the same.
// What is computed goes to the matrix cores all the same, since the vector unit would
// be the limit from four query heads a key head on. Everything stays in the wave's
// registers: no exchange, no shared memory in the loop, but for the maximum over four
// lanes.
//   - scores transposed, S^T = K Q^T (16 keys x 16 queries, v_mfma_f32_16x16x32_bf16):
//     a lane gives 8 neighbouring dimensions of one key, which lie next to each other
//     in a page, and gets scores of one query (lane % 16) and four keys
//     (4 (lane / 16) .. + 3). In which order dimensions are summed up is free, so
//     that 8-bit keys are loaded 16 at a time for two products.
//   - output transposed, O^T = V^T P^T: the sum over positions is free in its order,
//     too. So a lane's eight weights, of keys 16 t + 4 (lane / 16) + r, are its operand
//     as they are, and the other operand needs, of one dimension, the same eight keys:
//     a lane loads DP / 16 neighbouring dimensions of each of its eight keys (whole
//     rows of a page, 16 lanes a row), and pairs of keys are put together by one
//     v_perm each. Product i then holds dimensions lane % 16 * DP / 16 + i.
//   - e4m3 codes become BF16 exactly (v_cvt_scalef32_pk_bf16_fp8); a key's scale
//     multiplies its score, a value's scale its weight, both in FP32.
//   - a weight is split into two BF16 numbers, its rounding and the rest (together off
//     by 2^-16 of it, where one would be off by 2^-8, as much as the output's own
//     rounding). Up to 8 query heads, the products' 16 columns hold the rounded
//     weights in the lower and the rests in the upper half, which costs nothing; with
//     more of them there is a second product.
//
// Work is dealt out in tiles of 128 positions, 32 of each of a workgroup's four waves.
// The tiles of all sequences, one behind the other, are cut into columns of the same
// number of tiles, whatever the lengths are; a column has a workgroup for each key head,
// which go through the same positions side by side (that a head's workgroups took its
// positions one after the other instead cost 2 to 8%). A workgroup finds its column
// from the lengths on the device. What it has of a sequence that other columns also work
// on goes to its two places in the workspace (for the first and the last of its
// sequences), and a second launch joins these (a wave or a workgroup has a head of a
// sequence, or, where there are many, a wave a head of a column). Keys, values and
// queries of the next tile are on their way while one is computed, also across the end
// of a sequence (255 sequences of 50 to 150 tokens 41 us, with a start of its own for
// each 50).
// Where no sequence can have more than four tiles (eight, where there are workgroups for
// half of the compute units all the same) a workgroup takes a sequence's head, without
// that bookkeeping and without a second launch (one token over 77 positions, 16 heads,
// 4.5 us in a graph; 5.2 with the bookkeeping).
#include "uqm_device.h"
#include "uqm_kv.h"
#include "uqm_stage.h"

#include <algorithm>

namespace uqm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kWavePositions = 32, kTile = kWaves * kWavePositions;
// Workgroups of the main launch per compute unit. More of them read no faster, but
// leave more parts: 2, 3, 4 and 8 for 131071 tokens 94, 97, 96 and 102 us, for 32
// sequences of up to 2047 in BF16 52, 53, 56 and 55.
constexpr int kGroupsPerCu = 2;
// Up to this many parts a sequence on average a wave joins those of a head: 13 sequences
// (10 parts) 12.5 us, by workgroups 15.4; one of 4001 tokens (32) 13.7, by workgroups 12.0.
constexpr int kFewParts = 16;
constexpr int kWavesPerCu = 32;  // that there is room for
// Up to this many tiles a head is one workgroup's, a tile 1 us: 4 tiles 7.7 us and in
// parts 8.4; 8 tiles 11.6 and 8.5. (What a compute unit alone can load: with eight waves
// instead of four on it, 1000 positions 11.8 us.)
constexpr int kDirectTiles = 4;
// The same where that makes a workgroup for half of the compute units or more, so that
// parts would only add their joins. Heads of 128, sequences of 10 to 100% and of 90 to
// 100% of six tiles, whole and in parts: 32 of 28 heads on 4 in e4m3 10.1 and 10.6 us, in
// parts 12.5 and 15.7; 8 of 16 heads in BF16 14.5 and 14.9, in parts 13.0 and 16.9. Of
// eight tiles: 12.2 and 12.7 against 15.4 and 15.2; 18.1 and 19.0 against 16.9 and 17.9;
// 64 of 16 heads in BF16 64.8 and 89.5 against 57.8 and 92.2. Heads of 64: a quarter less
// than in parts on average. Of 16 tiles the longest sequence is waited for: 32 of 32
// heads on 8 in BF16 37.2 and 49.4, in parts 32.6 and 55.2.
// (It goes by tiles alone: the BF16 pairs that are slower whole lose 6 to 12%.)
constexpr int kManyDirectTiles = 8;

__device__ __forceinline__ f32x4_t mfma(const uint4 a, const uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// Codes 0, 1 (hi: 2, 3) of w as a BF16 pair; exact.
template <bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}
constexpr uint32_t kOutside = 0x80000000u;  // an offset behind every buffer's bytes
constexpr int kOnce = 2;                    // a load whose lines are not kept (nontemporal)
template <int HINT>
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t buf, uint32_t at) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buf, at, 0, HINT));
}
__device__ __forceinline__ float4 as_float4(uint4 w) {
  return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
}
// A barrier that waits for what the wave has in shared memory, not for its loads.
__device__ __forceinline__ void local_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// The value of lane ^ 8.
__device__ __forceinline__ float other_half(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));  // row_ror:8
}

// Lengths and page tables are read where all lanes want the same entry: through the
// scalar cache, so that a wait for an entry is none for the keys and values that are
// on their way (vector loads arrive in order). Nothing in a launch writes them.
typedef const __attribute__((address_space(4))) int32_t* Indexes;
__device__ __forceinline__ Indexes indexes(const int32_t* p) { return reinterpret_cast<Indexes>(reinterpret_cast<uintptr_t>(p)); }

struct Plan {
  int32_t columns;      // shares that the tiles of all sequences are cut into, each of a workgroup per head
  int32_t query_rows;   // query heads of a workgroup (at most)
  int32_t query_tiles;  // workgroups side by side for the query heads of a key head
  bool whole;           // a sequence is a column, whatever its length
};

// A sequence's units are its tiles from tile0 on; one without a position has one, too,
// which writes the zeros.
struct Sequence {
  int32_t length, first;  // positions seen: first .. length - 1
  int32_t tile0, units;
};
__device__ __forceinline__ Sequence sequence_of(const PagedAttentionArgs& a, int32_t given) {
  Sequence s;
  s.length = min(max(given, 0), a.pages.width << a.cache.page_log2);
  s.first = s.length > a.window ? s.length - a.window : 0;
  s.tile0 = static_cast<uint32_t>(s.first) / kTile;
  s.units = max(1, static_cast<int32_t>(static_cast<uint32_t>(s.length + kTile - 1) / kTile) - s.tile0);
  return s;
}

// Sum over the lanes up to this one; over all.
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int32_t wave_total(int32_t v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Units of sequences before `end`, and of all (below 2^31): four lengths a lane at once.
__device__ __forceinline__ int32_t units_before(const PagedAttentionArgs& a, int32_t end, int32_t* all) {
  constexpr int kAtOnce = 4;
  int32_t before = 0, total = 0;
  for (int32_t block = static_cast<int32_t>(threadIdx.x & 63); block < a.batch; block += 64 * kAtOnce) {
    int32_t given[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) given[i] = block + 64 * i < a.batch ? a.lengths[block + 64 * i] : 0;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int32_t units = block + 64 * i < a.batch ? sequence_of(a, given[i]).units : 0;
      total += units;
      before += block + 64 * i < end ? units : 0;
    }
  }
  *all = wave_total(total);
  return wave_total(before);
}
__device__ __forceinline__ int32_t units_per_column(int32_t units, const Plan& plan) {
  return (units + plan.columns - 1) / plan.columns;
}

// One unit of a workgroup's share, as the loop needs it.
struct Unit {
  int32_t b, tile, length, first;
  bool there, starts, ends;  // whether there is one; whether it is its sequence's first, or last
};

// A workgroup's share: units [at, end) of the sequences one after the other. Lengths
// are held 64 at a time, a lane each, so that the next sequence's is at hand.
template <bool WHOLE>
struct Share {
  int32_t at, end;
  int32_t b, base;       // the sequence of unit `at` (or the one before) and its first unit
  int32_t block, given;  // this lane's length is that of sequence block + lane
  Sequence seq;

  __device__ __forceinline__ void load_block(const PagedAttentionArgs& a) {
    const int32_t mine = block + static_cast<int32_t>(threadIdx.x & 63);
    given = mine < a.batch ? a.lengths[mine] : 0;
    asm volatile("" : "+v"(given));  // (the wait for it is here, not with every use, where it would be one for keys and values)
  }
  __device__ __forceinline__ void enter(const PagedAttentionArgs& a) {
    seq = sequence_of(a, __builtin_amdgcn_readlane(given, b - block));
  }
  __device__ __forceinline__ int32_t scan_block(const PagedAttentionArgs& a) const {
    return wave_scan(block + static_cast<int32_t>(threadIdx.x & 63) < a.batch ? sequence_of(a, given).units : 0);
  }
  // Column `column`; false: there is nothing for it.
  __device__ __forceinline__ bool find(const PagedAttentionArgs& a, const Plan& plan, int32_t column) {
    base = 0;
    if constexpr (WHOLE) {  // (a sequence to a column)
      b = column;
      seq = sequence_of(a, *indexes(a.lengths + b));
      at = 0;
      end = seq.units;
      return true;
    }
    block = 0;
    load_block(a);
    int32_t upto = scan_block(a), units = __builtin_amdgcn_readlane(upto, 63);
    if (a.batch > 64) units_before(a, 0, &units);
    const int32_t per = units_per_column(units, plan);
    at = column * per;
    end = min(at + per, units);
    if (at >= end) return false;
    int before;  // sequences that end at or before `at`
    // (`at` is below the sum; should a caller change lengths while the kernel runs, it still ends)
    while ((before = __popcll(__ballot(base + upto <= at))) == 64) {
      if (block + 64 >= a.batch) return false;
      base += __builtin_amdgcn_readlane(upto, 63);
      block += 64;
      load_block(a);
      upto = scan_block(a);
    }
    if (before > 0) base += __builtin_amdgcn_readlane(upto, before - 1);
    b = block + before;
    enter(a);
    return b < a.batch;
  }
  __device__ __forceinline__ Unit next(const PagedAttentionArgs& a) {
    Unit u;
    u.there = at < end;
    if (!WHOLE && u.there && at - base == seq.units) {  // (every sequence has a unit: `at` is in the next one)
      base += seq.units;
      if (++b == block + 64) {
        block += 64;
        load_block(a);
      }
      enter(a);
      u.there = b < a.batch;
    }
    u.b = b;
    u.tile = seq.tile0 + (at - base);
    u.length = u.there ? seq.length : 0;
    u.first = seq.first;
    u.starts = WHOLE || at == base;
    u.ends = at - base == seq.units - 1;
    ++at;
    return u;
  }
};

// A part of a row, a wave's or a workgroup's: weights relative to 2^most, their sum, the
// sum of weighted values. most is -inf for a part that saw nothing (sum 0, values 0) and
// for one all of whose scores were -inf (sum NaN: 0 / 0 unless other parts have finite
// scores). A factor that underflows to 0 multiplies like any other, so that a NaN or an
// infinity of a part far below the others stays one, as it does within a wave.
__device__ __forceinline__ float part_factor(float most, float all) {
  return most == -INFINITY ? (all == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(most - all);
}
// A part's sum relative to 2^all, f its factor: what has no weight is left out.
__device__ __forceinline__ float part_sum(float most, float all, float f, float sum) {
  return most == -INFINITY && all != -INFINITY ? 0.0f : f * sum;
}

// (registers for one, two or three workgroups a compute unit, so that none spills)
template <int DP, bool FP8, bool DUP, bool PAD, bool WHOLE>
__global__ __launch_bounds__(kThreads, DP == 256 && !FP8 ? 1 : DP == 256 || !FP8 || PAD ? 2 : 3) void paged_attention_kernel(PagedAttentionArgs a, Plan plan) {
  constexpr int kRows = DUP ? 8 : 16;      // query heads that there is room for
  constexpr int kVec = DP / 16;            // dimensions of a value row that a lane holds
  constexpr int kStep = FP8 ? 64 : 32;     // dimensions of one load of 16 keys
  constexpr int kLoads = DP / kStep;
  constexpr int kVWords = FP8 ? kVec / 4 : kVec / 2;
  // Lines that another load of the same rows takes a part of are kept: 8-bit keys (two
  // loads to a line; 64 sequences 310 us, not kept 328), keys of rows that do not begin
  // with a line (32 sequences of 2001 to 6001, heads of 80 in BF16 135 and 151), values of
  // 32 bytes a lane (the same with heads of 256 411 and 432; heads of 192, whose rows end
  // within a line, 307 and 280). BF16 keys, two loads to a line as well, are faster not
  // kept all the same (131071 tokens 91 to 94 us, kept 95 to 100).
  constexpr int kKeyHint = FP8 || PAD ? 0 : kOnce, kValueHint = kVWords > 4 ? 0 : kOnce;
  constexpr int kRowStride = DP + 4;       // (rows of the join four banks apart)
  constexpr bool kSharedQuery = DP == 256;  // (there are no registers for them beside keys and values on their way)
  __shared__ uint4 shared_query[kSharedQuery ? DP / 32 : 1][64];
  __shared__ float part_o[kWaves][kRows][kRowStride];
  __shared__ float part_m[kWaves][kRows], part_l[kWaves][kRows];

  const KvPages& kv = a.cache;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int dim = PAD ? kv.dim : DP;
  const int group = a.heads / kv.kv_heads, heads = kv.kv_heads * plan.query_tiles;
  const int row_bytes = FP8 ? dim : 2 * dim;

  const int32_t column = blockIdx.x / heads, index = blockIdx.x - column * heads;
  const int h = index / plan.query_tiles, query0 = (index - h * plan.query_tiles) * plan.query_rows;
  const int rows = min(plan.query_rows, group - query0);
  Share<WHOLE> share;
  if (!share.find(a, plan, column)) return;

  // ---- loads of a unit's 32 positions of this wave, as two blocks of 16 ----
  // (what lies behind a sequence's end, or behind the share's, counts as no page and
  // costs no memory; the loop has no branch around its loads, behind which a wait could
  // not tell them apart)
  auto entry_of = [&](const Unit& u, int s) -> int32_t {
    const int32_t p = u.tile * kTile + wave * kWavePositions + 16 * s;
    const int32_t* table = a.pages.table + u.b * a.pages.stride;
    return *indexes(u.length > 0 ? table + (min(p, u.length - 1) >> kv.page_log2) : a.lengths);
  };
  auto page_of = [&](const Unit& u, int s, int32_t entry) -> int32_t {
    return u.tile * kTile + wave * kWavePositions + 16 * s < u.length && entry < kv.pages ? entry : -1;  // (below 0: none, too)
  };
  // (no page: page 0, whose values are masked)
  const int64_t page_rows = static_cast<int64_t>(kv.kv_heads) << kv.page_log2;
  auto place_of = [&](const Unit& u, int s, int32_t page) -> int64_t {
    const int32_t slot = (u.tile * kTile + wave * kWavePositions + 16 * s) & ((1 << kv.page_log2) - 1);
    return max(page, 0) * page_rows + ((h << kv.page_log2) | slot);
  };
  // What a lane adds to the address of a block of 16 rows, which is the wave's.
  const uint32_t key_at = n * row_bytes + 16 * g;
  const uint32_t value_at = !PAD || n * kVec < dim ? 4 * g * row_bytes + n * (4 * kVWords) : kOutside;
  // Blocks are read through buffers that end behind their last position that is seen
  // (at once where there is no page): what lies behind reads as zeros and costs
  // nothing, as do dimensions behind the last.
  auto seen_of = [&](const Unit& u, int s, int32_t page) -> int32_t {
    return page >= 0 ? min(16, u.length - (u.tile * kTile + wave * kWavePositions + 16 * s)) : 0;
  };
  uint4 k[2][kLoads];
  float4 ks[2], vs[2];
  uint32_t v[2][4][kVWords];
  auto load_keys = [&](const Unit& u, const int32_t (&page)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t place = place_of(u, s, page[s]);
      const int32_t seen = seen_of(u, s, page[s]);
      const auto buf = stage_buffer(static_cast<const uint8_t*>(kv.key) + place * row_bytes, seen * row_bytes);
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        k[s][i] = load16<kKeyHint>(buf, (!PAD || i * kStep + g * (kStep / 4) < dim ? key_at : kOutside) + 64 * i);
      if constexpr (FP8) ks[s] = as_float4(load16<0>(stage_buffer(kv.key_scales + place, seen > 0 ? 64 : 0), 16u * g));
    }
  };
  auto load_values = [&](const Unit& u, const int32_t (&page)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t place = place_of(u, s, page[s]);
      const int32_t seen = seen_of(u, s, page[s]);
      const auto buf = stage_buffer(static_cast<const uint8_t*>(kv.value) + place * row_bytes, seen * row_bytes);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t at = value_at + r * row_bytes;
        if constexpr (kVWords == 1) {
          v[s][r][0] = __builtin_amdgcn_raw_buffer_load_b32(buf, at, 0, kValueHint);
        } else if constexpr (kVWords == 2) {
          const auto w = __builtin_amdgcn_raw_buffer_load_b64(buf, at, 0, kValueHint);
          v[s][r][0] = w[0], v[s][r][1] = w[1];
        } else {
#pragma unroll
          for (int i = 0; i < kVWords / 4; ++i) {
            const uint4 w = load16<kValueHint>(buf, at + 16 * i);
            v[s][r][4 * i] = w.x, v[s][r][4 * i + 1] = w.y, v[s][r][4 * i + 2] = w.z, v[s][r][4 * i + 3] = w.w;
          }
        }
      }
      if constexpr (FP8) vs[s] = as_float4(load16<0>(stage_buffer(kv.value_scales + place, seen > 0 ? 64 : 0), 16u * g));
    }
  };
  // The queries of column n (of the upper half as of the lower one), in the keys' order of dimensions.
  const int row = DUP ? n & 7 : n;
  auto load_query = [&](int32_t b, int j) {
    const int c = FP8 ? 64 * (j / 2) + 16 * g + 8 * (j % 2) : 32 * j + 8 * g;
    const int64_t at = static_cast<int64_t>(b) * a.heads + h * group + query0 + row;
    return row < rows && (!PAD || c < dim) ? ldg16(a.query + at * dim + c) : make_uint4(0u, 0u, 0u, 0u);
  };
  uint4 q[kSharedQuery ? 1 : DP / 32];
  auto load_queries = [&](int32_t b) {
    if constexpr (kSharedQuery) {
      for (int j = wave; j < DP / 32; j += kWaves) shared_query[j][lane] = load_query(b, j);
    } else {
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) q[j] = load_query(b, j);
    }
  };

  Unit unit = share.next(a), after = share.next(a);
  int32_t page[2], ahead[2], entry[2];  // pages of this unit and the next one, what the table says of the one behind
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    page[s] = page_of(unit, s, entry_of(unit, s));
    entry[s] = entry_of(after, s);
  }
  load_queries(unit.b);
  if constexpr (kSharedQuery) __syncthreads();
  load_keys(unit, page);
  __builtin_amdgcn_sched_barrier(0);  // (in this order, as in the loop)
  load_values(unit, page);
  __builtin_amdgcn_sched_barrier(0);

  const float scale = a.scale * 1.44269504088896340736f;
  const uint32_t rest = DUP && n >= 8 ? 0xFFFFFFFFu : 0u;
  f32x4_t o[kVec];
  float m = -INFINITY, l = 0.f;
  bool seen = false, from_start = unit.starts, first_head = true;
#pragma unroll
  for (int i = 0; i < kVec; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (;;) {
    const Unit behind = share.next(a);
    auto query = [&](int j) {
      if constexpr (kSharedQuery) return shared_query[j][lane];
      else return q[j];
    };
    f32x4_t s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int half = 0; half < (FP8 ? 2 : 1); ++half)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if constexpr (FP8) {
            const uint32_t lo = half == 0 ? k[t][i].x : k[t][i].z, hi = half == 0 ? k[t][i].y : k[t][i].w;
            s[t] = mfma(make_uint4(fp8_pair<false>(lo), fp8_pair<true>(lo), fp8_pair<false>(hi), fp8_pair<true>(hi)),
                        query(2 * i + half), s[t]);
          } else {
            s[t] = mfma(k[t][i], query(i), s[t]);
          }
        }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (FP8) {
        s[t][0] *= ks[t].x * scale, s[t][1] *= ks[t].y * scale, s[t][2] *= ks[t].z * scale, s[t][3] *= ks[t].w * scale;
      } else {
        s[t] *= scale;
      }
    }
    // Positions of this unit that are seen: lo <= place < hi of each block of 16.
    int lo[2], hi[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      lo[t] = max(0, unit.first - (unit.tile * kTile + wave * kWavePositions + 16 * t));
      hi[t] = seen_of(unit, t, page[t]);
    }
    const bool whole = lo[0] <= 0 && lo[1] <= 0 && hi[0] >= 16 && hi[1] >= 16;
    if (!whole) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * g + r < lo[t] || 4 * g + r >= hi[t]) s[t][r] = -INFINITY;
    }
    seen = seen || lo[0] < hi[0] || lo[1] < hi[1];
    const bool last = unit.ends || !after.there;  // of this head's part here
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ahead[t] = page_of(after, t, entry[t]);
      entry[t] = entry_of(behind, t);
    }
    if constexpr (!kSharedQuery && !WHOLE)
      if (last && after.there) load_queries(after.b);
    load_keys(after, ahead);
    __builtin_amdgcn_sched_barrier(0);

    float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    most = fmaxf(most, xor_partner<16>(most));
    most = fmaxf(most, xor_partner<32>(most));
    if (__any(most > m)) {  // (seldom after the first tiles)
      const float next = fmaxf(m, most);
      const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
      l *= keep;
#pragma unroll
      for (int i = 0; i < kVec; ++i) o[i] *= keep;
      m = next;
    }
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - from);
        l += s[t][r];
      }
    if constexpr (FP8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t][0] *= vs[t].x, s[t][1] *= vs[t].y, s[t][2] *= vs[t].z, s[t][3] *= vs[t].w;
    }
    if (!whole) {  // (what lies in places that are not seen may be NaN; values behind the last read as zeros)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (4 * g + r < lo[t] || 4 * g + r >= hi[t]) s[t][r] = 0.f;
#pragma unroll
          for (int i = 0; i < kVWords; ++i)
            if (4 * g + r < lo[t]) v[t][r][i] = 0u;
        }
    }
    // Weights as BF16 pairs: rounded (p), and what the rounding left (x).
    uint32_t p[4], x[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float y0 = s[t][2 * r], y1 = s[t][2 * r + 1];
        const uint32_t w = pack_bf16x2(y0, y1);
        if constexpr (DUP) {
          const uint32_t z = w & rest;
          p[2 * t + r] = pack_bf16x2(y0 - bf16lo(z), y1 - bf16hi(z));
        } else {
          p[2 * t + r] = w;
          x[2 * t + r] = pack_bf16x2(y0 - bf16lo(w), y1 - bf16hi(w));
        }
      }
    const uint4 weights = make_uint4(p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {  // two dimensions: a word of each of the eight keys
      uint32_t w[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (FP8) w[t][r] = i % 4 == 0 ? fp8_pair<false>(v[t][r][i / 4]) : fp8_pair<true>(v[t][r][i / 4]);
          else w[t][r] = v[t][r][i / 2];
        }
      const uint4 even = make_uint4(perm(w[0][1], w[0][0], 0x05040100u), perm(w[0][3], w[0][2], 0x05040100u),
                                    perm(w[1][1], w[1][0], 0x05040100u), perm(w[1][3], w[1][2], 0x05040100u));
      const uint4 odd = make_uint4(perm(w[0][1], w[0][0], 0x07060302u), perm(w[0][3], w[0][2], 0x07060302u),
                                   perm(w[1][1], w[1][0], 0x07060302u), perm(w[1][3], w[1][2], 0x07060302u));
      o[i] = mfma(even, weights, o[i]);
      o[i + 1] = mfma(odd, weights, o[i + 1]);
      if constexpr (!DUP) {
        const uint4 rests = make_uint4(x[0], x[1], x[2], x[3]);
        o[i] = mfma(even, rests, o[i]);
        o[i + 1] = mfma(odd, rests, o[i + 1]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(after, ahead);
    __builtin_amdgcn_sched_barrier(0);

    if (last) {
      // ---- join of the waves; the next head's keys and values are on their way ----
      l += xor_partner<16>(l);
      l += xor_partner<32>(l);
      if (m == -INFINITY && seen) {
        if (l == 0.f) l = NAN;  // every score -inf
        else m = 0.f;           // every score -inf or NaN
      }
      if constexpr (DUP) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][r] += other_half(o[i][r]);
      }
      local_barrier();  // (the last head's join has been read)
      if (n < rows) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < kVec; i += 4)
            *reinterpret_cast<float4*>(&part_o[wave][n][kVec * (4 * g + r) + i]) = make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
        if (g == 0) {
          part_m[wave][n] = m;
          part_l[wave][n] = l;
        }
      }
      if constexpr (kSharedQuery && !WHOLE)
        if (after.there) load_queries(after.b);
      local_barrier();
      const bool complete = WHOLE || (from_start && unit.ends);
      const int64_t slot = 2 * blockIdx.x + (first_head ? 0 : 1);
      float* part = a.workspace + slot * kRows * (DP + 2);
      const int64_t query_row = static_cast<int64_t>(unit.b) * a.heads + h * group + query0;
      for (int i = threadIdx.x; i < rows * (DP / 4); i += kThreads) {
        const int r = i / (DP / 4), c = 4 * (i % (DP / 4));
        float all = part_m[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = fmaxf(all, part_m[w][r]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = part_factor(part_m[w][r], all);
          const float4 y = *reinterpret_cast<const float4*>(&part_o[w][r][c]);
          sum += part_sum(part_m[w][r], all, f, part_l[w][r]);
          acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w;
        }
        if (complete) {
          if (!PAD || c < dim) {
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
            *reinterpret_cast<uint2*>(a.out + (query_row + r) * dim + c) =
                make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          }
        } else {
          *reinterpret_cast<float4*>(part + r * DP + c) = acc;
          if (c == 0) {
            part[kRows * DP + 2 * r] = all;
            part[kRows * DP + 2 * r + 1] = sum;
          }
        }
      }
      if (WHOLE || !after.there) return;
      m = -INFINITY, l = 0.f;
      seen = false, from_start = after.starts, first_head = false;
#pragma unroll
      for (int i = 0; i < kVec; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    unit = after;
    after = behind;
#pragma unroll
    for (int t = 0; t < 2; ++t) page[t] = ahead[t];
  }
}

// Sums of parts: relative to 2^most, the weights' and those of four dimensions.
struct Joined {
  float most, sum;
  float4 acc;
};
__device__ __forceinline__ void join(Joined& x, float most, float sum, const float4& acc) {
  const float all = fmaxf(x.most, most), f = part_factor(x.most, all), h = part_factor(most, all);
  x.sum = part_sum(x.most, all, f, x.sum) + part_sum(most, all, h, sum);
  x.acc = make_float4(f * x.acc.x + h * acc.x, f * x.acc.y + h * acc.y, f * x.acc.z + h * acc.z, f * x.acc.w + h * acc.w);
  x.most = all;
}
template <int O>
__device__ __forceinline__ float lane_xor(float v) {  // (xor_partner<8> would be lane ^ 15)
  if constexpr (O == 8) return other_half(v);
  else return xor_partner<O>(v);
}
template <int O>
__device__ __forceinline__ void join_lanes(Joined& x) {
  static_assert(O >= 8, "xor_partner<4> is lane ^ 7");
  const float most = lane_xor<O>(x.most), sum = lane_xor<O>(x.sum);
  join(x, most, sum, make_float4(lane_xor<O>(x.acc.x), lane_xor<O>(x.acc.y), lane_xor<O>(x.acc.z), lane_xor<O>(x.acc.w)));
}

// Joins the parts of query heads. Of few parts a wave has a head, four dimensions a lane;
// of many (kMany) a workgroup has 32 dimensions of a head, and 32 sets of 8 lanes share the
// parts (8 heads of 128 in 512 parts: 5.4 us, with a workgroup a head 12; 4096 heads in 2 to
// 3 parts: 5.5 us with a wave a head, with a workgroup 10).
// More heads than the card has room for waves (kColumns): a wave has a head of the sequence
// that a column begins within, where that is the sequence's second one, since a wave for each
// head of each sequence goes through all lengths as many times as there are sequences. Calls
// of 50 positions in wide tables: 65536 sequences of 8 heads 1.3 ms, a wave a head 14.4; 4096
// of 16 heads 93 us and 187; 300 of 28 heads 35.5 and 37.0. Below that a wave a head: 4096 of
// one head 60 us, by columns 71.
enum class Join { kFew, kMany, kColumns };
template <int DP, Join JOIN>
__global__ __launch_bounds__(kThreads) void join_parts_kernel(PagedAttentionArgs a, Plan plan) {
  constexpr bool FEW = JOIN != Join::kMany;
  constexpr int kSpan = FEW ? DP : 32, kLanes = kSpan / 4, kSets = (FEW ? 64 : kThreads) / kLanes;
  constexpr int kSpans = DP / kSpan, kAtOnce = 4;
  const KvPages& kv = a.cache;
  const int group = a.heads / kv.kv_heads, heads = kv.kv_heads * plan.query_tiles, rows = plan.query_rows <= 8 ? 8 : 16;
  const int32_t item = FEW ? blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x / kSpans;
  int32_t b = item / a.heads;
  const int32_t head = item - b * a.heads, h = head / group;
  const int32_t tile = (head - h * group) / plan.query_rows, row = (head - h * group) - tile * plan.query_rows;
  int32_t before, per, w0, w1;
  if constexpr (JOIN == Join::kColumns) {
    const int32_t column = b + 1;
    Share<false> share;
    if (column >= plan.columns || !share.find(a, plan, column)) return;
    b = share.b;
    before = share.base;
    per = share.at / column;
    w0 = before / per;
    if (w0 != column - 1) return;  // (it begins with this column, or further back)
    w1 = min((before + share.seq.units - 1) / per, plan.columns - 1);
  } else {
    if (FEW && b >= a.batch) return;
    const Sequence seq = sequence_of(a, indexes(a.lengths)[b]);
    int32_t units = seq.units;
    before = 0;
    if (a.batch > 1) before = units_before(a, b, &units);
    per = units_per_column(units, plan);
    w0 = before / per;
    w1 = min((before + seq.units - 1) / per, plan.columns - 1);
    if (w0 >= w1) return;  // one workgroup had it all
  }
  // (a part is in its workgroup's first place but where another head came before it there)
  const int64_t stride = static_cast<int64_t>(rows) * (DP + 2);
  const int32_t first_place = before != w0 * per ? 1 : 0, index = h * plan.query_tiles + tile;
  const int lane = threadIdx.x % kLanes, set = (FEW ? threadIdx.x & 63 : threadIdx.x) / kLanes;
  const int c = (FEW ? 0 : (blockIdx.x % kSpans) * kSpan) + 4 * lane;
  Joined x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int32_t w = w0 + set; w <= w1; w += kAtOnce * kSets) {
    float most[kAtOnce], sum[kAtOnce];
    float4 y[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int32_t at = min(w + i * kSets, w1);
      const float* part = a.workspace + (2 * (at * heads + index) + (at == w0 ? first_place : 0)) * stride;
      const float2 ml = *reinterpret_cast<const float2*>(part + rows * DP + 2 * row);
      y[i] = *reinterpret_cast<const float4*>(part + row * DP + c);
      const bool there = w + i * kSets <= w1;  // (else a part that saw nothing)
      most[i] = there ? ml.x : -INFINITY;
      sum[i] = there ? ml.y : 0.f;
      y[i] = there ? y[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float all = x.most;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) all = fmaxf(all, most[i]);
    const float f = part_factor(x.most, all);
    x.sum = part_sum(x.most, all, f, x.sum);
    x.acc = make_float4(f * x.acc.x, f * x.acc.y, f * x.acc.z, f * x.acc.w);
    x.most = all;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float h = part_factor(most[i], all);
      x.sum += part_sum(most[i], all, h, sum[i]);
      x.acc.x += h * y[i].x, x.acc.y += h * y[i].y, x.acc.z += h * y[i].z, x.acc.w += h * y[i].w;
    }
  }
  if constexpr (kLanes <= 8) join_lanes<8>(x);
  if constexpr (kLanes <= 16) join_lanes<16>(x);
  if constexpr (kLanes <= 32) join_lanes<32>(x);
  if constexpr (!FEW) {
    __shared__ Joined joined[kWaves][kLanes];
    if ((threadIdx.x & 63) < kLanes) joined[threadIdx.x >> 6][lane] = x;
    __syncthreads();
    if (set != 0) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) join(x, joined[i][lane].most, joined[i][lane].sum, joined[i][lane].acc);
  }
  if (set != 0 || c >= kv.dim) return;
  const float inv = x.sum == 0.f ? 0.f : 1.0f / x.sum;
  *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(b) * a.heads + head) * kv.dim + c) =
      make_uint2(pack_bf16x2(x.acc.x * inv, x.acc.y * inv), pack_bf16x2(x.acc.z * inv, x.acc.w * inv));
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Most tiles of a sequence, from the table's width and the window: lengths are on the device.
int64_t most_tiles(const PagedAttentionArgs& a) {
  const int64_t capacity = static_cast<int64_t>(a.pages.width) << a.cache.page_log2, tiles = (capacity + kTile - 1) / kTile;
  return a.window < capacity ? std::min<int64_t>(tiles, (a.window + kTile - 2) / kTile + 1) : tiles;  // (a window begins anywhere in a tile)
}
int query_tiles(const PagedAttentionArgs& a) { return (a.heads / a.cache.kv_heads + 15) / 16; }

Plan plan_of(const PagedAttentionArgs& a, int cus) {
  Plan p;
  const int group = a.heads / a.cache.kv_heads;
  p.query_tiles = query_tiles(a);
  p.query_rows = (group + p.query_tiles - 1) / p.query_tiles;
  const bool many = 2 * static_cast<int64_t>(a.batch) * a.cache.kv_heads * p.query_tiles >= cus;
  p.whole = most_tiles(a) <= (many ? kManyDirectTiles : kDirectTiles);
  const int64_t wanted = std::max<int64_t>(1, static_cast<int64_t>(kGroupsPerCu) * cus / (a.cache.kv_heads * p.query_tiles));
  p.columns = static_cast<int32_t>(p.whole ? a.batch : std::min(a.batch * most_tiles(a), wanted));
  return p;
}

template <int DP, bool FP8, bool DUP>
void launch_main(const PagedAttentionArgs& a, const Plan& p, hipStream_t stream) {
  const unsigned groups = static_cast<unsigned>(p.columns) * a.cache.kv_heads * p.query_tiles;
  if (p.whole) {
    if (a.cache.dim == DP) paged_attention_kernel<DP, FP8, DUP, false, true><<<groups, kThreads, 0, stream>>>(a, p);
    else paged_attention_kernel<DP, FP8, DUP, true, true><<<groups, kThreads, 0, stream>>>(a, p);
  } else {
    if (a.cache.dim == DP) paged_attention_kernel<DP, FP8, DUP, false, false><<<groups, kThreads, 0, stream>>>(a, p);
    else paged_attention_kernel<DP, FP8, DUP, true, false><<<groups, kThreads, 0, stream>>>(a, p);
  }
}
template <int DP>
hipError_t launch(const PagedAttentionArgs& a, const Plan& p, int cus, hipStream_t stream) {
  const bool fp8 = a.cache.key_scales != nullptr, dup = p.query_rows <= 8;
  if (fp8 && dup) launch_main<DP, true, true>(a, p, stream);
  else if (fp8) launch_main<DP, true, false>(a, p, stream);
  else if (dup) launch_main<DP, false, true>(a, p, stream);
  else launch_main<DP, false, false>(a, p, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.whole || p.columns == 1) return e;
  const bool by_columns = a.batch * a.heads > static_cast<int64_t>(kWavesPerCu) * cus;  // (there are fewer columns than sequences then)
  const unsigned items = static_cast<unsigned>(by_columns ? p.columns - 1 : a.batch) * a.heads, groups = (items + kWaves - 1) / kWaves;
  if (by_columns) join_parts_kernel<DP, Join::kColumns><<<groups, kThreads, 0, stream>>>(a, p);
  else if (p.columns <= kFewParts * a.batch) join_parts_kernel<DP, Join::kFew><<<groups, kThreads, 0, stream>>>(a, p);
  else join_parts_kernel<DP, Join::kMany><<<items * (DP / 32), kThreads, 0, stream>>>(a, p);
  return hipGetLastError();
}

}  // namespace

bool paged_attention_fits(const PagedAttentionArgs& a) {
  return std::max<int64_t>(1, most_tiles(a)) * query_tiles(a) * a.cache.kv_heads < (int64_t{1} << 30) / std::max<int64_t>(1, a.batch);
}

size_t paged_attention_workspace(const PagedAttentionArgs& a, int cus) {
  if (a.batch == 0) return 0;
  const Plan p = plan_of(a, cus);
  if (p.whole) return 0;
  return 2 * static_cast<size_t>(p.columns) * a.cache.kv_heads * p.query_tiles * (p.query_rows <= 8 ? 8 : 16) * (padded_dim(a.cache.dim) + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& a, int cus, hipStream_t stream) {
  const Plan p = plan_of(a, cus);
  switch (padded_dim(a.cache.dim)) {
    case 64: return launch<64>(a, p, cus, stream);
    case 128: return launch<128>(a, p, cus, stream);
    default: return launch<256>(a, p, cus, stream);
  }
}

}  // namespace uqm
