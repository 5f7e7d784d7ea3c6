// Paged K/V cache of 8-bit codes: append with rotation, and reading back.
//
// One layer holds codes [num_blocks][kv_heads][block][D] (int8, or e4m3) for
// the keys and for the values, and one fp32 scale for each (block, KV head) of
// either; a code c stands for c * scale.  A head's block is contiguous
// (block * D bytes), so that one warp writes, and one warp reads, whole lines.
//
// Append.  With M = 127 (int8) or 448 (e4m3), for each block b that the step
// writes to, and each head:
//   a  = the largest |x| of the step's tokens in the block (x: the value row,
//        or the key row rotated in fp32 and not rounded),
//   s0 = the block's scale if it holds a token of an earlier step, else 0,
//   s1 = max(s0, a / M), held as 0 below 2^-100 (such values are zeros),
//   codes of earlier tokens become round(c * (s0 / s1)) where s1 > s0, and the
//   new ones round(x / s1) within [-M, M].
// Codes past the request's end (drafts that were refused) are left alone; they
// count for nothing.  NaN is held as 0, infinities as the largest code.
#pragma once

#include <cuda_fp8.h>

#include "lvb_common.cuh"

namespace lvb {
namespace kv8 {

constexpr float kTinyScale = 0x1p-100f;

// Rounding to a code and back.  Both are the IEEE operations named here, so
// that the same inputs give the same codes everywhere.
template <bool kFp8>
struct Code {
  static constexpr float kTop = kFp8 ? 448.f : 127.f;
  static constexpr float kInvTop = 1.f / kTop;

  static __device__ __forceinline__ uint8_t encode(float y) {
    y = y == y ? fminf(fmaxf(y, -kTop), kTop) : 0.f;
    if constexpr (kFp8) {
      return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
    } else {
      return static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(y)));
    }
  }

  static __device__ __forceinline__ float decode(uint8_t c) {
    if constexpr (kFp8) {
      return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
    } else {
      return static_cast<float>(static_cast<int8_t>(c));
    }
  }
};

// The step's packed requests, and the cache they live in.
struct Step {
  const int32_t *tables;
  int64_t table_stride;
  const int32_t *computed;
  const int32_t *qsl;
  int num_seqs, num_tokens, max_query_len;
  int num_blocks, bs, hkv;
};

// Request r's query tokens [q0, q0 + qlen) and computed count; false (and the
// device error word set) when they are not a range of the batch or exceed the
// request's block table.
__device__ __forceinline__ bool request_range(const Step &s, int r, int &q0, int &qlen, int &computed) {
  q0 = s.qsl[r];
  const int q1 = s.qsl[r + 1];
  computed = s.computed[r];
  qlen = q1 - q0;
  if (q0 < 0 || qlen < 0 || q1 > s.num_tokens || computed < 0 || qlen > s.max_query_len ||
      static_cast<int64_t>(computed) + qlen > s.table_stride * s.bs) {
    record_device_error(LVB_DEVERR_INDEX);
    return false;
  }
  return true;
}

struct AppendArgs {
  Step step;
  const uint16_t *query;  // null: no queries
  int64_t query_stride;
  uint16_t *query_out;
  int64_t query_out_stride;
  const uint16_t *key, *value;
  int64_t key_stride, value_stride;
  const int32_t *positions;  // null: rows are appended as they are
  const uint16_t *cos, *sin;
  int table_rows, hq;
  uint8_t *key_codes, *value_codes;
  float *key_scales, *value_scales;
  int units;  // blocks to look at (bound)
};

// First unit of request r: a request of n tokens touches at most
// floor(n / bs) + 2 blocks, and floor((a + n) / bs) - floor(a / bs) is at
// least floor(n / bs); single tokens touch one block each.
__device__ __forceinline__ int first_unit(const Step &s, int r) {
  return s.max_query_len <= 1 ? r : s.qsl[r] / s.bs + 2 * r;
}

__host__ __device__ __forceinline__ int64_t append_units(int64_t num_seqs, int64_t num_tokens, int64_t max_query_len,
                                                         int64_t bs) {
  return max_query_len <= 1 ? num_seqs : num_tokens / bs + 2 * num_seqs;
}

// The elements of a head that lane l holds, kPairs (D / 64) at each of l *
// kPairs and D / 2 + l * kPairs: a rotation's two halves sit in one lane.
template <bool kBf16, int D>
__device__ __forceinline__ void load_row(const uint16_t *row, int lane, float (&x)[D / 32]) {
  constexpr int kPairs = D / 64;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    x[i] = to_float<kBf16>(row[lane * kPairs + i]);
    x[kPairs + i] = to_float<kBf16>(row[D / 2 + lane * kPairs + i]);
  }
}

template <bool kBf16, int D>
__device__ __forceinline__ void rotate_row(float (&x)[D / 32], const uint16_t *cos, const uint16_t *sin, int lane) {
  constexpr int kPairs = D / 64;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int a = lane * kPairs + i, b = D / 2 + a;
    const float x1 = x[i], x2 = x[kPairs + i];
    x[i] = rope_rotate(x1, to_float<kBf16>(cos[a]), -x2, to_float<kBf16>(sin[a]));
    x[kPairs + i] = rope_rotate(x2, to_float<kBf16>(cos[b]), x1, to_float<kBf16>(sin[b]));
  }
}

constexpr int kAppendThreads = 128;

// Blocks [0, units) of the grid: one warp for each (unit, KV head, keys or
// values).  Then one warp for each query row.
template <bool kBf16, bool kFp8, int D>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  constexpr int kPairs = D / 64;
  using C = Code<kFp8>;
  const Step &s = a.step;
  const int lane = threadIdx.x & 31;
  const int warps = kAppendThreads / 32;
  const int warp = threadIdx.x >> 5;
  const int per_unit = 2 * s.hkv;
  if (static_cast<int>(blockIdx.x) >= a.units) {  // queries
    const int rows = s.num_tokens * a.hq;
    for (int i = (blockIdx.x - a.units) * warps + warp; i < rows; i += (gridDim.x - a.units) * warps) {
      const int t = i / a.hq, h = i - t * a.hq;
      const int pos = a.positions[t];
      if (pos < 0 || pos >= a.table_rows) {
        record_device_error(LVB_DEVERR_INDEX);
        continue;
      }
      float x[D / 32];
      load_row<kBf16, D>(a.query + t * a.query_stride + h * D, lane, x);
      rotate_row<kBf16, D>(x, a.cos + static_cast<int64_t>(pos) * D, a.sin + static_cast<int64_t>(pos) * D, lane);
      uint16_t *out = a.query_out + t * a.query_out_stride + h * D;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        out[lane * kPairs + k] = from_float<kBf16>(x[k]);
        out[D / 2 + lane * kPairs + k] = from_float<kBf16>(x[kPairs + k]);
      }
    }
    return;
  }
  // The unit's request: the last whose first unit is not past it.
  const int unit = blockIdx.x;
  int lo = 0, hi = s.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_unit(s, mid) <= unit) lo = mid; else hi = mid - 1;
  }
  const int r = lo;
  int q0, qlen, computed;
  if (!request_range(s, r, q0, qlen, computed) || qlen == 0) return;
  const int blk = computed / s.bs + unit - first_unit(s, r);
  const int first = max(computed, blk * s.bs), end = min(computed + qlen, (blk + 1) * s.bs);
  if (first >= end) return;
  const int phys = s.tables[r * s.table_stride + blk];
  if (phys < 0 || phys >= s.num_blocks) {
    record_device_error(LVB_DEVERR_INDEX);
    return;
  }
  const int old = first - blk * s.bs;  // earlier tokens in the block
  for (int j = warp; j < per_unit; j += warps) {
    const int h = j >> 1;
    const bool is_key = (j & 1) == 0;
    const uint16_t *src = is_key ? a.key : a.value;
    const int64_t stride = is_key ? a.key_stride : a.value_stride;
    const bool turn = is_key && a.positions != nullptr;
    auto row = [&](int p, float (&x)[D / 32]) {  // position p's row; false where its rotation is outside the tables
      const int t = q0 + p - computed;
      load_row<kBf16, D>(src + t * stride + h * D, lane, x);
      if (!turn) return true;
      const int pos = a.positions[t];
      if (pos < 0 || pos >= a.table_rows) {
        record_device_error(LVB_DEVERR_INDEX);
        return false;
      }
      rotate_row<kBf16, D>(x, a.cos + static_cast<int64_t>(pos) * D, a.sin + static_cast<int64_t>(pos) * D, lane);
      return true;
    };
    float x[D / 32];
    float top = 0.f;
    for (int p = first; p < end; ++p) {
      if (!row(p, x)) continue;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) top = fmaxf(top, fabsf(x[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int64_t at = static_cast<int64_t>(phys) * s.hkv + h;
    uint8_t *codes = (is_key ? a.key_codes : a.value_codes) + at * s.bs * D;
    float *scale_at = (is_key ? a.key_scales : a.value_scales) + at;
    const float s0 = old > 0 ? *scale_at : 0.f;
    float s1 = fmaxf(s0, __fmul_rn(fminf(top, 3.0e38f), C::kInvTop));
    if (s1 < kTinyScale) s1 = 0.f;
    const float inv = s1 > 0.f ? __frcp_rn(s1) : 0.f;
    if (s1 > s0) {
      const float ratio = __fmul_rn(s0, inv);
      for (int i = lane; i < old * D; i += 32) codes[i] = C::encode(__fmul_rn(C::decode(codes[i]), ratio));
    }
    for (int p = first; p < end; ++p) {
      if (!row(p, x)) continue;
      uint8_t *out = codes + (p - blk * s.bs) * D;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        out[lane * kPairs + k] = C::encode(__fmul_rn(x[k], inv));
        out[D / 2 + lane * kPairs + k] = C::encode(__fmul_rn(x[kPairs + k], inv));
      }
    }
    __syncwarp();  // every lane has read the scale
    if (lane == 0) *scale_at = s1;
  }
}

// Values of whole blocks in the model's type: out[i][h][slot][d] = code *
// scale of block ids[i], for the keys and the values.  One thread for each 16
// codes; bound by the bytes it moves.
struct ReadArgs {
  const uint8_t *key_codes, *value_codes;
  const float *key_scales, *value_scales;
  const int32_t *ids;
  uint16_t *key_out, *value_out;
  int64_t per_side;  // 16-code chunks of the keys (and of the values)
  int num_blocks, hkv, chunks_per_head;
};

template <bool kBf16, bool kFp8>
__global__ void __launch_bounds__(256) read_blocks_kernel(const __grid_constant__ ReadArgs a) {
  pdl_wait();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= a.per_side) return;
  const bool is_key = blockIdx.y == 0;
  const int64_t head = c / a.chunks_per_head;
  const int inside = static_cast<int>(c - head * a.chunks_per_head);
  const int64_t i = head / a.hkv;
  const int id = a.ids[i];
  uint32_t out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (id < 0 || id >= a.num_blocks) {
    record_device_error(LVB_DEVERR_INDEX);
  } else {
    const int64_t at = static_cast<int64_t>(id) * a.hkv + (head - i * a.hkv);
    const float scale = (is_key ? a.key_scales : a.value_scales)[at];
    const uint4 v = reinterpret_cast<const uint4 *>(is_key ? a.key_codes : a.value_codes)[at * a.chunks_per_head + inside];
    const uint8_t *e = reinterpret_cast<const uint8_t *>(&v);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      out[k] = pack2<kBf16>(__fmul_rn(Code<kFp8>::decode(e[2 * k]), scale), __fmul_rn(Code<kFp8>::decode(e[2 * k + 1]), scale));
  }
  uint4 *dst = reinterpret_cast<uint4 *>(is_key ? a.key_out : a.value_out) + 2 * c;
  dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
  dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

}  // namespace kv8
}  // namespace lvb
