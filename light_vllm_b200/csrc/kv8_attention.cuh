// Attention of packed queries over the 8-bit paged cache (kv8_cache.cuh):
//   out[t][h] = sum_j exp(scale q.k_j - max) v_j / sum_j exp(scale q.k_j - max)
// over the positions j <= computed + offset of token t's request, with k_j =
// code * key scale and v_j = code * value scale of j's block.
#pragma once

#include "kv8_decode.cuh"

namespace lvb {
namespace kv8 {

// One warp for each (token, query head): lanes score 32 positions at a time,
// an fp32 online softmax runs over them, and each lane owns D / 32 elements.
template <bool kBf16, bool kFp8, int D>
__global__ void __launch_bounds__(32) attention_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  using C = Code<kFp8>;
  constexpr int kOwn = D / 32;
  __shared__ float q[D];
  const Step &s = a.step;
  const int lane = threadIdx.x, h = blockIdx.y, r = blockIdx.z;
  int q0, qlen, computed;
  if (!request_range(s, r, q0, qlen, computed) || static_cast<int>(blockIdx.x) >= qlen ||
      qlen <= kMaxRows / a.group)
    return;
  const int t = q0 + blockIdx.x;
  const int kvh = h / (a.hq / s.hkv);
  const int end = computed + blockIdx.x + 1;
  for (int d = lane; d < D; d += 32) q[d] = to_float<kBf16>(a.query[t * a.query_stride + h * D + d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) acc[i] = 0.f;
  for (int base = 0; base < end; base += 32) {
    const int p = base + lane;
    float x = -INFINITY, vs = 0.f;
    int64_t row = 0;
    if (p < end) {
      const int phys = s.tables[r * s.table_stride + p / s.bs];
      if (phys < 0 || phys >= s.num_blocks) {
        record_device_error(LVB_DEVERR_INDEX);
      } else {
        const int64_t at = static_cast<int64_t>(phys) * s.hkv + kvh;
        row = (at * s.bs + p % s.bs) * D;
        float dot = 0.f;
        for (int d = 0; d < D; ++d) dot = fmaf(C::decode(a.key_codes[row + d]), q[d], dot);
        x = dot * a.key_scales[at] * a.scale_log2;
        vs = a.value_scales[at];
      }
    }
    float mx = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m_new = fmaxf(m, mx);
    if (m_new == -INFINITY) continue;
    const float e = exp2f(x - m_new);
    float sum = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float alpha = exp2f(m - m_new);
    l = l * alpha + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) acc[i] *= alpha;
    for (int j = 0; j < 32 && base + j < end; ++j) {
      const float w = __shfl_sync(0xffffffffu, e * vs, j);
      const int64_t rj = __shfl_sync(0xffffffffu, row, j);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) acc[i] = fmaf(w, C::decode(a.value_codes[rj + lane * kOwn + i]), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i)
    a.out[t * a.out_stride + h * D + lane * kOwn + i] = from_float<kBf16>(l > 0.f ? acc[i] / l : 0.f);
}

}  // namespace kv8
}  // namespace lvb
