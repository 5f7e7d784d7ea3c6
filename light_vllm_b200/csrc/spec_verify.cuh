// Verification of drafted tokens by speculative sampling.
//
// A request of n drafts x_0 .. x_{n-1} has n + 1 rows p_0 .. p_n of the
// target's probabilities and (optionally) the draft model's rows q_i, from
// which x_i was drawn; without them q_i is 1 at x_i and 0 elsewhere.  Draft i
// is accepted while u_i q_i(x_i) < p_i(x_i), u_i uniform in [0, 1).  At the
// first refusal j the next token is drawn from max(p_j - q_j, 0), and after n
// acceptances from p_n: emitted tokens then follow the target's distribution
// exactly.
//
// The draw inverts the distribution function at a given uniform number in
// whole numbers: W_v = round(2^40 min(w_v, 1)) (0 for w_v <= 0 and NaN), bar =
// floor(u sum W), token = the lowest v whose prefix sum exceeds bar.  Sums of
// whole numbers are the same in every order, so the token does not depend on
// how the vocabulary is split.  A weight below 2^-41 is never drawn.  If every
// W is 0 (p = q up to rounding, or a draft that q gives no mass), the weights
// are p_j's own; if those are 0 too, the token is the last of the vocabulary.
#pragma once

#include "lvb_common.cuh"

namespace lvb {
namespace spec {

struct VerifyArgs {
  const float *target;
  int64_t target_stride;
  const float *draft;  // null: q = 1 at the drafted token
  int64_t draft_stride;
  const int64_t *tokens;  // the drafts, packed
  const float *accept, *sample;
  const int32_t *qsl;
  int64_t *out;  // [num_seqs][width]
  int32_t *accepted;
  int num_seqs, num_rows, width, vocab;
};

__device__ __forceinline__ long long fixed_weight(float w) {
  w = w > 0.f ? fminf(w, 1.f) : 0.f;
  return __float2ll_rn(w * 0x1p40f);
}

constexpr int kVerifyThreads = 1024;

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  pdl_wait();
  __shared__ int stop;  // first refused draft, or their number
  __shared__ long long sums[33];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = a.qsl[b], rows = a.qsl[b + 1] - row0;
  const int n = rows - 1, first = row0 - b;
  if (first < 0 || n < 0 || rows > a.width || row0 + rows > a.num_rows || first + n > a.num_rows - a.num_seqs) {
    if (tid == 0) {
      record_device_error(LVB_DEVERR_INDEX);
      a.accepted[b] = 0;
    }
    for (int i = tid; i < a.width; i += kVerifyThreads) a.out[static_cast<int64_t>(b) * a.width + i] = -1;
    return;
  }
  if (tid == 0) {
    int i = 0;
    for (; i < n; ++i) {
      const int64_t x = a.tokens[first + i];
      if (x < 0 || x >= a.vocab) {
        record_device_error(LVB_DEVERR_INDEX);
        break;
      }
      const float p = a.target[(row0 + i) * a.target_stride + x];
      const float q = a.draft != nullptr ? a.draft[(first + i) * a.draft_stride + x] : 1.f;
      if (!(__fmul_rn(a.accept[first + i], q) < p)) break;
    }
    stop = i;
    found = a.vocab - 1;
  }
  __syncthreads();
  const int j = stop;
  const float *p = a.target + (row0 + j) * a.target_stride;
  const float *q = j < n && a.draft != nullptr ? a.draft + (first + j) * a.draft_stride : nullptr;
  const int64_t gone = j < n && a.draft == nullptr ? a.tokens[first + j] : -1;
  bool residual = true;
  auto weight = [&](int v) {
    if (!residual) return fixed_weight(p[v]);
    if (v == gone) return 0ll;
    return fixed_weight(q != nullptr ? __fsub_rn(p[v], q[v]) : p[v]);
  };
  auto block_sum = [&](long long x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if (lane == 0) sums[warp] = x;
    __syncthreads();
    long long t = 0;
    for (int w = 0; w < kVerifyThreads / 32; ++w) t += sums[w];
    return t;
  };
  // Each thread owns a run of the vocabulary.
  const int run = (a.vocab + kVerifyThreads - 1) / kVerifyThreads;
  const int v0 = min(a.vocab, tid * run), v1 = min(a.vocab, v0 + run);
  long long own = 0;
  for (int v = v0; v < v1; ++v) own += weight(v);
  long long total = block_sum(own);
  if (total == 0) {
    residual = false;
    own = 0;
    for (int v = v0; v < v1; ++v) own += weight(v);
    total = block_sum(own);
  }
  if (total > 0) {
    long long before = own;  // inclusive scan over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += sums[w];
    long long bar = static_cast<long long>(floor(static_cast<double>(a.sample[b]) * static_cast<double>(total)));
    bar = max(0ll, min(bar, total - 1));
    if (before - own <= bar && bar < before) {
      long long upto = before - own;
      for (int v = v0; v < v1; ++v) {
        upto += weight(v);
        if (upto > bar) {
          found = v;
          break;
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) a.accepted[b] = j;
  for (int i = tid; i < a.width; i += kVerifyThreads)
    a.out[static_cast<int64_t>(b) * a.width + i] = i < j ? a.tokens[first + i] : i == j ? found : -1;
}

}  // namespace spec
}  // namespace lvb
