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
  int num_seqs, num_rows, width, vocab, chunk;
  unsigned long long *scratch;
};

__device__ __forceinline__ long long fixed_weight(float w) {
  w = w > 0.f ? fminf(w, 1.f) : 0.f;
  return __float2ll_rn(w * 0x1p40f);
}

// Scratch of a request: a counter of its finished CTAs (zero between calls),
// then the sums of its chunks.  The stride is fixed, so that one request's
// counter never lies where another call's sums do.
constexpr int kMaxChunks = 126;
constexpr int kScratchWords = kMaxChunks + 2;  // of 8 bytes
constexpr int kVerifyThreads = 256;

// One CTA for each (chunk of the vocabulary, request).  Every CTA of a request
// finds the refused draft for itself (a few loads, in L2 after the first), sums
// its chunk's weights, and the last one to finish finds the chunk and then the
// token at which the prefix sum passes the bar.  Bound by reading one row (two
// after a refusal) of the vocabulary once; a call of one request by the latency
// of its dependent loads.  kVec: rows allow 16-byte loads.
template <bool kVec>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  pdl_wait();
  __shared__ int stop_sm, last_sm, found_sm;
  __shared__ long long sums[kVerifyThreads / 32];
  constexpr int kWarps = kVerifyThreads / 32;
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = a.qsl[b], rows = a.qsl[b + 1] - row0;
  const int n = rows - 1, first = row0 - b;
  int64_t *out = a.out + static_cast<int64_t>(b) * a.width;
  if (first < 0 || n < 0 || rows > a.width || row0 + rows > a.num_rows || first + n > a.num_rows - a.num_seqs) {
    if (chunk != 0) return;
    if (tid == 0) {
      record_device_error(LVB_DEVERR_INDEX);
      a.accepted[b] = 0;
    }
    for (int i = tid; i < a.width; i += kVerifyThreads) out[i] = -1;
    return;
  }
  // The first refused draft (n: none).
  if (warp == 0) {
    int stop = n;
    for (int base = 0; base < n; base += 32) {
      const int i = base + lane;
      bool good = true, known = true;
      if (i < n) {
        const int64_t x = a.tokens[first + i];
        known = x >= 0 && x < a.vocab;
        good = known;
        if (known) {
          const float u = a.accept[first + i], p = a.target[(row0 + i) * a.target_stride + x];
          const float q = a.draft != nullptr ? a.draft[(first + i) * a.draft_stride + x] : 1.f;
          good = __fmul_rn(u, q) < p;
        }
      }
      const uint32_t bad = __ballot_sync(0xffffffffu, !good);
      if (bad != 0) {
        const int at = __ffs(bad) - 1;
        stop = base + at;
        if (lane == at && !known && chunk == 0) record_device_error(LVB_DEVERR_INDEX);
        break;
      }
    }
    if (lane == 0) stop_sm = stop;
  }
  __syncthreads();
  const int j = stop_sm;
  const float *p = a.target + (row0 + j) * a.target_stride;
  const float *q = j < n && a.draft != nullptr ? a.draft + (first + j) * a.draft_stride : nullptr;
  const int64_t gone = j < n && a.draft == nullptr ? a.tokens[first + j] : -1;

  // Weights of the elements v .. v + 3 (kVec) or v.
  constexpr int kStep = kVec ? 4 : 1;
  auto weights = [&](int v, bool residual, long long (&w)[kStep]) {
    float x[kStep], y[kStep];
    if constexpr (kVec) {
      const float4 t = __ldg(reinterpret_cast<const float4 *>(p + v));
      x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
      if (residual && q != nullptr) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(q + v));
        y[0] = u.x, y[1] = u.y, y[2] = u.z, y[3] = u.w;
      }
    } else {
      x[0] = __ldg(p + v);
      if (residual && q != nullptr) y[0] = __ldg(q + v);
    }
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      if (residual && q != nullptr) x[i] = __fsub_rn(x[i], y[i]);
      w[i] = residual && v + i == gone ? 0ll : fixed_weight(x[i]);
    }
  };
  auto range_sum = [&](int v0, int v1, bool residual) {
    long long own = 0;
#pragma unroll 4
    for (int v = v0 + tid * kStep; v < v1; v += kVerifyThreads * kStep) {
      long long w[kStep];
      weights(v, residual, w);
#pragma unroll
      for (int i = 0; i < kStep; ++i) own += w[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    __syncthreads();
    if (lane == 0) sums[warp] = own;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += sums[w];
    return total;
  };
  auto bar_of = [&](long long total) {
    const long long bar = static_cast<long long>(floor(static_cast<double>(a.sample[b]) * static_cast<double>(total)));
    return max(0ll, min(bar, total - 1));
  };

  const int v0 = min(a.vocab, chunk * a.chunk), v1 = min(a.vocab, v0 + a.chunk);
  const long long mine = range_sum(v0, v1, true);
  unsigned long long *scratch = a.scratch + static_cast<int64_t>(b) * kScratchWords;
  if (gridDim.x > 1) {
    if (tid == 0) {
      scratch[1 + chunk] = static_cast<unsigned long long>(mine);
      __threadfence();
      last_sm = atomicAdd(scratch, 1ull) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last_sm) return;
    __threadfence();
  }
  // The chunk that the bar falls into, and the prefix sum before it.
  long long total = 0, before = 0, bar = 0;
  int at = 0;
  bool residual = true;
  if (tid == 0) found_sm = a.vocab - 1;
  if (gridDim.x == 1) {
    total = mine;
    bar = bar_of(total);
  } else {
    for (int c = 0; c < static_cast<int>(gridDim.x); ++c) total += static_cast<long long>(__ldcg(scratch + 1 + c));
    bar = bar_of(total);
    while (at + 1 < static_cast<int>(gridDim.x)) {
      const long long w = static_cast<long long>(__ldcg(scratch + 1 + at));
      if (before + w > bar) break;
      before += w;
      ++at;
    }
    __syncthreads();
    if (tid == 0) scratch[0] = 0;
  }
  int lo = at * a.chunk, hi = min(a.vocab, lo + a.chunk);
  if (total == 0) {  // nothing is left of p: its own weights, over the whole row
    residual = false;
    total = range_sum(0, a.vocab, false);
    bar = bar_of(total);
    before = 0;
    lo = 0;
    hi = a.vocab;
  }
  if (total > 0) {
    for (int v = lo; v < hi; v += kVerifyThreads * kStep) {
      const int own_v = v + tid * kStep;
      long long w[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) w[i] = 0;
      if (own_v < hi) weights(own_v, residual, w);
      long long own = 0;
#pragma unroll
      for (int i = 0; i < kStep; ++i) own += w[i];
      long long upto = own;  // inclusive prefix over the CTA
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      __syncthreads();
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      long long all = 0;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        if (k < warp) upto += sums[k];
        all += sums[k];
      }
      if (before + all > bar) {  // the token is here
        long long sum = before + upto - own;
        if (sum <= bar && bar < before + upto) {
          int i = 0;
          for (; i < kStep - 1; ++i) {
            sum += w[i];
            if (sum > bar) break;
          }
          found_sm = own_v + i;
        }
        break;
      }
      before += all;
    }
  }
  __syncthreads();
  if (tid == 0) a.accepted[b] = j;
  for (int i = tid; i < a.width; i += kVerifyThreads) out[i] = i < j ? a.tokens[first + i] : i == j ? found_sm : -1;
}

}  // namespace spec
}  // namespace lvb
