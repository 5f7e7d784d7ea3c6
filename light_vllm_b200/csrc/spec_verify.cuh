// Verification of drafted tokens by speculative sampling.
//
// A request of n drafts x_0 .. x_{n-1} has n + 1 rows p_0 .. p_n of the
// target's probabilities and (optionally) the draft model's rows q_i, from
// which x_i was drawn; without them q_i is 1 at x_i and 0 elsewhere.  Draft i
// is accepted while u_i q_i(x_i) < p_i(x_i), u_i uniform in [0, 1).  At the
// first refusal j the next token is drawn from max(p_j - q_j, 0), and after n
// acceptances from p_n: emitted tokens then follow the target's distribution, as
// finely as the uniform numbers allow.  Those are fp32; a generator's are multiples
// of 2^-24, so acceptance and draw move in steps of 2^-24, and a token with less of
// the mass is drawn with probability 0 or 2^-24.
//
// The draw inverts the distribution function at a given uniform number in
// whole numbers: W_v = round(2^40 min(w_v, 1)) (0 for w_v <= 0 and NaN; the sum
// of 2^22 words at most fits 63 bits), bar =
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
  int num_seqs, num_rows, width, vocab, segment;
  unsigned long long *scratch;
};

// W of a weight w in [0, 1] as hi 2^20 + lo, by four additions (a conversion to 64
// bits takes some twenty instructions): w 2^40 + 1.5 2^43 is rounded to a multiple
// of 2^20, which its low bits then hold; what is left is below 2^20 and rounds to
// a whole number in the same way (ties to even: hi 2^20 is even).  Both parts are
// held with their constants' bits on top, and sums of them are taken modulo 2^32.
struct Fixed {
  static constexpr float kHi = 1.5f * 0x1p43f, kLo = 1.5f * 0x1p23f;
  static constexpr uint32_t kHiBits = 0x55400000u, kLoBits = 0x4b400000u;
  uint32_t hi = 0, lo = 0;
  __device__ __forceinline__ void add(float w) {
    const float h = __fmaf_rn(w, 0x1p40f, kHi);
    hi += __float_as_uint(h);
    lo += __float_as_uint(__fadd_rn(__fmaf_rn(w, 0x1p40f, -__fadd_rn(h, -kHi)), kLo));
  }
  // The sum of `count` weights, up to 2^10 of them.
  __device__ __forceinline__ long long value(uint32_t count) const {
    return (static_cast<long long>(static_cast<int32_t>(hi - count * kHiBits)) << 20) +
           static_cast<int32_t>(lo - count * kLoBits);
  }
};

__device__ __forceinline__ long long fixed_weight(float w) {
  Fixed f;
  f.add(w);
  return f.value(1);
}

// The vocabulary is cut into segments, one for each warp; a CTA of kWarps warps
// takes as many neighbouring ones.  Scratch of a request: a counter of its
// finished CTAs (zero between calls), then the segments' sums.  The stride is
// fixed, so that one request's counter never lies where another call's sums do.
constexpr int kWarps = 8;
constexpr int kVerifyThreads = kWarps * 32;
constexpr int kCtasPerSm = 5;
constexpr int kMaxChunks = 126;
constexpr int kScratchWords = kMaxChunks * kWarps + 2;  // of 8 bytes

// One CTA for each (chunk of the vocabulary, request).  Every CTA of a request
// finds the refused draft for itself (a few loads, in L2 after the first), sums
// its segments' weights, and the last one to finish finds the segment and then
// the token at which the prefix sum passes the bar.  Bound by reading one row (two
// after a refusal) of the vocabulary once; a call of one request by the latency
// of its dependent loads.  64 requests of 4 drafts over 152064 words: 19.5 us, 49 %
// of the measured copy rate's (21.0 us with conversions to 64 bits, 27 us with a
// block scan for every chunk as well, 110 us with one CTA a request); one request:
// 6 us.
__global__ void __launch_bounds__(kVerifyThreads, kCtasPerSm) verify_kernel(const __grid_constant__ VerifyArgs a) {
  pdl_wait();
  __shared__ int stop_sm, last_sm, found_sm, segment_sm;
  __shared__ long long sums[kWarps], before_sm;
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

  // Groups of four elements that lie on 16 bytes in p: group k is elements 4 k -
  // shift .. + 3, and those outside [lo, hi) count for nothing.  q is read alike
  // where it lies the same way.
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 2 & 3);
  const bool alike = q == nullptr || static_cast<int>(reinterpret_cast<uintptr_t>(q) >> 2 & 3) == shift;
  auto weights = [&](int v, int lo, int hi, bool residual, float (&x)[4]) {
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    x[0] = x[1] = x[2] = x[3] = 0.f;
    const bool less = residual && q != nullptr;
    if (v >= lo && v + 4 <= hi) {
      const float4 t = __ldg(reinterpret_cast<const float4 *>(p + v));
      x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
      if (less && alike) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(q + v));
        y[0] = u.x, y[1] = u.y, y[2] = u.z, y[3] = u.w;
      } else if (less) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __ldg(q + v + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i >= lo && v + i < hi) {
          x[i] = __ldg(p + v + i);
          if (less) y[i] = __ldg(q + v + i);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __saturatef(__fsub_rn(x[i], y[i]));  // (NaN: 0)
  };
  auto group_start = [&](int v) { return (v + shift) / 4 * 4 - shift; };
  // Sum over [v0, v1) by one warp (every lane's result).
  auto warp_sum_of = [&](int v0, int v1, bool residual) {
    long long own = 0;
    constexpr int kTogether = 4;
    int v = group_start(v0) + lane * 4;
#pragma unroll 1
    for (; v < v1; v += kTogether * 128) {
      float x[kTogether][4];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
        if (v + i * 128 < v1) weights(v + i * 128, v0, v1, residual, x[i]);
      }
      Fixed f;
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) f.add(x[i][k]);
      own += f.value(4 * kTogether);
    }
    if (residual && lane == 0 && gone >= v0 && gone < v1) own -= fixed_weight(__saturatef(__ldg(p + gone)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    return own;
  };
  // Inclusive prefix of `own` over the CTA; `all` is the total.
  auto block_prefix = [&](long long own, long long &all) {
    long long upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += sums[w];
      all += sums[w];
    }
    return upto;
  };

  const int segments = gridDim.x * kWarps;
  unsigned long long *scratch = a.scratch + static_cast<int64_t>(b) * kScratchWords;
  const int v0 = min(a.vocab, (chunk * kWarps + warp) * a.segment), v1 = min(a.vocab, v0 + a.segment);
  const long long mine = warp_sum_of(v0, v1, true);
  if (lane == 0) __stcg(scratch + 1 + chunk * kWarps + warp, static_cast<unsigned long long>(mine));
  __threadfence();
  __syncthreads();
  if (tid == 0) last_sm = gridDim.x == 1 || atomicAdd(scratch, 1ull) == gridDim.x - 1;
  __syncthreads();
  if (!last_sm) return;
  __threadfence();
  // The segment that the bar falls into, and the prefix sum before it.
  constexpr int kPer = (kMaxChunks * kWarps + kVerifyThreads - 1) / kVerifyThreads;
  long long part[kPer], own = 0, total, bar = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = tid * kPer + i;
    part[i] = at < segments ? static_cast<long long>(__ldcg(scratch + 1 + at)) : 0;
    own += part[i];
  }
  if (tid == 0) found_sm = a.vocab - 1;
  bool residual = true;
  long long upto = block_prefix(own, total) - own;
  if (tid == 0 && gridDim.x > 1) scratch[0] = 0;
  if (total == 0) {  // nothing is left of p: its own weights
    residual = false;
    own = 0;
    for (int i = warp; i < segments; i += kWarps) {
      const long long w = warp_sum_of(min(a.vocab, i * a.segment), min(a.vocab, (i + 1) * a.segment), false);
      if (lane == 0) __stcg(scratch + 1 + i, static_cast<unsigned long long>(w));
    }
    __threadfence();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = tid * kPer + i;
      part[i] = at < segments ? static_cast<long long>(__ldcg(scratch + 1 + at)) : 0;
      own += part[i];
    }
    upto = block_prefix(own, total) - own;
  }
  if (total > 0) {
    bar = static_cast<long long>(floor(static_cast<double>(a.sample[b]) * static_cast<double>(total)));
    bar = max(0ll, min(bar, total - 1));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (upto <= bar && bar < upto + part[i]) {
        segment_sm = tid * kPer + i;
        before_sm = upto;
      }
      upto += part[i];
    }
    __syncthreads();
    long long before = before_sm;
    const int lo = segment_sm * a.segment, hi = min(a.vocab, lo + a.segment);
    for (int v = group_start(lo); v < hi; v += kVerifyThreads * 4) {
      const int own_v = v + tid * 4;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      long long w[4], all;
      if (own_v < hi) weights(own_v, lo, hi, residual, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = residual && own_v + i == gone ? 0ll : fixed_weight(x[i]);
      own = (w[0] + w[1]) + (w[2] + w[3]);
      const long long mine_upto = block_prefix(own, all);
      if (before + all > bar) {  // the token is here
        long long sum = before + mine_upto - own;
        if (sum <= bar && bar < before + mine_upto) {
          int i = 0;
          for (; i < 3; ++i) {
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
