// Attention of few query rows over the 8-bit paged cache: requests whose query
// tokens times the query heads of one KV head are at most 16 (decode steps, and
// the verification of a draft or two), so that K and V are read once for all of
// them.  Bound by those bytes.
//
// Mathematics.  With f_b = scale log2(e) key_scale_b and w_b = value_scale_b of
// a position's block b, x_j = (q . key code_j) f_b + log2 w_b and a running
// maximum m of x, the sums
//     O = sum_j 2^(x_j - m) value code_j        L = sum_j 2^(x_j - m) / w_b
// give out = O / L: the value scale rides in the exponent, so the weights that
// enter the second product lie in (0, 1] whatever the scales are, and no code is
// ever multiplied by a scale.  They enter it as fp16, times 2^8 (kHead) and up to
// 2^4 (kLazy) more, so that a weight 2^-22 of the largest still has 11 bits; O, L,
// m and the scores are fp32.  m moves only when it would grow by more than kLazy:
// a rescaling of O is rare.
//
// Tensor cores.  Both products are m16n8k16 warp MMAs with the query rows as M
// (the tensor pipe is not what bounds this).  Codes are exact in fp16: int8 by
// setting the byte under the exponent of 1024 and subtracting 1152, e4m3 by the
// hardware's conversion.  Operands go from global memory straight to the
// fragments' registers: the order of the head's elements in q k^T, and of a
// page's 16 positions, is free as long as both operands agree, so lane (g, t) of
// the fragment takes 16 consecutive bytes of key row g (its q fragments are laid
// out alike) and 16 consecutive bytes of value rows 2t, 2t + 1, 2t + 8, 2t + 9.
//
// Split.  The pages of all (request, KV head) items are laid end to end and cut
// into one equal run for each resident CTA, whatever the contexts' lengths; the
// warps of a CTA take its pages in turn.  An item that ends in another CTA leaves
// partial (O, m, L) in the workspace, and the last of its CTAs to finish (a
// counter for each item) sums them in order, so results do not depend on timing.
#pragma once

#include "kv8_cache.cuh"

namespace lvb {
namespace kv8 {

constexpr float kHead = 8.f;
constexpr float kLazy = 4.f;
constexpr int kPage = 16;     // positions a warp takes at a time
constexpr int kMaxRows = 16;  // query rows of a decode item
constexpr int kMinRun = 16;   // pages of a CTA, at least: more CTAs only merge more

struct AttnArgs {
  Step step;
  const uint16_t *query;
  int64_t query_stride;
  uint16_t *out;
  int64_t out_stride;
  const uint8_t *key_codes, *value_codes;
  const float *key_scales, *value_scales;
  int hq, group;
  float scale_log2;  // softmax scale * log2(e)
  // decode kernel
  float *part_o;      // [2 * CTAs][kMaxRows][D]
  float2 *part_ml;    // [2 * CTAs][kMaxRows]: m, L
  uint32_t *counts;   // [num_seqs][hkv], zero between calls
};

// Two fp16 values of bytes 0, 1 (kHi: 2, 3) of four codes.
template <bool kFp8>
struct Pair;

template <>
struct Pair<false> {
  static __device__ __forceinline__ uint32_t bias(uint32_t four) { return four ^ 0x80808080u; }
  template <bool kHi>
  static __device__ __forceinline__ uint32_t get(uint32_t biased) {
    const uint32_t v = __byte_perm(biased, 0x64646464u, kHi ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};

template <>
struct Pair<true> {
  static __device__ __forceinline__ uint32_t bias(uint32_t four) { return four; }
  template <bool kHi>
  static __device__ __forceinline__ uint32_t get(uint32_t four) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(kHi ? four >> 16 : four & 0xffffu),
                                                     __NV_E4M3);
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
  }
};

// D += A B with rows 8..15 of A zero: half the accumulator registers.
__device__ __forceinline__ void mma_rows8(float &d0, float &d1, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  float x, y;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%6,%5,%6}, {%7,%8}, {%0,%1,%9,%9};"
      : "+f"(d0), "+f"(d1), "=f"(x), "=f"(y)
      : "r"(a0), "r"(a2), "r"(0u), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) { return pack2<false>(lo, hi); }

// A row of queries as fp16 times 2^shift (returned as 2^-shift): fp16 rows as
// they are; bf16 rows with their largest element brought to [2^7, 2^8), which
// keeps every element down to 2^-22 of it exact, and smaller ones to 2^-32 of it.
template <bool kBf16, int N>
__device__ __forceinline__ float query_shift(const float (&x)[N]) {
  if constexpr (!kBf16) {
    return 1.f;
  } else {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // exponent field of 2^(7 - e): 127 + 7 - (field - 127), kept in the normal range
    const int field = static_cast<int>(__float_as_uint(top) >> 23);
    return __uint_as_float(static_cast<uint32_t>(min(max(261 - field, 1), 254)) << 23);
  }
}

// One run of pages of one item.
struct Segment {
  int r, kvh, first, last;  // pages [first, last)
  int pages;                // of the whole item
  int q0, rows, computed;
};

template <bool kBf16, bool kFp8, int D, bool kRows8>
struct DecodeCfg {
  static constexpr int kWarps = kRows8 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtasPerSm = kRows8 ? 2 : 3;
  static constexpr int kRowSlots = kRows8 ? 8 : 16;
  static constexpr int kPad = D + 4;  // a row of O in shared memory
};

template <bool kBf16, bool kFp8, int D, bool kRows8>
__global__ void __launch_bounds__(DecodeCfg<kBf16, kFp8, D, kRows8>::kThreads, DecodeCfg<kBf16, kFp8, D, kRows8>::kCtasPerSm)
    decode_kernel(const __grid_constant__ AttnArgs a) {
  using Cfg = DecodeCfg<kBf16, kFp8, D, kRows8>;
  using P = Pair<kFp8>;
  constexpr int kWarps = Cfg::kWarps, kThreads = Cfg::kThreads, kSlots = Cfg::kRowSlots;
  constexpr int kKSteps = D / 16;   // MMAs of a score
  constexpr int kNTiles = D / 8;    // MMAs of O
  constexpr int kKChunks = D / 64;  // 16-byte pieces of a key row that a lane takes
  constexpr int kVWords = D / 32;   // words of a value row that a lane takes
  constexpr int kHalves = kRows8 ? 1 : 2;
  __shared__ float o_sm[kWarps][kSlots][Cfg::kPad];
  __shared__ float m_sm[kWarps][kSlots], l_sm[kWarps][kSlots];
  __shared__ int scan[kWarps];
  __shared__ long long scan_total;
  __shared__ int start_sm[2];  // first request of the run, its pages before the run
  __shared__ int last_sm;
  pdl_wait();
  const Step &s = a.step;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // Pages of request r's items (0: not this kernel's, or refused).
  auto request_pages = [&](int r) {
    int q0, n, c;
    if (!request_range(s, r, q0, n, c) || n == 0 || n > kSlots / a.group) return 0;
    return (c + n + kPage - 1) / kPage;
  };
  // Exclusive prefix of a value over the CTA; `sum` is the total.
  auto block_scan = [&](int v, int &sum) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int before = 0;
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      sum += scan[w];
    }
    return before + x - v;
  };

  // The whole batch's pages, the run of each CTA, and where this one's begins.
  long long total = 0;
  for (int base = 0; base < s.num_seqs; base += kThreads) {
    int sum;
    block_scan(base + tid < s.num_seqs ? request_pages(base + tid) : 0, sum);
    total += static_cast<long long>(sum) * s.hkv;
  }
  long long run = (total + gridDim.x - 1) / gridDim.x;
  if (run < kMinRun) run = kMinRun;
  const long long begin = run * blockIdx.x;
  if (begin >= total) return;
  const long long end = begin + run < total ? begin + run : total;
  {
    long long before = 0;
    for (int base = 0; base < s.num_seqs; base += kThreads) {
      const int mine = base + tid < s.num_seqs ? request_pages(base + tid) : 0;
      int sum;
      const int ex = block_scan(mine, sum);
      const long long lo = before + static_cast<long long>(ex) * s.hkv, hi = lo + static_cast<long long>(mine) * s.hkv;
      if (lo <= begin && begin < hi) {
        start_sm[0] = base + tid;
        scan_total = lo;
      }
      before += static_cast<long long>(sum) * s.hkv;
    }
    __syncthreads();
  }

  // Walk of the run: `at` is the flat index of segment `seg`'s first page.
  auto describe = [&](int r, int kvh, int first, long long left, Segment &seg) {
    seg.r = r;
    seg.kvh = kvh;
    seg.q0 = s.qsl[r];
    seg.computed = s.computed[r];
    const int n = s.qsl[r + 1] - seg.q0;
    seg.rows = n * a.group;
    seg.pages = (seg.computed + n + kPage - 1) / kPage;
    seg.first = first;
    seg.last = static_cast<int>(left < seg.pages - first ? first + left : seg.pages);
  };
  long long at = begin;
  Segment seg;
  {
    const int r = start_sm[0];
    const int pages = request_pages(r);
    const int inside = static_cast<int>(begin - scan_total);
    describe(r, inside / pages, inside % pages, end - begin, seg);
  }

  const int ppb = s.bs / kPage;
  uint32_t kreg[2][kKChunks][4], vreg[4][kVWords];
  float ks = 0.f, vs = 1.f;   // scales of the page in kreg / vreg
  int bad = 0;                // its block id is out of range
  int64_t head_at = 0;        // first byte of the next page's head
  float ks_next, vs_next;
  int bad_next;

  // Start of page p of item (r, kvh): its place and scales.
  auto locate = [&](int r, int kvh, int p) {
    const int blk = ppb == 1 ? p : p / ppb;
    int phys = s.tables[r * s.table_stride + blk];
    bad_next = phys < 0 || phys >= s.num_blocks;
    if (bad_next) {
      record_device_error(LVB_DEVERR_INDEX);
      phys = 0;
    }
    const int64_t h = static_cast<int64_t>(phys) * s.hkv + kvh;
    ks_next = a.key_scales[h];
    vs_next = a.value_scales[h];
    head_at = (h * s.bs + (p - blk * ppb) * kPage) * D;
  };
  auto load_keys = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kKChunks; ++c) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(a.key_codes + head_at + (g + 8 * i) * D + c * 64 + t * 16));
        kreg[i][c][0] = v.x, kreg[i][c][1] = v.y, kreg[i][c][2] = v.z, kreg[i][c][3] = v.w;
      }
  };
  auto load_values = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *src = a.value_codes + head_at + (2 * t + (i & 1) + (i >> 1) * 8) * D + g * (D / 8);
      if constexpr (D == 128) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src));
        vreg[i][0] = v.x, vreg[i][1] = v.y, vreg[i][2] = v.z, vreg[i][3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src));
        vreg[i][0] = v.x, vreg[i][1] = v.y;
      }
    }
  };
  // Item after (r, kvh); false at the end of the run.
  auto next_segment = [&](const Segment &from, Segment &to) {
    const long long left = end - at - (from.last - from.first);
    if (left <= 0) return false;
    int r = from.r, kvh = from.kvh + 1;
    if (kvh == s.hkv) {
      kvh = 0;
      do {
        ++r;
      } while (request_pages(r) == 0);  // pages are left, so a request is
    }
    describe(r, kvh, 0, left, to);
    return true;
  };

  bool more = true;
  if (seg.first + warp < seg.last) {
    locate(seg.r, seg.kvh, seg.first + warp);
    load_keys();
    load_values();
  }
  while (more) {
    Segment nseg;
    more = next_segment(seg, nseg);
    // Query rows g and g + 8: row i is token i / group, head i % group.
    uint32_t qa[kKSteps][kRows8 ? 2 : 4];
    float f[kHalves];
    int limit[kHalves];  // last position that the row sees
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const bool ok = row < seg.rows;
      const int tok = ok ? row / a.group : 0, head = ok ? row - tok * a.group : 0;
      const uint16_t *src = a.query + (seg.q0 + tok) * a.query_stride + (seg.kvh * a.group + head) * D + t * 16;
      float x[kKChunks * 16];
#pragma unroll
      for (int c = 0; c < kKChunks; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[c * 16 + i] = ok ? to_float<kBf16>(src[c * 64 + i]) : 0.f;
      const float up = query_shift<kBf16>(x);
      f[h] = a.scale_log2 / up;
#pragma unroll
      for (int k = 0; k < kKSteps; ++k) {
        const int i = k * 4;
        qa[k][h] = pack_half(x[i] * up, x[i + 1] * up);
        qa[k][kHalves + h] = pack_half(x[i + 2] * up, x[i + 3] * up);
      }
      limit[h] = ok ? seg.computed + tok : -1;
    }
    float o[kNTiles][2 * kHalves], m[kHalves], l[kHalves];
#pragma unroll
    for (int j = 0; j < kNTiles; ++j)
#pragma unroll
      for (int i = 0; i < 2 * kHalves; ++i) o[j][i] = 0.f;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) m[h] = -INFINITY, l[h] = 0.f;

    const bool has_next_seg = more && nseg.first + warp < nseg.last;
    for (int p = seg.first + warp; p < seg.last; p += kWarps) {
      ks = ks_next, vs = vs_next, bad = bad_next;
      bool next = p + kWarps < seg.last;
      if (next) {
        locate(seg.r, seg.kvh, p + kWarps);
      } else if (has_next_seg) {
        locate(nseg.r, nseg.kvh, nseg.first + warp);
        next = true;
      }
      // Scores of 16 positions: columns of two MMA tiles.
      float sc[2][2 * kHalves];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 2 * kHalves; ++e) sc[i][e] = 0.f;
#pragma unroll
        for (int k = 0; k < kKSteps; ++k) {
          const uint32_t w = P::bias(kreg[i][k >> 2][k & 3]);
          const uint32_t b0 = P::template get<false>(w), b1 = P::template get<true>(w);
          if constexpr (kRows8)
            mma_rows8(sc[i][0], sc[i][1], qa[k][0], qa[k][1], b0, b1);
          else
            mma_16816_nv<false>(sc[i], qa[k], b0, b1);
        }
      }
      if (next) load_keys();
      const float vw = vs > 0.f ? vs : 1.f;
      const float lw = log2_fast(vw), iw = 1.f / vw;
      const int pos = p * kPage + 2 * t;  // of column 0 of this lane
      const bool masked = bad || p * kPage + kPage - 1 > seg.computed;
      float top[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float fk = f[h] * ks;
        top[h] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaf(sc[i][2 * h + e], fk, lw);
            if (masked && (bad || pos + 8 * i + e > limit[h])) x = -INFINITY;
            sc[i][2 * h + e] = x;
            top[h] = fmaxf(top[h], x);
          }
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      }
      bool grow = false;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) grow |= top[h] > m[h] + kLazy;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const float now = fmaxf(m[h], top[h]);
          const float alpha = now == -INFINITY ? 1.f : exp2_fast(m[h] - now);
          m[h] = now;
          l[h] *= alpha;
#pragma unroll
          for (int j = 0; j < kNTiles; ++j) o[j][2 * h] *= alpha, o[j][2 * h + 1] *= alpha;
        }
      }
      uint32_t pa[2 * kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float base = m[h] == -INFINITY ? 0.f : m[h] - kHead;
        float e[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          e[i][0] = exp2_fast(sc[i][2 * h] - base);
          e[i][1] = exp2_fast(sc[i][2 * h + 1] - base);
          pa[i * kHalves + h] = pack_half(e[i][0], e[i][1]);
        }
        l[h] = fmaf((e[0][0] + e[0][1]) + (e[1][0] + e[1][1]), iw, l[h]);
      }
      if (kFp8 && masked) {
        // Slots past the end may hold NaN patterns: 0 * NaN is not 0.
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (bad || p * kPage + 2 * t + (i & 1) + (i >> 1) * 8 >= seg.computed + seg.rows / a.group)
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vreg[i][w] = 0;
      }
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // bytes (2 half, 2 half + 1) of rows (0, 1) and (2, 3), interleaved
          const uint32_t lo = P::bias(__byte_perm(vreg[0][w], vreg[1][w], half ? 0x7362 : 0x5140));
          const uint32_t hi = P::bias(__byte_perm(vreg[2][w], vreg[3][w], half ? 0x7362 : 0x5140));
          const int j = w * 4 + half * 2;
          if constexpr (kRows8) {
            mma_rows8(o[j][0], o[j][1], pa[0], pa[1], P::template get<false>(lo), P::template get<false>(hi));
            mma_rows8(o[j + 1][0], o[j + 1][1], pa[0], pa[1], P::template get<true>(lo), P::template get<true>(hi));
          } else {
            mma_16816_nv<false>(o[j], pa, P::template get<false>(lo), P::template get<false>(hi));
            mma_16816_nv<false>(o[j + 1], pa, P::template get<true>(lo), P::template get<true>(hi));
          }
        }
      }
      if (next) load_values();
    }
    if (seg.first + warp >= seg.last && has_next_seg) {  // no page of this segment: fetch the next one's
      locate(nseg.r, nseg.kvh, nseg.first + warp);
      load_keys();
      load_values();
    }

    // The warps' sums: O of row g at elements (D / 4) t + j and (D / 4) t + D / 8 + j.
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = g + 8 * h;
      if (t == 0) m_sm[warp][row] = m[h], l_sm[warp][row] = l[h];
#pragma unroll
      for (int j = 0; j < kNTiles; ++j) {
        o_sm[warp][row][t * (D / 4) + j] = o[j][2 * h];
        o_sm[warp][row][t * (D / 4) + D / 8 + j] = o[j][2 * h + 1];
      }
    }
    __syncthreads();
    const bool whole = seg.first == 0 && seg.last == seg.pages;
    const int slot = 2 * blockIdx.x + (seg.first == 0 ? 1 : 0);
    for (int i = tid; i < seg.rows * (D / 4); i += kThreads) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_sm[w][row]);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float wt = m_sm[w][row] == -INFINITY ? 0.f : exp2_fast(m_sm[w][row] - top);
        const float4 v = *reinterpret_cast<const float4 *>(&o_sm[w][row][d]);
        sum = fmaf(wt, l_sm[w][row], sum);
        acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y);
        acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
      }
      if (whole) {
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        const int tok = row / a.group, head = row - tok * a.group;
        uint16_t *dst = a.out + (seg.q0 + tok) * a.out_stride + (seg.kvh * a.group + head) * D + d;
        dst[0] = from_float<kBf16>(acc.x * inv), dst[1] = from_float<kBf16>(acc.y * inv);
        dst[2] = from_float<kBf16>(acc.z * inv), dst[3] = from_float<kBf16>(acc.w * inv);
      } else {
        *reinterpret_cast<float4 *>(a.part_o + (static_cast<int64_t>(slot) * kMaxRows + row) * D + d) = acc;
        if (d == 0) a.part_ml[slot * kMaxRows + row] = make_float2(top, sum);
      }
    }
    if (!whole) {
      // The item's flat range, the CTAs that hold a piece of it, and how many.
      const long long item = at - seg.first;
      const int c0 = static_cast<int>(item / run), c1 = static_cast<int>((item + seg.pages - 1) / run);
      uint32_t *count = a.counts + static_cast<int64_t>(seg.r) * s.hkv + seg.kvh;
      __threadfence();
      __syncthreads();
      if (tid == 0) last_sm = atomicAdd(count, 1u) == static_cast<uint32_t>(c1 - c0);
      __syncthreads();
      if (last_sm) {
        __threadfence();
        if (tid == 0) *count = 0;
        for (int i = tid; i < seg.rows * (D / 4); i += kThreads) {
          const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
          float top = -INFINITY;
          for (int c = c0; c <= c1; ++c) {
            const int sl = 2 * c + (c == c0 ? 1 : 0);
            top = fmaxf(top, __ldcg(&a.part_ml[sl * kMaxRows + row]).x);
          }
          float sum = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c = c0; c <= c1; ++c) {
            const int sl = 2 * c + (c == c0 ? 1 : 0);
            const float2 ml = __ldcg(&a.part_ml[sl * kMaxRows + row]);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(a.part_o + (static_cast<int64_t>(sl) * kMaxRows + row) * D + d));
            const float wt = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top);
            sum = fmaf(wt, ml.y, sum);
            acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y);
            acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
          }
          const float inv = sum > 0.f ? 1.f / sum : 0.f;
          const int tok = row / a.group, head = row - tok * a.group;
          uint16_t *dst = a.out + (seg.q0 + tok) * a.out_stride + (seg.kvh * a.group + head) * D + d;
          dst[0] = from_float<kBf16>(acc.x * inv), dst[1] = from_float<kBf16>(acc.y * inv);
          dst[2] = from_float<kBf16>(acc.z * inv), dst[3] = from_float<kBf16>(acc.w * inv);
        }
      }
    }
    __syncthreads();  // o_sm is free again
    at += seg.last - seg.first;
    seg = nseg;
  }
}

}  // namespace kv8
}  // namespace lvb
