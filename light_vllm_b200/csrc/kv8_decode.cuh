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
// ever multiplied by a scale.  They enter it as fp16, times 2^6 (kHead) and up to
// 2^8 (kLazy) more, so that a weight 2^-20 of the largest still has 11 bits; O, L,
// m and the scores are fp32.  m moves only when it would grow by more than kLazy:
// a rescaling of O is rare.
//
// Tensor cores.  Both products are m16n8k16 warp MMAs with 16 positions (then 16
// elements of the head) as M and the query rows as N, so up to 8 rows waste
// nothing.  Codes are exact in fp16: int8 by setting the byte under the exponent
// of 1024 and subtracting 1152, e4m3 by the hardware's conversion.  The order of
// the head's elements in q k^T, and of a page's positions, is free as long as
// both operands agree, so lane (g, t) of the fragment takes 16 consecutive bytes
// of key rows g and g + 8, and of value rows 2t, 2t + 1, 2t + 8, 2t + 9.  A lane
// only ever reads what it fetched itself: asynchronous copies bring its pieces
// of the next two pages into its own slots of shared memory, with no barrier.
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

constexpr float kHead = 6.f;
constexpr float kLazy = 8.f;
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
  bool query_vec, out_vec;  // rows allow 16-byte loads, 8-byte stores
  float scale_log2;  // softmax scale * log2(e)
  int few_rows;      // requests of up to this many query rows are the decode kernel's
  // Pieces of items that cross CTAs, and how many of an item's CTAs are done
  // (kept at the CTA that the item begins in; zero between calls).
  float *part_o;         // decode kernel: [2 * CTAs][kMaxRows][D]
  float2 *part_ml;       // [2 * CTAs][kMaxRows]: m, L
  uint32_t *counts;      // [CTAs]
  float *tile_o;         // tile kernel: [2 * CTAs][kTileRows][D]
  float2 *tile_ml;       // [2 * CTAs][kTileRows]
  uint32_t *tile_counts;  // [CTAs]
};

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

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void lds_16(uint32_t (&v)[4], uint32_t src) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}

__device__ __forceinline__ void lds_8(uint32_t (&v)[2], uint32_t src) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(src) : "memory");
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) { return pack2<false>(lo, hi); }

// Eight elements of a row, one load where rows are 16-byte aligned.
template <bool kBf16>
__device__ __forceinline__ void load8(const uint16_t *src, bool some, bool vec, float (&x)[8]) {
  uint4 v = make_uint4(0, 0, 0, 0);
  uint16_t *e = reinterpret_cast<uint16_t *>(&v);
  if (some && vec) {
    v = *reinterpret_cast<const uint4 *>(src);
  } else if (some) {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = src[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<kBf16>(e[i]);
}

template <bool kBf16>
__device__ __forceinline__ void store8(uint16_t *dst, bool vec, const float (&x)[8]) {
  if (vec) {
    *reinterpret_cast<uint4 *>(dst) =
        make_uint4(pack2<kBf16>(x[0], x[1]), pack2<kBf16>(x[2], x[3]), pack2<kBf16>(x[4], x[5]), pack2<kBf16>(x[6], x[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = from_float<kBf16>(x[i]);
  }
}

// The power of two that brings `top` to [2^to, 2^(to + 1)), within the normal range.
__device__ __forceinline__ float scale_to(float top, int to) {
  const int field = static_cast<int>(__float_as_uint(top) >> 23);
  return __uint_as_float(static_cast<uint32_t>(min(max(254 + to - field, 1), 254)) << 23);
}

__device__ __forceinline__ void named_barrier_256() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

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
    return scale_to(top, 7);
  }
}

// One run of pages of one item.
struct Segment {
  int r, kvh, first, last;  // pages [first, last)
  int pages;                // of the whole item
  int q0, rows, computed;
};

// kNT: tiles of 8 query rows.
template <int D, int kNT>
struct DecodeCfg {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtasPerSm = kNT == 1 ? 2 : 1;
  static constexpr int kRows = 8 * kNT;
  static constexpr int kPad = D + 4;                // floats of a row of O in shared memory
  static constexpr int kPageBytes = 2 * kPage * D;  // K and V
  static constexpr int kSlots = 2;                  // pages in flight for each warp
  static constexpr int kRingBytes = kWarps * kSlots * kPageBytes;
  static constexpr int kOBytes = kWarps * kRows * kPad * 4;
  static constexpr int kSmemBytes = kRingBytes + kOBytes;
};

__device__ __forceinline__ void cp_async_8(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

template <bool kBf16, bool kFp8, int D, int kNT>
__global__ void __launch_bounds__(DecodeCfg<D, kNT>::kThreads, DecodeCfg<D, kNT>::kCtasPerSm)
    decode_kernel(const __grid_constant__ AttnArgs a) {
  using Cfg = DecodeCfg<D, kNT>;
  using P = Pair<kFp8>;
  constexpr int kWarps = Cfg::kWarps, kThreads = Cfg::kThreads, kRows = Cfg::kRows;
  constexpr int kKSteps = D / 16;   // MMAs of a score tile
  constexpr int kDTiles = D / 16;   // MMAs of O
  constexpr int kKChunks = D / 64;  // 16-byte pieces of a key row that a lane takes
  constexpr int kVWords = D / 32;   // words of a value row that a lane takes
  constexpr float kNone = -1e30f;   // m before any position
  extern __shared__ __align__(16) uint8_t smem[];
  float *o_sm = reinterpret_cast<float *>(smem + Cfg::kRingBytes);  // [warp][row][kPad]
  __shared__ float m_sm[kWarps][kRows], l_sm[kWarps][kRows];
  __shared__ int scan[kWarps];
  __shared__ long long start_pages;  // pages before the run's first request
  __shared__ int start_request, last_sm;
  pdl_wait();
  const Step &s = a.step;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // Pages of request r's items (0: not this kernel's, or refused).
  auto request_pages = [&](int r) {
    int q0, n, c;
    if (!request_range(s, r, q0, n, c) || n == 0 || n * a.group > a.few_rows) return 0;
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
  int mine = 0, sum = 0, ex = 0;
  for (int base = 0; base < s.num_seqs; base += kThreads) {
    mine = base + tid < s.num_seqs ? request_pages(base + tid) : 0;
    ex = block_scan(mine, sum);
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
      if (s.num_seqs > kThreads) {
        mine = base + tid < s.num_seqs ? request_pages(base + tid) : 0;
        ex = block_scan(mine, sum);
      }
      const long long lo = before + static_cast<long long>(ex) * s.hkv, hi = lo + static_cast<long long>(mine) * s.hkv;
      if (lo <= begin && begin < hi) {
        start_request = base + tid;
        start_pages = lo;
      }
      before += static_cast<long long>(sum) * s.hkv;
    }
    __syncthreads();
  }

  auto describe = [&](int r, int kvh, int first, int left, Segment &seg) {
    seg.r = r;
    seg.kvh = kvh;
    seg.q0 = s.qsl[r];
    seg.computed = s.computed[r];
    const int n = s.qsl[r + 1] - seg.q0;
    seg.rows = n * a.group;
    seg.pages = (seg.computed + n + kPage - 1) / kPage;
    seg.first = first;
    seg.last = left < seg.pages - first ? first + left : seg.pages;
  };
  int left = static_cast<int>(end - begin);  // pages of the run from the present segment on
  Segment seg;
  {
    const int r = start_request;
    const int pages = request_pages(r);
    const int inside = static_cast<int>(begin - start_pages);
    describe(r, inside / pages, inside % pages, left, seg);
  }
  // The segment after `from`; false at the end of the run.
  auto next_segment = [&](const Segment &from, Segment &to) {
    const int rest = left - (from.last - from.first);
    if (rest <= 0) return false;
    int r = from.r, kvh = from.kvh + 1;
    if (kvh == s.hkv) {
      kvh = 0;
      do {
        ++r;
      } while (request_pages(r) == 0);  // pages are left, so a request is
    }
    describe(r, kvh, 0, rest, to);
    return true;
  };

  // This lane's pieces of a page: 2 kKChunks of 16 bytes of K, four of 4 kVWords bytes of V.
  const uint32_t ring = smem_u32(smem) + warp * (Cfg::kSlots * Cfg::kPageBytes);
  const int ppb = s.bs / kPage;
  const uint32_t head_bytes = static_cast<uint32_t>(s.bs) * D;
  const uint8_t *k_lane = a.key_codes + g * D + t * 16;
  const uint8_t *v_lane = a.value_codes + 2 * t * D + g * (D / 8);
  float ks_ring[Cfg::kSlots], vs_ring[Cfg::kSlots];  // scales; ks NaN: block id out of range
  auto fetch = [&](const Segment &of, int p, int slot) {
    const int blk = ppb == 1 ? p : p / ppb;
    int phys = s.tables[of.r * s.table_stride + blk];
    const bool bad = static_cast<uint32_t>(phys) >= static_cast<uint32_t>(s.num_blocks);
    if (bad) {
      record_device_error(LVB_DEVERR_INDEX);
      phys = 0;
    }
    const uint32_t h = static_cast<uint32_t>(phys) * s.hkv + of.kvh;
    ks_ring[slot] = bad ? NAN : __ldg(a.key_scales + h);
    vs_ring[slot] = __ldg(a.value_scales + h);
    const uint64_t at = static_cast<uint64_t>(h) * head_bytes + (p - blk * ppb) * (kPage * D);
    const uint8_t *kp = k_lane + at, *vp = v_lane + at;
    const uint32_t dst = ring + slot * Cfg::kPageBytes;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kKChunks; ++c)
        cp_async_16(dst + ((i * kKChunks + c) * 32 + lane) * 16, kp + i * 8 * D + c * 64, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *src = vp + ((i & 1) + (i >> 1) * 8) * D;
      if constexpr (D == 128)
        cp_async_16(dst + kPage * D + (i * 32 + lane) * 16, src, 16);
      else
        cp_async_8(dst + kPage * D + (i * 32 + lane) * 8, src);
    }
  };

  // Pages of the run that this warp takes, in order, across segments: (fs, fp)
  // is the next one to fetch.
  Segment fs = seg;
  int fp = seg.first + warp;
  int fleft = left;
  bool fmore = true;
  auto fetch_next = [&](int slot) {
    while (fmore && fp >= fs.last) {
      Segment n;
      const int keep = left;
      left = fleft;
      fmore = next_segment(fs, n);
      left = keep;
      if (fmore) {
        fleft -= fs.last - fs.first;
        fs = n;
        fp = fs.first + warp;
      }
    }
    if (fmore) {
      fetch(fs, fp, slot);
      fp += kWarps;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < Cfg::kSlots; ++i) fetch_next(i);
  int slot = 0;

  bool more = true;
  while (more) {
    // Query rows n = g (B fragments), and rows 2t, 2t + 1 (scores): row i is
    // token i / group, head i % group.
    uint32_t qb[kNT][kKSteps][2];
    float f[kNT][2];
    int limit[kNT][2];  // last position that the row sees
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int row = n * 8 + g;
      const bool ok = row < seg.rows;
      const int tok = ok ? row / a.group : 0, head = ok ? row - tok * a.group : 0;
      const uint16_t *src = a.query + (seg.q0 + tok) * a.query_stride + (seg.kvh * a.group + head) * D + t * 16;
      float x[kKChunks * 16];
#pragma unroll
      for (int c = 0; c < kKChunks; ++c) {
        if (a.query_vec) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (ok) v = *reinterpret_cast<const uint4 *>(src + c * 64 + i * 8);
            const uint16_t *e = reinterpret_cast<const uint16_t *>(&v);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[c * 16 + i * 8 + k] = to_float<kBf16>(e[k]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[c * 16 + i] = ok ? to_float<kBf16>(src[c * 64 + i]) : 0.f;
        }
      }
      const float up = query_shift<kBf16>(x);
      const float fr = a.scale_log2 / up;
      const int lim = ok ? seg.computed + tok : -1;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[n][e] = __shfl_sync(0xffffffffu, fr, (2 * t + e) * 4);
        limit[n][e] = __shfl_sync(0xffffffffu, lim, (2 * t + e) * 4);
      }
#pragma unroll
      for (int k = 0; k < kKSteps; ++k) {
        qb[n][k][0] = pack_half(x[4 * k] * up, x[4 * k + 1] * up);
        qb[n][k][1] = pack_half(x[4 * k + 2] * up, x[4 * k + 3] * up);
      }
    }
    float o[kNT][kDTiles][4], m[kNT][2], l[kNT][2];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int j = 0; j < kDTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) m[n][e] = kNone, l[n][e] = 0.f;
    }

    for (int p = seg.first + warp; p < seg.last; p += kWarps) {
      cp_async_wait_group<Cfg::kSlots - 1>();
      const uint32_t src = ring + slot * Cfg::kPageBytes;
      const float ks = slot == 0 ? ks_ring[0] : ks_ring[1], vs = slot == 0 ? vs_ring[0] : vs_ring[1];
      const bool bad = ks != ks;
      uint32_t kreg[2][kKChunks][4], vreg[4][kVWords];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < kKChunks; ++c) lds_16(kreg[i][c], src + ((i * kKChunks + c) * 32 + lane) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (D == 128)
          lds_16(vreg[i], src + kPage * D + (i * 32 + lane) * 16);
        else
          lds_8(vreg[i], src + kPage * D + (i * 32 + lane) * 8);
      }
      // Scores: positions g and g + 8 by rows 2t and 2t + 1.
      float sc[kNT][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < kKSteps; ++k) {
        const uint32_t w0 = P::bias(kreg[0][k >> 2][k & 3]), w1 = P::bias(kreg[1][k >> 2][k & 3]);
        const uint32_t ka[4] = {P::template get<false>(w0), P::template get<false>(w1), P::template get<true>(w0),
                                P::template get<true>(w1)};
#pragma unroll
        for (int n = 0; n < kNT; ++n) mma_16816_nv<false>(sc[n], ka, qb[n][k][0], qb[n][k][1]);
      }
      const float vw = vs > 0.f ? vs : 1.f;
      const float lw = log2_fast(vw), iw = rcp_fast(vw);
      const bool masked = bad || p * kPage + kPage - 1 > seg.computed;
      // Exponents against the present m, plus kHead.
      float y[kNT][4];
      auto exponents = [&]() {
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[n][i] = fmaf(sc[n][i], f[n][i & 1] * ks, lw - m[n][i & 1] + kHead);
        if (masked) {
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (bad || p * kPage + g + (i >> 1) * 8 > limit[n][i & 1]) y[n][i] = -INFINITY;
        }
      };
      exponents();
      bool grow = false;
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) grow |= y[n][i] > kHead + kLazy;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // the scores themselves: y is too coarse beside m = kNone
            float top = m[n][e];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (y[n][2 * i + e] != -INFINITY) top = fmaxf(top, fmaf(sc[n][2 * i + e], f[n][e] * ks, lw));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float alpha = exp2_fast(m[n][e] - top);
            m[n][e] = top;
            l[n][e] *= alpha;
#pragma unroll
            for (int j = 0; j < kDTiles; ++j) o[n][j][e] *= alpha, o[n][j][2 + e] *= alpha;
          }
        exponents();
      }
      uint32_t pb[kNT][2];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[n][i] = exp2_fast(y[n][i]);
        l[n][0] = fmaf(y[n][0] + y[n][2], iw, l[n][0]);
        l[n][1] = fmaf(y[n][1] + y[n][3], iw, l[n][1]);
        pb[n][0] = movmatrix_trans(pack_half(y[n][0], y[n][1]));
        pb[n][1] = movmatrix_trans(pack_half(y[n][2], y[n][3]));
      }
      if (kFp8 && masked) {
        // Slots past the end may hold NaN patterns: 0 * NaN is not 0.
        const int stop = bad ? 0 : seg.computed + seg.rows / a.group;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p * kPage + 2 * t + (i & 1) + (i >> 1) * 8 >= stop)
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vreg[i][w] = 0;
      }
      // O: elements (D / 8) g + 2 j (rows g of the tile) and + 1 (rows g + 8).
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // bytes (2 half, 2 half + 1) of value rows (0, 1) and (2, 3), interleaved
          const uint32_t lo = P::bias(__byte_perm(vreg[0][w], vreg[1][w], half ? 0x7362 : 0x5140));
          const uint32_t hi = P::bias(__byte_perm(vreg[2][w], vreg[3][w], half ? 0x7362 : 0x5140));
          const uint32_t va[4] = {P::template get<false>(lo), P::template get<true>(lo), P::template get<false>(hi),
                                  P::template get<true>(hi)};
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma_16816_nv<false>(o[n][2 * w + half], va, pb[n][0], pb[n][1]);
        }
      }
      // Everything of this slot is in registers and used: refill it.
      if (slot == 0) fetch_next(0); else fetch_next(1);
      slot ^= 1;
    }

    // The warps' sums.
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        const int row = n * 8 + 2 * t + e;
        if (g == 0) m_sm[warp][row] = m[n][e], l_sm[warp][row] = l[n][e];
        float *dst = o_sm + (warp * kRows + row) * Cfg::kPad + g * (D / 8);
#pragma unroll
        for (int j = 0; j < kDTiles; j += 2)
          *reinterpret_cast<float4 *>(dst + 2 * j) = make_float4(o[n][j][e], o[n][j][2 + e], o[n][j + 1][e], o[n][j + 1][2 + e]);
      }
    __syncthreads();
    const bool whole = seg.first == 0 && seg.last == seg.pages;
    const int piece = 2 * blockIdx.x + (seg.first == 0 ? 1 : 0);
    auto store = [&](int row, int d, float4 v, float total_l) {
      const float inv = total_l > 0.f ? 1.f / total_l : 0.f;
      const int tok = row / a.group, head = row - tok * a.group;
      uint16_t *dst = a.out + (seg.q0 + tok) * a.out_stride + (seg.kvh * a.group + head) * D + d;
      if (a.out_vec) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<kBf16>(v.x * inv, v.y * inv), pack2<kBf16>(v.z * inv, v.w * inv));
      } else {
        dst[0] = from_float<kBf16>(v.x * inv), dst[1] = from_float<kBf16>(v.y * inv);
        dst[2] = from_float<kBf16>(v.z * inv), dst[3] = from_float<kBf16>(v.w * inv);
      }
    };
    for (int i = tid; i < seg.rows * (D / 4); i += kThreads) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
      float top = kNone;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_sm[w][row]);
      float sum_l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float wt = exp2_fast(m_sm[w][row] - top);
        const float4 v = *reinterpret_cast<const float4 *>(o_sm + (w * kRows + row) * Cfg::kPad + d);
        sum_l = fmaf(wt, l_sm[w][row], sum_l);
        acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y);
        acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
      }
      if (whole) {
        store(row, d, acc, sum_l);
      } else {
        *reinterpret_cast<float4 *>(a.part_o + (static_cast<int64_t>(piece) * kMaxRows + row) * D + d) = acc;
        if (d == 0) a.part_ml[piece * kMaxRows + row] = make_float2(top, sum_l);
      }
    }
    if (!whole) {
      // The CTAs that hold a piece of the item.
      const long long item = end - left - seg.first;
      const int c0 = static_cast<int>(item / run), c1 = static_cast<int>((item + seg.pages - 1) / run);
      uint32_t *count = a.counts + c0;
      __threadfence();
      __syncthreads();
      if (tid == 0) last_sm = atomicAdd(count, 1u) == static_cast<uint32_t>(c1 - c0);
      __syncthreads();
      if (last_sm) {
        __threadfence();
        if (tid == 0) *count = 0;
        for (int i = tid; i < seg.rows * (D / 4); i += kThreads) {
          const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
          float top = kNone;
          for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(&a.part_ml[(2 * c + (c == c0)) * kMaxRows + row]).x);
          float sum_l = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = c0; c <= c1; ++c) {
            const int at = (2 * c + (c == c0)) * kMaxRows + row;
            const float2 ml = __ldcg(&a.part_ml[at]);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(a.part_o + static_cast<int64_t>(at) * D + d));
            const float wt = exp2_fast(ml.x - top);
            sum_l = fmaf(wt, ml.y, sum_l);
            acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y);
            acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
          }
          store(row, d, acc, sum_l);
        }
      }
    }
    __syncthreads();  // o_sm is free again
    Segment n;
    more = next_segment(seg, n);
    left -= seg.last - seg.first;
    if (more) seg = n;
  }
}

}  // namespace kv8
}  // namespace lvb
