// Attention of few query rows over the 8-bit paged cache: requests whose query
// tokens times the query heads of one KV head are at most 64 (decode steps, and
// the verification of a few drafts).  Up to 32 rows (40 for heads of 64) K and V
// are read once for all of them, above by two row groups that follow each other
// (the second time from L2).  Bound by those bytes.
//
// Mathematics.  With f_b = scale log2(e) key_scale_b and w_b = value_scale_b of
// a position's block b, x_j = (q . key code_j) f_b + log2 w_b and a running
// maximum m of x, the sums
//     O = sum_j 2^(x_j - m) value code_j        L = sum_j 2^(x_j - m) / w_b
// give out = O / L: the value scale rides in the exponent, so the weights that
// enter the second product lie in (0, 1] whatever the scales are, and no code is
// ever multiplied by a scale.  (w_b = 0, a block of zeros, stands as kZeroWeight,
// below every live block's: it adds to L and does not raise m, which would push the
// others' weights out of fp16.)  They enter it as fp16, times 2^6 (kHead) and up to
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
// of the next pages into its own slots of shared memory, with no barrier, keys as
// soon as the present ones are used, values likewise.  A step takes two pages (one
// where there are many rows), so that their chains of MMAs and exponentials overlap.
// Nothing of the page loop waits for a load of its own: the blocks of
// 32 pages are read at once and ahead of the copies, scales come with the codes (a register that a branch
// or a select touches waits for its load there: 1 us of each page), and nothing of
// it lies in local memory.
//
// Split.  The pages of all (request, KV head, row group) items are laid end to
// end, each item preceded by pages' worth of what it costs besides (kItemCost), and
// cut into one equal run for each resident CTA, whatever the contexts' lengths;
// the warps of a CTA take its pages in turn.  An item that ends in another CTA
// leaves partial (O, m, L) in the workspace, and the last of its CTAs to finish (a
// counter for each item) sums them in order, so results do not depend on timing.
//
// Measured: 64 requests of 512 to 4096 tokens, 28/4 heads of 128, int8: 49 us (3.1
// TB/s): 25 in which pages pass at about 6 TB/s, 7 of start, 5 of joins, some 8 in
// which SMs have ended (they are active for 78 of 92 thousand cycles: some reach
// memory more slowly than others), the launch.  5 tokens each for 32 requests of up
// to 8000, 14/2 heads of 64: 36 us.
#pragma once

#include <type_traits>

#include "kv8_cache.cuh"

namespace lvb {
namespace kv8 {

constexpr float kHead = 6.f;
constexpr float kLazy = 8.f;
// With it L stays below 2^(80 + 6 + 8) for each position, and a weight at the least
// scale that append keeps, 2^-100, is a normal fp16 beside a block of zeros.
constexpr float kZeroWeight = 0x1p-80f;
constexpr int kPage = 16;     // positions a warp takes at a time
// Query rows of a decode item (their O in registers: 80 of them at 40 x 64).
template <int D>
constexpr int kMaxRows = D == 64 ? 40 : 32;
constexpr int kMinRun = 16;    // pages of a CTA, at least: more CTAs only merge more
constexpr int kSmallCost = 8;  // and pages' worth of an item's beginning there

struct AttnArgs {
  Step step;
  const uint16_t *query;
  int64_t query_stride;
  uint16_t *out;
  int64_t out_stride;
  const uint8_t *key_codes, *value_codes;
  const float *key_scales, *value_scales;
  int group;         // query heads of a KV head
  float scale_log2;  // softmax scale * log2(e)
  int few_rows;      // requests of up to this many query rows are the decode kernel's
  // Pieces of items that cross CTAs, and how many of an item's CTAs are done
  // (kept at the CTA that the item begins in; zero between calls).
  float *part_o;         // decode kernel: [2 * CTAs][its rows][D]
  float2 *part_ml;       // [2 * CTAs][its rows]: m, L
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

// Shared-memory loads and copies at constant offsets (in the instruction, not in
// registers of their own).
template <int kOff>
__device__ __forceinline__ void lds_16(uint32_t (&v)[4], uint32_t src) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(src), "n"(kOff)
               : "memory");
}

template <int kOff>
__device__ __forceinline__ void lds_8(uint32_t (&v)[2], uint32_t src) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2 + %3];" : "=r"(v[0]), "=r"(v[1]) : "r"(src), "n"(kOff) : "memory");
}

template <int kBytes, int kDst, int kSrc>
__device__ __forceinline__ void copy_at(uint32_t dst, const void *src) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(kDst), "n"(kSrc) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0 + %2], [%1 + %3], 8;" ::"r"(dst), "l"(src), "n"(kDst), "n"(kSrc) : "memory");
}

// f(integral_constant 0), .., f(integral_constant N - 1)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F &&f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) { return pack2<false>(lo, hi); }

// The power of two that brings `top` to [2^to, 2^(to + 1)), within the normal range.
__device__ __forceinline__ float scale_to(float top, int to) {
  const int field = static_cast<int>(__float_as_uint(top) >> 23);
  return __uint_as_float(static_cast<uint32_t>(min(max(254 + to - field, 1), 254)) << 23);
}

__device__ __forceinline__ void named_barrier_256() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// A row of queries as fp16 times 2^shift (returned): fp16 rows as they are; bf16
// rows with their largest element brought to [2^7, 2^8), which keeps every element
// down to 2^-22 of it exact, and smaller ones to 2^-32 of it.
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
  int r, kvh, group;        // the item
  int first, last, pages;   // pages [first, last) of it, and all
  int q0, rows, computed;   // rows: of the whole request and KV head
  long long at;             // flat place of the item's first page
};

// kNT: tiles of 8 query rows.
template <int D, int kNT>
struct DecodeCfg {
  // (Small CTAs, so that one's end of an item passes beside the others' pages.)
  static constexpr int kWarps = kNT == 1 ? 4 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtasPerSm = kNT == 1 ? 4 : 1;
  static constexpr int kRows = 8 * kNT;
  static constexpr int kPad = D + 4;                // floats of a row of O in shared memory
  static constexpr int kPages = kNT <= (D == 64 ? 3 : 2) ? 2 : 1;  // pages of a step
  // An item's queries, sums and joining in pages of the CTA's time: with 5 tiles
  // of rows and heads of 64 they take 14K cycles and a page 280.  Measured at 2 to 5
  // tiles and two groups of 3, heads of 64 and 128, batches of 32 and 64 requests:
  // 20 is 5 to 22 % slower and 10 up to 33 %, 80 within 6 % either way; 8 requests of
  // up to 3000 tokens take 40 best too (20: up to 18 % slower, 80: up to 9 %).
  static constexpr int kItemCost = kNT == 1 ? 8 : 40;
  static constexpr int kSide = kPage * D;           // K (or V) of a page
  static constexpr int kRingBytes = kWarps * kPages * 2 * kSide;
  // The warps' sums meet in shared memory in two halves.
  static constexpr int kMeet = kWarps / 2;
  static constexpr int kOBytes = kMeet * kRows * kPad * 4;
  static constexpr int kQBytes = kNT == 1 ? 0 : kNT * (D / 16) * 32 * 8;  // query fragments
  static constexpr int kScaleOff = kRingBytes + kOBytes + kQBytes;  // float [warp][page]{key, value}
  static constexpr int kSmemBytes = kScaleOff + kWarps * kPages * 8;
};

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A request of the decode kernel's: its first token, tokens and computed count;
// n = 0: not its, or refused.
struct Request {
  int q0, n, computed;
};

__device__ __forceinline__ Request decode_request(const Step &s, int group, int few_rows, int r) {
  Request q;
  if (!request_range(s, r, q.q0, q.n, q.computed) || q.n * group > few_rows) q.n = 0;
  return q;
}

__device__ __forceinline__ int pages_of(const Request &q) { return (q.computed + q.n + kPage - 1) / kPage; }

// To the run's next item with pages of the run; false at its end.  The flat order
// is walked in steps of an item's cost, its pages and `more`, rounded up to `unit`.
__device__ __noinline__ bool next_item(const Step &s, int group_heads, int few_rows, int rows_each, int unit, int more,
                                       long long end, Segment &seg) {
  const int cost = (seg.pages + more + unit - 1) / unit * unit;
  const long long at = seg.at + cost;
  if (at >= end) return false;
  int r = seg.r, kvh = seg.kvh, group = seg.group + 1;
  if (group * rows_each >= seg.rows) {
    group = 0;
    if (++kvh == s.hkv) {
      kvh = 0;
      Request q;
      do {
        if (++r == s.num_seqs) return false;
        q = decode_request(s, group_heads, few_rows, r);
      } while (q.n == 0);
      seg.r = r;
      seg.q0 = q.q0;
      seg.computed = q.computed;
      seg.rows = q.n * group_heads;
      seg.pages = pages_of(q);
    }
  }
  seg.kvh = kvh;
  seg.group = group;
  seg.at = at;
  seg.first = 0;  // (the run began before)
  seg.last = static_cast<int>(end - at < seg.pages ? end - at : seg.pages);
  return true;
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
  float *o_sm = reinterpret_cast<float *>(smem + Cfg::kRingBytes);                        // [kMeet][row][kPad]
  uint2 *q_sm = reinterpret_cast<uint2 *>(smem + Cfg::kRingBytes + Cfg::kOBytes);         // [kNT][kKSteps][32]
  __shared__ float m_sm[kWarps][kRows], l_sm[kWarps][kRows];
  __shared__ longlong2 scan[kWarps];
  __shared__ Segment start_sm;
  __shared__ int last_sm;
  pdl_wait();
  const Step &s = a.step;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // What the items of a request come to (rounded up to `unit` each).
  auto request_cost = [&](const Request &q, int unit, int more) {
    if (q.n == 0) return 0ll;
    const int cost = (pages_of(q) + more + unit - 1) / unit * unit;
    return static_cast<long long>(cost) * ((q.n * a.group + kRows - 1) / kRows) * s.hkv;
  };
  // Inclusive prefix of two values over the CTA; `all` are the totals.
  auto block_scan = [&](longlong2 v, longlong2 &all) {
    longlong2 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x.x, o), z = __shfl_up_sync(0xffffffffu, x.y, o);
      if (lane >= o) x.x += y, x.y += z;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    all = make_longlong2(0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) x.x += scan[w].x, x.y += scan[w].y;
      all.x += scan[w].x, all.y += scan[w].y;
    }
    return x;
  };
  // A batch that gives every CTA at most kSmallRun pages is cut at the items'
  // starts: a piece each for the CTAs, and short items are not cut at all.
  // Otherwise the flat order is cut into equal runs.
  constexpr int kItemCost = Cfg::kItemCost, kSmallRun = kMinRun + kSmallCost;
  Request mine{};
  longlong2 totals = make_longlong2(0, 0), sum, upto = totals;  // x: equal runs, y: pieces
#pragma unroll 1
  for (int base = 0; base < s.num_seqs; base += kThreads) {
    mine.n = 0;
    if (base + tid < s.num_seqs) mine = decode_request(s, a.group, a.few_rows, base + tid);
    upto = block_scan(make_longlong2(request_cost(mine, 1, kItemCost), request_cost(mine, kSmallRun, kSmallCost)), sum);
    totals.x += sum.x;
    totals.y += sum.y;
  }
  const int unit = totals.y <= static_cast<long long>(kSmallRun) * gridDim.x ? kSmallRun : 1;
  const int item_cost = unit > 1 ? kSmallCost : kItemCost;
  const long long total = unit > 1 ? totals.y : totals.x;
  const long long run = unit > 1 ? unit : (total + gridDim.x - 1) / gridDim.x;
  const long long begin = run * blockIdx.x;
  if (begin >= total) return;
  const long long end = begin + run < total ? begin + run : total;
  {
    long long before = 0;
#pragma unroll 1
    for (int base = 0; base < s.num_seqs; base += kThreads) {
      if (s.num_seqs > kThreads) {
        mine.n = 0;
        if (base + tid < s.num_seqs) mine = decode_request(s, a.group, a.few_rows, base + tid);
        upto = block_scan(make_longlong2(request_cost(mine, 1, kItemCost), request_cost(mine, kSmallRun, kSmallCost)), sum);
      }
      const long long hi = before + (unit > 1 ? upto.y : upto.x), lo = hi - request_cost(mine, unit, item_cost);
      if (lo <= begin && begin < hi) {
        // The run begins in one of this thread's request's items.
        const int pages = pages_of(mine), cost = (pages + item_cost + unit - 1) / unit * unit, rows = mine.n * a.group;
        const int item = static_cast<int>((begin - lo) / cost), groups = (rows + kRows - 1) / kRows;
        Segment seg;
        seg.r = base + tid;
        seg.kvh = item / groups;
        seg.group = item % groups;
        seg.at = lo + static_cast<long long>(item) * cost + item_cost;
        seg.q0 = mine.q0;
        seg.rows = rows;
        seg.computed = mine.computed;
        seg.pages = pages;
        seg.first = static_cast<int>(begin > seg.at ? begin - seg.at : 0);
        seg.last = static_cast<int>(end - seg.at < pages ? (end > seg.at ? end - seg.at : 0) : pages);
        start_sm = seg;
      }
      if (s.num_seqs > kThreads) before += unit > 1 ? sum.y : sum.x;
    }
    __syncthreads();
  }
  // Walked twice, by the page loop and, ahead of it, by the copies.
  Segment walk_m = start_sm, walk_f = walk_m;
  auto advance = [&](Segment &walk) { return next_item(s, a.group, a.few_rows, kRows, unit, item_cost, end, walk); };

  // This lane's pieces of a page: 2 kKChunks of 16 bytes of K, four of 4 kVWords bytes of V.
  constexpr int kPages = Cfg::kPages, kSideBytes = Cfg::kSide;
  const uint32_t ring = smem_u32(smem) + warp * (kPages * 2 * kSideBytes);  // [page][K, V][piece][lane]
  const uint32_t ring16 = ring + lane * 16, ring_v = ring + kSideBytes + lane * (D / 8);
  const int ppb = s.bs / kPage;
  const uint32_t per_block = ppb > 1 ? 0xffffffffu / ppb + 1 : 0u;  // 2^32 / ppb, rounded up: exact for p * ppb < 2^32
  auto block_of = [&](int p) { return ppb == 1 ? p : static_cast<int>(__umulhi(p, per_block)); };
  const uint8_t *k_lane = a.key_codes + g * D + t * 16;
  const uint8_t *v_lane = a.value_codes + 2 * t * D + g * (D / 8);
  // Scales come the same way: lane 2 i brings page i's key scale, 2 i + 1 its value scale.
  const uint32_t scale_ring = smem_u32(smem) + Cfg::kScaleOff + warp * (kPages * 8);
  const float *scale_lane = (lane & 1) == 0 ? a.key_scales : a.value_scales;
  // The next step's pages (f_p .. of f_last, their KV head and table).  The blocks
  // of the next 32 pages are in the lanes' f_ids, read in one go, so that no copy
  // waits for its block.
  const int32_t *f_table = s.tables + walk_f.r * s.table_stride;
  int f_p = walk_f.first + warp * kPages, f_last = walk_f.last, f_kvh = walk_f.kvh, f_ids = 0, f_used = 32;
  asm volatile("" : "+l"(f_table), "+r"(f_last), "+r"(f_kvh));  // not to be read again from local memory
  bool f_more = true;
  uint32_t f_at[kPages];   // the pages' places, in pages of one head, for the values that follow the keys
  uint32_t f_there = 0;    // bit i: page i of the step that was fetched last exists
  auto settle = [&]() {
#pragma unroll 1
    while (f_more && f_p >= f_last) {
      f_more = advance(walk_f);
      f_table = s.tables + walk_f.r * s.table_stride;
      f_p = walk_f.first + warp * kPages;
      f_last = walk_f.last;
      f_kvh = walk_f.kvh;
      f_used = 32;
      asm volatile("" : "+l"(f_table), "+r"(f_last), "+r"(f_kvh));
    }
    if (f_more && f_used == 32) {
      const int p = f_p + lane / kPages * (kWarps * kPages) + lane % kPages;
      f_ids = __ldg(f_table + block_of(min(p, f_last - 1)));
      f_used = 0;
    }
  };
  auto fetch_keys = [&]() {
    f_there = 0;
    if (f_more) {
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const uint32_t phys = __shfl_sync(0xffffffffu, f_ids, f_used + i);
        const bool bad = phys >= static_cast<uint32_t>(s.num_blocks);
        const uint32_t h = bad ? 0u : phys * s.hkv + f_kvh;
        f_at[i] = (h - block_of(f_p + i)) * ppb + f_p + i;
        if (bad && f_p + i < f_last) record_device_error(LVB_DEVERR_INDEX);
        if (!bad && f_p + i < f_last) {
          f_there |= 1u << i;
          if (lane >> 1 == i) cp_async_4(scale_ring + lane * 4, scale_lane + h);
          const uint8_t *src = k_lane + static_cast<uint64_t>(f_at[i]) * kSideBytes;
          const uint32_t dst = ring16 + i * (2 * kSideBytes);
          each<2 * kKChunks>([&](auto k) {
            constexpr int kK = decltype(k)::value;
            copy_at<16, kK * 512, kK / kKChunks * 8 * D + kK % kKChunks * 64>(dst, src);
          });
        }
      }
    }
    cp_async_commit();
  };
  auto fetch_values = [&]() {  // of the pages whose keys were fetched, then on to the next step's
#pragma unroll
    for (int i = 0; i < kPages; ++i)
      if (f_there >> i & 1u) {
        const uint8_t *src = v_lane + static_cast<uint64_t>(f_at[i]) * kSideBytes;
        const uint32_t dst = ring_v + i * (2 * kSideBytes);
        each<4>([&](auto r) {
          constexpr int kR = decltype(r)::value;
          copy_at<D / 8, kR * 32 * (D / 8), (kR % 2 + kR / 2 * 8) * D>(dst, src);
        });
      }
    cp_async_commit();
    f_p += kWarps * kPages;
    f_used += kPages;
    settle();
  };
  settle();
  fetch_keys();
  uint32_t there = f_there;  // the present step's
  fetch_values();

  bool more = true;
#pragma unroll 1
  while (more) {
    const Segment seg = walk_m;  // in registers
    if (seg.first >= seg.last) {  // nothing of this item but its beginning
      more = advance(walk_m);
      continue;
    }
    const int row0 = seg.group * kRows, rows = min(seg.rows - row0, kRows);
    // Query rows n = g (B fragments), and rows 2t, 2t + 1 (scores): row i is
    // token i / group, head i % group.
    uint32_t qb[kNT == 1 ? kKSteps : 1][2];
    float f[kNT][2];
    int limit[kNT][2];  // last position that the row sees
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int row = n * 8 + g;
      const bool ok = row < rows;
      const int tok = ok ? (row0 + row) / a.group : 0, head = ok ? row0 + row - tok * a.group : 0;
      const uint16_t *src = a.query + (seg.q0 + tok) * a.query_stride + (seg.kvh * a.group + head) * D + t * 16;
      float x[kKChunks * 16];
#pragma unroll
      for (int c = 0; c < kKChunks; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (ok) v = *reinterpret_cast<const uint4 *>(src + c * 64 + i * 8);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[c * 16 + i * 8 + k] = to_float<kBf16>(reinterpret_cast<const uint16_t *>(&v)[k]);
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
        const uint32_t lo = pack_half(x[4 * k] * up, x[4 * k + 1] * up), hi = pack_half(x[4 * k + 2] * up, x[4 * k + 3] * up);
        if constexpr (kNT == 1) {
          qb[k][0] = lo, qb[k][1] = hi;
        } else if (warp == n) {
          q_sm[(n * kKSteps + k) * 32 + lane] = make_uint2(lo, hi);
        }
      }
    }
    if constexpr (kNT > 1) __syncthreads();
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

    int last = seg.last, mask_from = (seg.computed + 1) / kPage;  // pages from there on are not seen whole by every row
    asm volatile("" : "+r"(last), "+r"(mask_from));               // in registers
#pragma unroll 1
    for (int p = seg.first + warp * kPages; p < last; p += kWarps * kPages) {
      // Scores: positions g and g + 8 by rows 2t and 2t + 1 of each page.
      cp_async_wait_group<1>();
      __syncwarp();  // (the scales are other lanes' copies)
      float sc[kPages][kNT][4], ks[kPages], vs[kPages];
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const uint32_t src = ring16 + i * (2 * kSideBytes);
        uint32_t scales[2], kreg[2][kKChunks][4];
        lds_8<0>(scales, scale_ring + i * 8);
        ks[i] = __uint_as_float(scales[0]), vs[i] = __uint_as_float(scales[1]);
        each<2 * kKChunks>([&](auto k) {
          constexpr int kK = decltype(k)::value;
          lds_16<kK * 512>(kreg[kK / kKChunks][kK % kKChunks], src);
        });
#pragma unroll
        for (int n = 0; n < kNT; ++n) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.f;
#pragma unroll
        for (int k = 0; k < kKSteps; ++k) {
          const uint32_t w0 = P::bias(kreg[0][k >> 2][k & 3]), w1 = P::bias(kreg[1][k >> 2][k & 3]);
          const uint32_t ka[4] = {P::template get<false>(w0), P::template get<false>(w1), P::template get<true>(w0),
                                  P::template get<true>(w1)};
          if constexpr (kNT == 1) {
            mma_16816_nv<false>(sc[i][0], ka, qb[k][0], qb[k][1]);
          } else {
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
              const uint2 b = q_sm[(n * kKSteps + k) * 32 + lane];
              mma_16816_nv<false>(sc[i][n], ka, b.x, b.y);
            }
          }
        }
      }
      const uint32_t now = there;
      __syncwarp();
      fetch_keys();  // the present ones are in registers and used
      there = f_there;
      const bool masked = now != (1u << kPages) - 1 || p + kPages - 1 >= mask_from;
      // Exponents against the present m, plus kHead.
      float y[kPages][kNT][4], lw[kPages], iw[kPages];
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const float vw = (now >> i & 1u) && vs[i] > 0.f ? vs[i] : kZeroWeight;  // (a page that does not exist brings no scales)
        lw[i] = log2_fast(vw);
        iw[i] = rcp_fast(vw);
      }
      auto exponents = [&]() {
        float high = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPages; ++i)
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const float b0 = (lw[i] + kHead) - m[n][0], b1 = (lw[i] + kHead) - m[n][1];
            const float f0 = f[n][0] * ks[i], f1 = f[n][1] * ks[i];
            y[i][n][0] = fmaf(sc[i][n][0], f0, b0), y[i][n][1] = fmaf(sc[i][n][1], f1, b1);
            y[i][n][2] = fmaf(sc[i][n][2], f0, b0), y[i][n][3] = fmaf(sc[i][n][3], f1, b1);
            if (masked) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(now >> i & 1u) || (p + i) * kPage + g + (e >> 1) * 8 > limit[n][e & 1]) y[i][n][e] = -INFINITY;
            }
            high = fmaxf(fmaxf(fmaxf(y[i][n][0], y[i][n][1]), fmaxf(y[i][n][2], y[i][n][3])), high);
          }
        return high;
      };
      if (__any_sync(0xffffffffu, exponents() > kHead + kLazy)) {
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // the scores themselves: y is too coarse beside m = kNone
            float top = m[n][e];
#pragma unroll
            for (int i = 0; i < kPages; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (y[i][n][2 * r + e] != -INFINITY) top = fmaxf(top, fmaf(sc[i][n][2 * r + e], f[n][e] * ks[i], lw[i]));
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
      uint32_t pb[kPages][kNT][2];
#pragma unroll
      for (int i = 0; i < kPages; ++i)
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i][n][e] = exp2_fast(y[i][n][e]);
          l[n][0] = fmaf(y[i][n][0] + y[i][n][2], iw[i], l[n][0]);
          l[n][1] = fmaf(y[i][n][1] + y[i][n][3], iw[i], l[n][1]);
          pb[i][n][0] = movmatrix_trans(pack_half(y[i][n][0], y[i][n][1]));
          pb[i][n][1] = movmatrix_trans(pack_half(y[i][n][2], y[i][n][3]));
        }
      // O: elements (D / 8) g + 2 j (rows g of the tile) and + 1 (rows g + 8).
      cp_async_wait_group<1>();
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const uint32_t src = ring_v + i * (2 * kSideBytes);
        uint32_t vreg[4][kVWords];
        each<4>([&](auto r) {
          constexpr int kR = decltype(r)::value;
          if constexpr (D == 128)
            lds_16<kR * 512>(vreg[kR], src);
          else
            lds_8<kR * 256>(vreg[kR], src);
        });
        if (kFp8 && masked) {
          // Slots past the end may hold NaN patterns: 0 * NaN is not 0.
          const int stop = now >> i & 1u ? seg.computed + seg.rows / a.group : 0;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((p + i) * kPage + 2 * t + (r & 1) + (r >> 1) * 8 >= stop)
#pragma unroll
              for (int w = 0; w < kVWords; ++w) vreg[r][w] = 0;
        }
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
            for (int n = 0; n < kNT; ++n) mma_16816_nv<false>(o[n][2 * w + half], va, pb[i][n][0], pb[i][n][1]);
          }
        }
      }
      fetch_values();
    }

    // The warps' sums, half of the warps at a time.
    const bool whole = seg.first == 0 && seg.last == seg.pages;
    const int piece = 2 * blockIdx.x + (seg.first == 0 ? 1 : 0);
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        const int row = n * 8 + 2 * t + e;
        if (g == 0) m_sm[warp][row] = m[n][e], l_sm[warp][row] = l[n][e];
      }
    auto put = [&]() {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float *dst = o_sm + ((warp % Cfg::kMeet) * kRows + n * 8 + 2 * t + e) * Cfg::kPad + g * (D / 8);
#pragma unroll
          for (int j = 0; j < kDTiles; j += 2)
            *reinterpret_cast<float4 *>(dst + 2 * j) =
                make_float4(o[n][j][e], o[n][j][2 + e], o[n][j + 1][e], o[n][j + 1][2 + e]);
        }
    };
    // A warp adds up rows warp, warp + 8, ..: D / 4 lanes of 4 elements for each (two rows at once for D = 64).
    constexpr int kLanes = D / 4, kSide = 32 / kLanes, kOwn = (kRows + kWarps * kSide - 1) / (kWarps * kSide);
    const int d = lane % kLanes * 4;
    float4 acc[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto take = [&](int from) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int row = (i * kWarps + warp) * kSide + lane / kLanes;
        if (row >= rows) continue;
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_sm[w][row]);
#pragma unroll
        for (int w = 0; w < Cfg::kMeet; ++w) {
          const float wt = exp2_fast(m_sm[from + w][row] - top);
          const float4 v = *reinterpret_cast<const float4 *>(o_sm + (w * kRows + row) * Cfg::kPad + d);
          acc[i].x = fmaf(wt, v.x, acc[i].x), acc[i].y = fmaf(wt, v.y, acc[i].y);
          acc[i].z = fmaf(wt, v.z, acc[i].z), acc[i].w = fmaf(wt, v.w, acc[i].w);
        }
      }
    };
    if (warp < Cfg::kMeet) put();
    __syncthreads();
    take(0);
    __syncthreads();
    if (warp >= Cfg::kMeet) put();
    __syncthreads();
    take(Cfg::kMeet);
    auto store = [&](int row, float4 v, float total_l) {
      const float inv = total_l == 0.f ? 0.f : 1.f / total_l;
      const int tok = (row0 + row) / a.group, head = row0 + row - tok * a.group;
      uint16_t *dst = a.out + (seg.q0 + tok) * a.out_stride + (seg.kvh * a.group + head) * D + d;
      const uint32_t lo = pack2<kBf16>(v.x * inv, v.y * inv), hi = pack2<kBf16>(v.z * inv, v.w * inv);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
    };
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int row = (i * kWarps + warp) * kSide + lane / kLanes;
      if (row >= rows) continue;
      float top = kNone, sum_l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_sm[w][row]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum_l = fmaf(exp2_fast(m_sm[w][row] - top), l_sm[w][row], sum_l);
      if (whole) {
        store(row, acc[i], sum_l);
      } else {
        const int64_t at = static_cast<int64_t>(piece) * kRows + row;
        *reinterpret_cast<float4 *>(a.part_o + at * D + d) = acc[i];
        if (d == 0) a.part_ml[at] = make_float2(top, sum_l);
      }
    }
    if (!whole) {
      // The CTAs that hold a piece of the item.
      const int c0 = static_cast<int>(seg.at / run), c1 = static_cast<int>((seg.at + seg.pages - 1) / run);
      __threadfence();
      __syncthreads();
      if (tid == 0) last_sm = atomicAdd(a.counts + c0, 1u) == static_cast<uint32_t>(c1 - c0);
      __syncthreads();
      if (last_sm) {
        __threadfence();
        if (tid == 0) a.counts[c0] = 0;
#pragma unroll 1
        for (int row = warp * kSide + lane / kLanes; row < rows; row += kWarps * kSide) {
          float top = kNone, sum_l = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          // Pieces in order, a few on their way; the sums move to a larger maximum as it comes.
#pragma unroll 4
          for (int c = c0; c <= c1; ++c) {
            const int64_t at = static_cast<int64_t>(2 * c + (c == c0)) * kRows + row;
            const float2 ml = __ldcg(a.part_ml + at);
            const float4 u = __ldcg(reinterpret_cast<const float4 *>(a.part_o + at * D + d));
            const float grown = fmaxf(top, ml.x);
            const float keep = exp2_fast(top - grown), wt = exp2_fast(ml.x - grown);
            top = grown;
            sum_l = fmaf(wt, ml.y, sum_l * keep);
            v.x = fmaf(wt, u.x, v.x * keep), v.y = fmaf(wt, u.y, v.y * keep);
            v.z = fmaf(wt, u.z, v.z * keep), v.w = fmaf(wt, u.w, v.w * keep);
          }
          store(row, v, sum_l);
        }
      }
    }
    __syncthreads();  // the shared rows are free again
    more = advance(walk_m);
  }
}

}  // namespace kv8
}  // namespace lvb
