// Attention of many query rows over the 8-bit paged cache (prompt chunks, long
// verifications): tcgen05 with fp32 accumulators in tensor memory.
//
// An item is one request, one KV head and up to 256 of its query rows (row R is
// token R / group, head R % group), taken as two tiles A and B of 128 rows that
// share every K/V tile of 128 positions.  Roles of a CTA (one per SM):
//   warps 0..3, 4..7  softmax of tile A, B: one thread for each row
//   warps 8..11       converters: codes from global memory to registers one tile
//                     ahead, to fp16 (exact for both formats), to shared memory
//                     in the 128-byte-swizzled operand layouts (K: K-major, V:
//                     MN-major as it lies), double-buffered
//   warp 12           one thread issues the MMAs: S = Q K^T (both operands in
//                     shared memory), O += P V (P in tensor memory)
// The softmax takes a K/V tile in two halves of 64 positions; P takes the place of
// the first half of its own scores.  While one tile's softmax runs, the tensor core
// works for the other.  (Scores of 64 positions by one MMA, with two in flight,
// were slower: an MMA of N = 64 reads 6 KB of shared memory for 32 cycles of work.)
//
// Mathematics as in the decode kernel: x_j = (q . key code_j) f_b + log2 w_b,
// O = sum 2^(x_j - m) code_j, L = sum 2^(x_j - m) / w_b, out = O / L.  A row's
// maximum of 16 positions of a block is taken over raw scores (f_b >= 0), so the
// scales cost one multiply-add for 16.  Weights enter the second product as
// fp16 times 2^kHead; O is rescaled in tensor memory only when m would grow by
// more than kLazy.
//
// What bounds it: for each 256 x 128 scores 4 x 512 cycles of MMA, 2048 cycles of
// exponentials (16 a cycle and SM), and about 7000 issue slots of 4 a cycle; a step
// takes 5200, since a tile's scores, softmax, weights and product wait for one
// another.  Measured: a chunk of 2048 tokens after 4096 (40/8 heads of 128): 341 us,
// 630 TFLOP/s.
//
// Split.  K/V tiles of all items are laid end to end and cut into one equal run
// for each CTA; items that cross a cut are joined by the last of their CTAs to
// finish, in order (the decode kernel's scheme).
#pragma once

#include "kv8_decode.cuh"

namespace lvb {
namespace kv8 {

constexpr int kTileRows = 256;  // query rows of an item
constexpr int kTilePos = 128;   // positions of a K/V tile
constexpr int kHalfPos = 64;    // that the softmax takes at a time
constexpr int kMinTiles = 2;    // K/V tiles of a CTA, at least

// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16.
__device__ __forceinline__ void umma_f16_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two fp32 values in a register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t join2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}

__device__ __forceinline__ uint64_t dup2(float x) { return join2(__float_as_uint(x), __float_as_uint(x)); }

__device__ __forceinline__ void split2(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 16 codes to fp16.
template <bool kFp8>
__device__ __forceinline__ void codes_to_half(const uint4 &v, uint4 &lo, uint4 &hi) {
  using P = Pair<kFp8>;
  const uint32_t a = P::bias(v.x), b = P::bias(v.y), c = P::bias(v.z), d = P::bias(v.w);
  lo = make_uint4(P::template get<false>(a), P::template get<true>(a), P::template get<false>(b), P::template get<true>(b));
  hi = make_uint4(P::template get<false>(c), P::template get<true>(c), P::template get<false>(d), P::template get<true>(d));
}

template <int D>
struct TileCfg {
  static constexpr int kThreads = 13 * 32;
  static constexpr int kQBytes = 128 * D * 2;        // one tile's queries
  static constexpr int kSideBytes = kTilePos * D * 2;  // K (or V) of a K/V tile
  static constexpr int kHalf = 128 * 128;            // 64 elements of 128 rows
  static constexpr int kKOff = 2 * kQBytes;          // [2 stages]
  static constexpr int kVOff = kKOff + 2 * kSideBytes;
  static constexpr int kScaleOff = kVOff + 2 * kSideBytes;  // float4 [4][8]: key scale, log2 and inverse of the value scale
  static constexpr int kBookOff = kScaleOff + 4 * 8 * 16;
  static constexpr int kSmemBytes = 1024 + kBookOff + 512;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

// One run of K/V tiles of one item.
struct TileSegment {
  int r, kvh, tile;     // rows [256 tile, ..)
  int first, last;      // K/V tiles [first, last)
  int units;            // of the whole item
  int q0, n, computed;  // the request's
  int rows;             // of this item
};

__device__ const uint4 g_zeros = {0, 0, 0, 0};

// mbar_wait with everything after the first probe out of line (polling before it
// took issue slots from the softmax: 549 -> 619 thousand cycles of a prompt chunk).
__device__ __noinline__ bool tile_wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return mbar_wait(bar, parity, abort_flag);
}

__device__ __forceinline__ bool tile_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return mbar_try_wait(bar, parity) || tile_wait_slow(bar, parity, abort_flag);
}

// K/V tiles of the rows [256 i, 256 i + 256) of a request of n tokens.
__device__ __forceinline__ int item_units(int group, int n, int computed, int i) {
  const int tok = (min(n * group, (i + 1) * kTileRows) - 1) / group;
  return (computed + tok + kTilePos) / kTilePos;
}

// K/V tiles of one KV head of request r (0: the decode kernel's, or refused).
// Out of line, like all that runs once a segment: the roles' loops share the
// instruction cache, and with this code inlined in each of them (150 KB in all)
// the MMA issuer waited for its own instructions.
__device__ __noinline__ long long request_units(const Step &s, int group, int few_rows, int r) {
  int q0, n, c;
  long long sum = 0;
  if (request_range(s, r, q0, n, c) && n * group > few_rows) {
    const int tiles = (n * group + kTileRows - 1) / kTileRows;
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) sum += item_units(group, n, c, i);
  }
  return sum;
}

__device__ __noinline__ void describe_segment(const Step &s, int group, int r, int kvh, int tile, int first, long long left,
                                              TileSegment &seg) {
  seg.r = r;
  seg.kvh = kvh;
  seg.tile = tile;
  seg.q0 = s.qsl[r];
  seg.n = s.qsl[r + 1] - seg.q0;
  seg.computed = s.computed[r];
  seg.rows = min(kTileRows, seg.n * group - tile * kTileRows);
  seg.units = item_units(group, seg.n, seg.computed, tile);
  seg.first = first;
  seg.last = left < seg.units - first ? first + static_cast<int>(left) : seg.units;
}

// To the run's next segment, `left` K/V tiles of the run counted from the present
// one's start; false at the end.
__device__ __noinline__ bool advance_segment(const Step &s, int group, int few_rows, long long &left, TileSegment &seg) {
  left -= seg.last - seg.first;
  if (left <= 0) return false;
  int r = seg.r, kvh = seg.kvh, tile = seg.tile + 1;
  if (tile * kTileRows >= seg.n * group) {
    tile = 0;
    if (++kvh == s.hkv) {
      kvh = 0;
      do {
        ++r;
      } while (request_units(s, group, few_rows, r) == 0);  // tiles are left, so a request is
    }
  }
  describe_segment(s, group, r, kvh, tile, 0, left, seg);
  return true;
}

template <bool kBf16, bool kFp8, int D>
__global__ void __launch_bounds__(TileCfg<D>::kThreads, 1) tile_kernel(const __grid_constant__ AttnArgs a) {
  using Cfg = TileCfg<D>;
  constexpr float kNone = -1e30f;
  constexpr float kLeast = 1.2e-38f;  // a factor that leaves -inf what it is, and makes 0 of every score
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float4 *scale_sm = reinterpret_cast<float4 *>(smem + Cfg::kScaleOff);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kBookOff);
  uint64_t *k_full = bars, *v_full = bars + 2, *k_empty = bars + 4, *v_empty = bars + 6, *sc_full = bars + 8,
           *s_full = bars + 12, *p_full = bars + 16, *o_done = bars + 20, *q_full = bars + 24;  // p, o: [tile][half]
  long long *scan = reinterpret_cast<long long *>(bars + 26);  // [13]
  long long *start_units = scan + 13;
  uint32_t *tmem_sm = reinterpret_cast<uint32_t *>(start_units + 1);
  int *start_request = reinterpret_cast<int *>(tmem_sm + 1);
  int *last_sm = start_request + 1;  // [2]
  volatile int *abort_flag = last_sm + 2;

  pdl_wait();
  const Step &s = a.step;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  auto block_scan = [&](long long v, long long &sum) {
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    long long before = 0;
    sum = 0;
#pragma unroll 1
    for (int w = 0; w < 13; ++w) {
      if (w < warp) before += scan[w];
      sum += scan[w];
    }
    return before + x - v;
  };
  long long total = 0, mine = 0, sum = 0, ex = 0;
  for (int base = 0; base < s.num_seqs; base += Cfg::kThreads) {
    mine = base + tid < s.num_seqs ? request_units(s, a.group, a.few_rows, base + tid) : 0;
    ex = block_scan(mine, sum);
    total += sum * s.hkv;
  }
  long long run = (total + gridDim.x - 1) / gridDim.x;
  if (run < kMinTiles) run = kMinTiles;
  const long long begin = run * blockIdx.x;
  if (begin >= total) return;
  const long long end = begin + run < total ? begin + run : total;
  {
    long long before = 0;
    for (int base = 0; base < s.num_seqs; base += Cfg::kThreads) {
      if (s.num_seqs > Cfg::kThreads) {
        mine = base + tid < s.num_seqs ? request_units(s, a.group, a.few_rows, base + tid) : 0;
        ex = block_scan(mine, sum);
      }
      const long long lo = before + ex * s.hkv, hi = lo + mine * s.hkv;
      if (lo <= begin && begin < hi) {
        *start_request = base + tid;
        *start_units = lo;
      }
      before += sum * s.hkv;
    }
  }
  if (warp == 0) {
    tmem_alloc(tmem_sm, 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 4);
      mbar_init(v_full + i, 4);
      mbar_init(k_empty + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(q_full + i, 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(sc_full + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(o_done + i, 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_sm;

  TileSegment seg;
  long long left = end - begin;  // K/V tiles of the run from the present segment on
  {
    const int r = *start_request;
    const long long per_head = request_units(s, a.group, a.few_rows, r);
    long long inside = begin - *start_units;
    const int kvh = static_cast<int>(inside / per_head);
    inside -= kvh * per_head;
    const int c = s.computed[r], n = s.qsl[r + 1] - s.qsl[r];
    int tile = 0;
#pragma unroll 1
    while (inside >= item_units(a.group, n, c, tile)) inside -= item_units(a.group, n, c, tile++);
    describe_segment(s, a.group, r, kvh, tile, static_cast<int>(inside), left, seg);
  }
  auto advance = [&]() { return advance_segment(s, a.group, a.few_rows, left, seg); };

  TileSegment joins[2];  // pieces of items that other CTAs hold pieces of
  long long join_item[2];
  int num_joins = 0;
  bool ok = true, more = true;

  if (warp >= 8 && warp < 12) {
    // ---------------- converters ----------------
    // Lanes are laid out so that eight neighbours store to all banks: four
    // pieces of one 64-element half for two rows.
    constexpr int kChunks = D / 16;            // 16-byte pieces of a row
    constexpr int kRowsPass = 128 / kChunks;   // rows that the 128 threads take at a time
    constexpr int kPasses = kTilePos / kRowsPass;
    const int ct = tid - 256;
    const int c = D == 128 ? (ct & 3) + (ct >> 1 & 4) : ct & 3;
    const int row0 = D == 128 ? (ct >> 2 & 1) + (ct >> 4) * 2 : ct >> 2;
    const int ppb = s.bs / kPage;
    uint32_t page_at = 0;  // lane i < 8: page i's place, in pages of one head
    uint4 kreg[kPasses], vreg[kPasses];
    float ksc = 0.f, vsc = 1.f;
    // Where a tile's pages are.
    auto locate = [&](const TileSegment &of, int tile) {
      const int p = tile * (kTilePos / kPage) + (lane & 7);
      const int pages = (of.computed + of.n + kPage - 1) / kPage;
      int phys = p < pages ? s.tables[of.r * s.table_stride + p / ppb] : -1;
      const bool there = static_cast<uint32_t>(phys) < static_cast<uint32_t>(s.num_blocks);
      if (p < pages && !there) record_device_error(LVB_DEVERR_INDEX);
      const uint32_t h = there ? static_cast<uint32_t>(phys) * s.hkv + of.kvh : 0u;
      page_at = there ? h * ppb + p % ppb : ~0u;
      ksc = vsc = -1.f;  // no such page
      if (there) ksc = __ldg(a.key_scales + h), vsc = __ldg(a.value_scales + h);
    };
    const uint8_t *k_lane = a.key_codes + (row0 % kPage) * D + c * 16, *v_lane = a.value_codes + (row0 % kPage) * D + c * 16;
    auto load = [&](int stop, const uint8_t *lane_base, uint4 (&reg)[kPasses]) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int row = i * kRowsPass + row0;
        const uint32_t at = __shfl_sync(0xffffffffu, page_at, row / kPage);
        const uint8_t *src = lane_base + static_cast<uint64_t>(at) * (kPage * D);
        // zeros past the end: 0 times what a stale slot holds may be NaN
        if (row >= stop || at == ~0u) src = reinterpret_cast<const uint8_t *>(&g_zeros);
        reg[i] = __ldg(reinterpret_cast<const uint4 *>(src));
      }
    };
    // Registers to a stage's operand rows.
    uint8_t *const piece_lo = smem + (c >> 2) * Cfg::kHalf + row0 * 128 + ((((2 * c) & 7) ^ (row0 & 7)) << 4);
    uint8_t *const piece_hi = smem + (c >> 2) * Cfg::kHalf + row0 * 128 + ((((2 * c + 1) & 7) ^ (row0 & 7)) << 4);
    auto convert = [&](int at, const uint4 (&reg)[kPasses]) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        uint4 lo, hi;
        codes_to_half<kFp8>(reg[i], lo, hi);
        *reinterpret_cast<uint4 *>(piece_lo + at + i * (kRowsPass * 128)) = lo;
        *reinterpret_cast<uint4 *>(piece_hi + at + i * (kRowsPass * 128)) = hi;
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    // Tile g goes to shared memory while the next one's codes come.
    int g = 0;
    bool have = false;
    TileSegment now = seg;  // in registers: seg itself lives in local memory
    int t = now.first;
#pragma unroll 1
    while (have || more) {
      const int st = g & 1, stop = now.computed + now.n - t * kTilePos;
      if (have) {
        if (warp == 8) {
          if (lane < 8) {
            const float vw = vsc > 0.f ? vsc : kZeroWeight;
            // a page that does not exist weighs nothing
            scale_sm[(g & 3) * 8 + lane] =
                ksc < 0.f ? make_float4(1.f, -INFINITY, 0.f, 0.f) : make_float4(ksc, log2_fast(vw), rcp_fast(vw), 0.f);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sc_full + (g & 3));
        }
        if (g >= 2) ok = ok && tile_wait(k_empty + st, ((g >> 1) - 1) & 1, abort_flag);
        convert(Cfg::kKOff + st * Cfg::kSideBytes, kreg);
        if (lane == 0) mbar_arrive(k_full + st);
      }
      if (more) {
        locate(now, t);
        load(stop, k_lane, kreg);
      }
      if (have) {
        if (g >= 2) ok = ok && tile_wait(v_empty + st, ((g >> 1) - 1) & 1, abort_flag);
        convert(Cfg::kVOff + st * Cfg::kSideBytes, vreg);
        if (lane == 0) mbar_arrive(v_full + st);
        ++g;
      }
      have = more;
      if (more) {
        load(stop, v_lane, vreg);
        if (++t == now.last) {
          more = advance();
          now = seg;
          t = now.first;
        }
      }
    }
  } else if (warp == 12) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      constexpr uint32_t kIdescS = umma_idesc_f16(128, kTilePos, 0, 0, 0, 0);
      constexpr uint32_t kIdescO = umma_idesc_f16(128, D, 0, 0, 0, 1);
      constexpr int kKSteps = D / 16;
      const uint32_t base = smem_u32(smem);
      int g = 0;
      uint32_t q_phase = 0, tile_phase = 0;  // bit x: tile x's
      while (more && ok) {
        // (what the loops use is in registers: a local-memory access here waits on the codes' stream)
        const int tiles = seg.rows > 128 ? 2 : 1;
        const int count = seg.last - seg.first;
        auto scores = [&](int x, int st) {
          const uint64_t q_desc = umma_smem_desc_sw128(base + x * Cfg::kQBytes, 16, 1024);
          const uint64_t k_desc = umma_smem_desc_sw128(base + Cfg::kKOff + st * Cfg::kSideBytes, 16, 1024);
#pragma unroll
          for (int k = 0; k < kKSteps; ++k) {
            const uint64_t off = (k >> 2) * (Cfg::kHalf >> 4) + (k & 3) * 2;
            umma_f16(tmem + x * 128, q_desc + off, k_desc + off, kIdescS, k > 0);
          }
          umma_commit(s_full + x);
        };
#pragma unroll 1
        for (int x = 0; x < tiles && ok; ++x) ok = tile_wait(q_full + x, q_phase >> x & 1, abort_flag);
        q_phase ^= tiles == 2 ? 3u : 1u;
        ok = ok && tile_wait(k_full + (g & 1), (g >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int x = 0; x < tiles; ++x) scores(x, g & 1);
        umma_commit(k_empty + (g & 1));
#pragma unroll 1
        for (int t = 0; t < count && ok; ++t, ++g) {
          const int st = g & 1;
          const bool next = t + 1 < count;
          ok = tile_wait(v_full + st, (g >> 1) & 1, abort_flag);
          if (next) ok = ok && tile_wait(k_full + (st ^ 1), ((g + 1) >> 1) & 1, abort_flag);
#pragma unroll 1
          for (int x = 0; x < tiles && ok; ++x) {
#pragma unroll 1
            for (int half = 0; half < 2 && ok; ++half) {
              ok = tile_wait(p_full + 2 * x + half, tile_phase >> x & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              const uint64_t v_desc = umma_smem_desc_sw128(
                  base + Cfg::kVOff + st * Cfg::kSideBytes + half * (kHalfPos * 128), Cfg::kHalf, 1024);
#pragma unroll
              for (int k = 0; k < kHalfPos / 16; ++k)
                umma_f16_tmem_a(tmem + 256 + x * 128, tmem + x * 128 + half * kHalfPos + k * 8, v_desc + k * 128, kIdescO,
                                t > 0 || half > 0 || k > 0);
              umma_commit(o_done + 2 * x + half);
            }
            tile_phase ^= 1u << x;
            if (ok && next) scores(x, st ^ 1);
          }
          if (!ok) break;
          umma_commit(v_empty + st);
          if (next) umma_commit(k_empty + (st ^ 1));
        }
        more = advance();
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax ----------------
    const int x = warp >> 2;           // tile A or B
    const int row_in = tid & 127;      // row of the tile = tensor memory lane
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t t_s = tmem + lanes + x * 128, t_o = tmem + lanes + 256 + x * 128;
    // 16-byte piece of a row of 128 in an operand's layout; a warp's rows are its own.
    auto place = [](int row, int piece) { return (piece >> 3) * Cfg::kHalf + row * 128 + (((piece & 7) ^ (row & 7)) << 4); };
    int g = 0, phase = 0;  // K/V tiles of the CTA, and of this tile
    while (more) {
      const TileSegment now = seg;  // in registers: seg itself lives in local memory
      const int rows = now.rows - x * 128;
      if (rows > 0) {
        // The warp's queries, D / 8 lanes for a row, brought to fp16 by a power of
        // two where they are bf16.  This lane's own row is row_in.
        const int first_row = now.tile * kTileRows + x * 128;
        const bool some = row_in < rows;
        const int tok = some ? (first_row + row_in) / a.group : 0, head = some ? first_row + row_in - tok * a.group : 0;
        const uint32_t src_row = (now.q0 + tok), src_head = now.kvh * a.group + head;
        float fr = 0.f;
        {
          constexpr int kLanes = D / 8, kRows = 32 / kLanes;
          const int piece = lane % kLanes;
          uint4 raw[32 / kRows];
#pragma unroll
          for (int i = 0; i < 32; i += kRows) {
            const int from = i + lane / kLanes, in = (warp & 3) * 32 + from;  // row of the warp, of the tile
            const uint32_t r_tok = __shfl_sync(0xffffffffu, src_row, from), r_head = __shfl_sync(0xffffffffu, src_head, from);
            raw[i / kRows] = make_uint4(0, 0, 0, 0);
            if (in < rows) raw[i / kRows] = *reinterpret_cast<const uint4 *>(a.query + r_tok * a.query_stride + r_head * D + piece * 8);
          }
#pragma unroll
          for (int i = 0; i < 32; i += kRows) {
            const int in = (warp & 3) * 32 + i + lane / kLanes;
            float e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = to_float<kBf16>(reinterpret_cast<const uint16_t *>(&raw[i / kRows])[k]);
            float up = a.scale_log2 < 0.f ? -1.f : 1.f;
            if constexpr (kBf16) {
              float top = 0.f;
#pragma unroll
              for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(e[k]));
#pragma unroll
              for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              up *= scale_to(top, 7);
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
              const float u = __shfl_sync(0xffffffffu, up, k * kLanes);
              if (lane == i + k) fr = a.scale_log2 / u;
            }
            *reinterpret_cast<uint4 *>(smem + x * Cfg::kQBytes + place(in, piece)) =
                make_uint4(pack2<false>(e[0] * up, e[1] * up), pack2<false>(e[2] * up, e[3] * up),
                           pack2<false>(e[4] * up, e[5] * up), pack2<false>(e[6] * up, e[7] * up));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full + x);

        const int limit = some ? now.computed + tok : -1;  // last position that the row sees
        const bool idle = (warp & 3) * 32 >= rows;  // none of the warp's rows exists
        float m = kNone, l = 0.f;
        for (int t = now.first; t < now.last; ++t, ++g, ++phase) {
          ok = ok && tile_wait(sc_full + (g & 3), (g >> 2) & 1, abort_flag);
          ok = ok && tile_wait(s_full + x, phase & 1, abort_flag);
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            if (idle) {
              if (lane == 0) mbar_arrive(p_full + 2 * x + half);
              continue;
            }
            tc_fence_after();
            const uint32_t t_half = t_s + half * kHalfPos;
            uint32_t v[2][32];
            tmem_ld_x32(t_half, v[0]);
            tmem_ld_x32(t_half + 32, v[1]);
            const float4 *scales = scale_sm + (g & 3) * 8 + half * 4;
            const int seen = limit - t * kTilePos - half * kHalfPos;  // positions 0 .. seen of the half are visible
            const bool masked = __any_sync(0xffffffffu, seen < kHalfPos - 1);
            tmem_wait_ld();
            if (masked) {
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (c * 32 + i > seen) v[c][i] = 0xff800000u;  // -inf
            }
            float top = kNone;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              auto s_at = [&](int i) { return __uint_as_float(v[h >> 1][(h & 1) * 16 + i]); };
              float mx = max3(s_at(0), s_at(1), s_at(2)), my = max3(s_at(3), s_at(4), s_at(5));
#pragma unroll
              for (int i = 6; i < 14; i += 4) {
                mx = max3(mx, s_at(i), s_at(i + 1));
                my = max3(my, s_at(i + 2), s_at(i + 3));
              }
              mx = fmaxf(max3(mx, s_at(14), s_at(15)), my);
              const float4 sc = scales[h];
              top = fmaxf(top, fmaf(mx, fmaxf(fr * sc.x, kLeast), sc.y));
            }
            // O is rescaled when the maximum grows by more than kLazy.
            if (__any_sync(0xffffffffu, top > m + kLazy)) {
              const float grown = fmaxf(m, top);
              const float alpha = exp2_fast(m - grown);
              m = grown;
              l *= alpha;
              if (t > now.first || half > 0) {
                // the product before is done
                ok = ok && tile_wait(o_done + 2 * x + (half ^ 1), (phase + half + 1) & 1, abort_flag);
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                  uint32_t w[16];
                  tmem_ld_x16(t_o + c * 16, w);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * alpha);
                  tmem_st_x16(t_o + c * 16, w);
                }
              }
            }
            const float base = m - kHead;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t pk[16];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float4 sc = scales[c * 2 + h];
                const uint64_t fk = dup2(fmaxf(fr * sc.x, kLeast)), add = dup2(sc.y - base);
                uint64_t part = 0;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  float e0, e1;
                  split2(fma2(join2(v[c][h * 16 + i], v[c][h * 16 + i + 1]), fk, add), e0, e1);
                  e0 = exp2_fast(e0);
                  e1 = exp2_fast(e1);
                  part = add2(part, join2(__float_as_uint(e0), __float_as_uint(e1)));
                  pk[h * 8 + i / 2] = pack2<false>(e0, e1);
                }
                float p0, p1;
                split2(part, p0, p1);
                l = fmaf(p0 + p1, sc.z, l);
              }
              tmem_st_x16(t_half + c * 16, pk);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 2 * x + half);
          }
        }
        // The item's (or piece's) result.
        ok = ok && tile_wait(o_done + 2 * x + 1, (phase + 1) & 1, abort_flag);
        tc_fence_after();
        const bool whole = now.first == 0 && now.last == now.units;
        const int64_t piece = (2 * blockIdx.x + (now.first == 0 ? 1 : 0)) * static_cast<int64_t>(kTileRows) + x * 128 + row_in;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (!idle) {
          // Whole rows go through the queries' place in shared memory, so that stores cover lines.
          uint8_t *rows_sm = smem + x * Cfg::kQBytes;
          constexpr int kPieces = D / 8;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t w[32];
            tmem_ld_x32(t_o + c * 32, w);
            tmem_wait_ld();
            if (whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                const int at = c * 4 + i / 8;
                *reinterpret_cast<uint4 *>(rows_sm + place(row_in, at)) = make_uint4(
                    pack2<kBf16>(__uint_as_float(w[i]) * inv, __uint_as_float(w[i + 1]) * inv),
                    pack2<kBf16>(__uint_as_float(w[i + 2]) * inv, __uint_as_float(w[i + 3]) * inv),
                    pack2<kBf16>(__uint_as_float(w[i + 4]) * inv, __uint_as_float(w[i + 5]) * inv),
                    pack2<kBf16>(__uint_as_float(w[i + 6]) * inv, __uint_as_float(w[i + 7]) * inv));
              }
            } else if (some && ok) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4 *>(a.tile_o + piece * D + c * 32 + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            }
          }
          __syncwarp();
          if (whole && ok) {
#pragma unroll 4
            for (int i = lane; i < 32 * kPieces; i += 32) {
              const int from = i / kPieces, at = i % kPieces, in = (warp & 3) * 32 + from;
              const uint32_t r_tok = __shfl_sync(0xffffffffu, src_row, from), r_head = __shfl_sync(0xffffffffu, src_head, from);
              if (in >= rows) continue;
              const uint4 v = *reinterpret_cast<const uint4 *>(rows_sm + place(in, at));
              *reinterpret_cast<uint4 *>(a.out + r_tok * a.out_stride + r_head * D + at * 8) = v;
            }
          }
          __syncwarp();
        }
        if (!whole) a.tile_ml[piece] = make_float2(m, some ? l : 0.f);
        tc_fence_before();
      } else {
        g += now.last - now.first;
      }
      if (!(now.first == 0 && now.last == now.units)) {
        joins[num_joins] = now;
        join_item[num_joins++] = end - left - now.first;
      }
      more = advance();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
  if (tid >= 256) return;

  // Items that other CTAs hold pieces of: whoever finishes an item last adds its pieces up, in order.
  __threadfence();
  named_barrier_256();
  for (int i = 0; i < num_joins; ++i) {
    const TileSegment &j = joins[i];
    const int c0 = static_cast<int>(join_item[i] / run), c1 = static_cast<int>((join_item[i] + j.units - 1) / run);
    if (tid == 0) last_sm[i] = atomicAdd(a.tile_counts + c0, 1u) == static_cast<uint32_t>(c1 - c0);
  }
  named_barrier_256();
  __threadfence();
#pragma unroll 1
  for (int i = 0; i < num_joins; ++i) {
    if (!last_sm[i]) continue;
    const TileSegment &j = joins[i];
    const int c0 = static_cast<int>(join_item[i] / run), c1 = static_cast<int>((join_item[i] + j.units - 1) / run);
    if (tid == 0) a.tile_counts[c0] = 0;
    // A warp takes kBatch of the item's rows at a time, D / 4 lanes for each.
    constexpr int kLanes = D / 4, kSide = 32 / kLanes, kBatch = 4;
    const int d = lane % kLanes * 4;
#pragma unroll 1
    for (int base = warp * (kBatch * kSide); base < j.rows; base += 8 * kBatch * kSide) {
      float top[kBatch], sum_l[kBatch];
      float4 acc[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        top[i] = kNone;
        sum_l[i] = 0.f;
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      // Pieces in order, two at a time on their way; sums move to a larger maximum as it comes.
#pragma unroll 2
      for (int c = c0; c <= c1; ++c) {
        const int64_t at = static_cast<int64_t>(2 * c + (c == c0)) * kTileRows + base + lane / kLanes;
        float2 ml[kBatch];
        float4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          ml[i] = __ldcg(a.tile_ml + at + i * kSide);
          v[i] = __ldcg(reinterpret_cast<const float4 *>(a.tile_o + (at + i * kSide) * D + d));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (base + i * kSide + lane / kLanes >= j.rows) ml[i] = make_float2(kNone, 0.f), v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          const float grown = fmaxf(top[i], ml[i].x);
          const float keep = exp2_fast(top[i] - grown), wt = exp2_fast(ml[i].x - grown);
          top[i] = grown;
          sum_l[i] = fmaf(wt, ml[i].y, sum_l[i] * keep);
          acc[i].x = fmaf(wt, v[i].x, acc[i].x * keep), acc[i].y = fmaf(wt, v[i].y, acc[i].y * keep);
          acc[i].z = fmaf(wt, v[i].z, acc[i].z * keep), acc[i].w = fmaf(wt, v[i].w, acc[i].w * keep);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int row = base + i * kSide + lane / kLanes;
        if (row >= j.rows) continue;
        const float inv = sum_l[i] == 0.f ? 0.f : 1.f / sum_l[i];
        const int abs_row = j.tile * kTileRows + row;
        const int tok = abs_row / a.group, head = abs_row - tok * a.group;
        uint16_t *dst = a.out + (j.q0 + tok) * a.out_stride + (j.kvh * a.group + head) * D + d;
        const uint32_t lo = pack2<kBf16>(acc[i].x * inv, acc[i].y * inv), hi = pack2<kBf16>(acc[i].z * inv, acc[i].w * inv);
        *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
      }
    }
  }
}

}  // namespace kv8
}  // namespace lvb
