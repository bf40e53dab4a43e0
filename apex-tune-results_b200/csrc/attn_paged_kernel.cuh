// Attention over a paged 8-bit K/V cache (the layout kv_cache_kernels.cuh writes) for sm_100a.
//
// For query rows q_i of one K/V head (the heads of its group and a request's new tokens
// together) and cached tokens j with codes k_j, v_j and block scales a_j, b_j:
//   x_ij = sm_scale * log2(e) * a_j * (q_i . k_j)          (base-2 scores)
//   o_i  = sum_j 2^x_ij b_j v_j / sum_j 2^x_ij
//
// The codes never leave 8 bits: both products run on tcgen05.mma kind::f8f6f4 with the cache
// tiles as the TMA wrote them to shared memory, so nothing converts the cache. What is not
// e4m3 is split into e4m3 terms that add up to it, two for bf16 calls and three for fp16 ones:
//   * q, scaled per row by a power of two so that its largest magnitude lies in (224, 448]: its
//     8 or 11 significant bits in pieces of 4, exact but for values below 2^-9 of that range;
//   * the weight p'_ij = 2^(x_ij + log2 b_j - m_i) (the V scale goes into the exponent, one
//     addition per token), rounded to fp16: off by 2^-8 (two terms) or 2^-12 of itself, or by
//     2^-10 absolutely. With two terms an fp16 output was 3.3 times as far from its float64
//     value as rounding alone puts it; a bf16 output's own rounding hides the difference.
// fp32 accumulation of e4m3 products on this card is exact to 2^-23 of the magnitudes.
//
// Tokens, not query rows, are the M side: S^T = K Q^T and O^T = V^T P, M = 128 tokens resp. 128
// columns of the head dim, N = 16 .. 128 query rows. A decode step has 1 to 16 query rows per
// K/V head; as the M side they would leave most of a 128-row tile empty. Thread t owns token t of a
// tile: its scales are per-thread scalars and its row of P is 16 contiguous bytes per 16 query
// rows. The price is that a row's maximum runs across threads; so the running maximum is only
// moved when some p' would pass 2^8.75 (one vote per tile, folded into a barrier that the
// tile needs anyway), which is rare after a row's first tile.
//
// m_i tracks the maximum of x_ij + log2 b_j, kept 2^6 below p's top so that small weights stay
// above e4m3's floor: the largest weight of a row is held at 2^6 .. 2^8.75 (e4m3's largest is 448).
// The row sum sum_j 2^(x_ij - m_i) = sum_j p'_ij / b_j is taken from the fp32 p'.
//
// Work: an item is (request, K/V head, query-row tile); its tiles of 128 tokens line up with all
// other items' in one sequence, which is cut into equal ranges, one per CTA, whatever the
// lengths. A CTA writes what it has of an item that it shares to the workspace (normalised
// rows and their base-2 logsumexp) and attn_paged_combine_kernel joins them in a fixed order.
// Lengths are read on the device only.
//
// Warps: 4 or 8 softmax (32 token rows of TMEM each), then TMA producer, MMA issuer, scales.
#pragma once

#include "attn_fwd_kernel.cuh"
#include "kv_cache_kernels.cuh"

namespace apex {

constexpr int kPagedTile = 128;      // cached tokens per tile
constexpr float kPagedTop = 6.0f;    // log2 of the weight that a row's maximum maps to
constexpr float kPagedMost = 8.75f;  // a weight above 2^this moves the maximum (448 = 2^8.807)
constexpr float kPagedUnset = -1e30f;
// V scales below 2^-100 (0 among them) count as 2^-100, so that 1 / b stays in range.
constexpr float kPagedLeastScale = 7.888609052210118e-31f;

struct PagedParams {
  const void* q;  // [total_q, H, D]
  void* o;
  float* lse;  // nullable, [H, total_q]
  const float* k_scale;  // [num_blocks, H_kv]
  const float* v_scale;
  const int* block_table;  // [batch, table_width], row stride table_stride
  const int* seq_lens;     // [batch] tokens in the cache
  const int* cu_seqlens_q; // [batch + 1]; null: total_q / batch query tokens each
  float* part_o;    // [2 * CTAs][NQ][D], see PagedShare
  float* part_lse;  // [2 * CTAs][NQ]
  int* share;       // [2 * CTAs][kShareInts]
  int* status;
  int* host_flag;
  unsigned long long timeout_ns;
  long long table_stride;
  long long q_st, q_sh, o_st, o_sh;  // token, head strides (elements)
  int batch, heads_kv, group, total_q, max_q;
  int num_blocks, block_shift, table_width;
  int causal, window, zero_rest;
  int stream_once;   // the cache is read once per call: do not keep it in L2
  float scale_log2;  // sm_scale * log2(e)
};

// One entry per CTA for the item that reaches it from the CTA before (2c) and for the one
// that it leaves to the next (2c + 1): batch, head, query tile, first and last CTA; batch -1:
// none.
constexpr int kShareInts = 8;

template <typename T, int D, int NQ>
struct PagedCfg {
  static_assert(D == 64 || D == 128 || D == 256, "head dims 64, 128, 256");
  static constexpr int kRow = D < 128 ? D : 128;         // bytes of a token row in a column chunk
  static constexpr int kChunks = (D + 127) / 128;
  static constexpr uint32_t kSwizzle = kRow == 128 ? 2 : 4;
  static constexpr int kTerms = std::is_same<T, __half>::value ? 3 : 2;  // of q
  static constexpr int kWG = NQ >= 64 ? 2 : 1;           // softmax warpgroups, NC query rows each
  static constexpr int kNC = NQ / kWG;
  static constexpr int kSoftWarps = 4 * kWG;
  static constexpr int kThreads = 128 * kWG + 96;
  // Two CTAs per SM cover each other's latencies where their shared memory fits.
  static constexpr int kCtas = (D <= 128 && NQ <= 32) ? 2 : 1;
  static constexpr int kSlotBytes = kPagedTile * D;      // one K or V tile
  static constexpr int kPBufs = 2;
  static constexpr int kQBytes = kTerms * NQ * D;
  static constexpr int kPTerm = kPagedTile * NQ;         // one term of one P buffer
  static constexpr int kBudget = kCtas == 2 ? 115712 : 232448;
  static constexpr int kMiscBytes = 1280 + NQ * 40;      // what the plan below adds
  static constexpr int kNSMax = (kBudget - kQBytes - kPBufs * kTerms * kPTerm - kMiscBytes) / kSlotBytes;
  static constexpr int kNS = kNSMax > 12 ? 12 : kNSMax;  // ring slots
  static_assert(kNS >= 3, "the ring needs K(j + 1) beside K(j) and V(j)");
  static constexpr int kScaleRing = 4;
  // TMEM: S buffers at 0 and NQ, O (one block of NQ columns per 128 of the head dim) from 2 NQ.
  static constexpr int kTmemCols = (2 + kChunks) * NQ <= 64 ? 64
                                   : ((2 + kChunks) * NQ <= 128 ? 128 : ((2 + kChunks) * NQ <= 256 ? 256 : 512));
  static_assert((2 + kChunks) * NQ <= 512 && kCtas * kTmemCols <= 512, "TMEM plan");
  // shared-memory plan
  static constexpr int kQ = kNS * kSlotBytes;
  static constexpr int kP = kQ + kQBytes;
  static constexpr int kBars = kP + kPBufs * kTerms * kPTerm;
  static constexpr int kKvFull = 0, kKvEmpty = kNS, kQFull = 2 * kNS, kSFull = kQFull + 1, kSFree = kSFull + 2,
                       kPFull = kSFree + 2, kPvDone = kPFull + 2, kScFull = kPvDone + 2,
                       kScEmpty = kScFull + kScaleRing, kDrain = kScEmpty + kScaleRing, kNumBars = kDrain + 1;
  static constexpr int kScales = (kBars + kNumBars * 8 + 15) / 16 * 16;  // float4 [kScaleRing][8 pages]
  static constexpr int kCol = kScales + kScaleRing * 8 * 16;  // per query row: m, q scale, factor, hi, lo
  static constexpr int kRed = kCol + 5 * NQ * 4;              // [kWG][4 warps][kNC]
  static constexpr int kScan = (kRed + 4 * NQ * 4 + 15) / 16 * 16;       // long long [32], start of the CTA's range
  static constexpr int kMisc = kScan + 32 * 8 + 32;
  static constexpr int kBytes = kMisc + 16;
  static_assert(kBytes <= kBudget, "shared-memory plan");
};

// The query rows of request b and where they stand.
struct PagedRequest {
  int q0, nq, len;  // first row, rows, cached tokens
};

__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int b) {
  PagedRequest r;
  if (p.cu_seqlens_q != nullptr) {
    r.q0 = min(max(__ldg(p.cu_seqlens_q + b), 0), p.total_q);
    r.nq = min(max(__ldg(p.cu_seqlens_q + b + 1), r.q0), p.total_q) - r.q0;
    r.nq = min(r.nq, p.max_q);
  } else {
    r.nq = p.max_q;
    r.q0 = b * r.nq;
  }
  r.len = min(max(__ldg(p.seq_lens + b), 0), p.table_width << p.block_shift);
  return r;
}

// Tokens [lo, hi) are what the rows of query tile qt see together; [t0, t0 + n) are their tiles.
struct PagedSpan {
  int lo, hi, t0, n;
};

template <int NQ>
__device__ __forceinline__ PagedSpan paged_span(const PagedParams& p, const PagedRequest& r, int qt) {
  const int i0 = qt * NQ / p.group;
  const int i1 = (min(r.nq * p.group, (qt + 1) * NQ) - 1) / p.group;
  const int first = r.len - r.nq + i0, last = r.len - r.nq + i1;  // positions
  PagedSpan s;
  s.hi = p.causal ? min(r.len, last + 1) : r.len;
  s.lo = p.window >= 0 ? max(0, first - p.window) : 0;
  s.t0 = s.lo / kPagedTile;
  s.n = s.hi > s.lo ? (s.hi + kPagedTile - 1) / kPagedTile - s.t0 : 0;
  return s;
}

template <int NQ>
__device__ __forceinline__ int paged_qtiles(const PagedParams& p, const PagedRequest& r) {
  return (r.nq * p.group + NQ - 1) / NQ;
}

// Units of one K/V head of a request: its items' tiles, at least one each (an item that sees
// nothing still has rows to write).
template <int NQ>
__device__ __forceinline__ int paged_head_units(const PagedParams& p, const PagedRequest& r) {
  const int qts = paged_qtiles<NQ>(p, r);
  int units = 0;
  for (int qt = 0; qt < qts; ++qt) units += max(1, paged_span<NQ>(p, r, qt).n);
  return units;
}

// A CTA's part of an item.
struct PagedSegment {
  int b, h, qt;
  PagedRequest r;
  PagedSpan span;
  int tile, n;        // tiles [tile, tile + n) of the cache
  int slot;           // -1: the whole item; else its entry of the workspace
  int c0, c1;         // CTAs that share the item
};

// Where every role walks from: the CTA's range of units and the item that it begins in.
struct PagedStart {
  long long unit, end;     // the CTA's range
  long long total;         // units of the whole call
  long long request_unit;  // first unit of request b
  int b, ctas;
};

template <int NQ>
struct PagedWalk {
  const PagedParams& p;
  long long unit, end, total;
  int ctas;
  int b, h, qt, qts;
  long long item;  // first unit of the item (b, h, qt)
  PagedRequest r;

  __device__ __forceinline__ PagedWalk(const PagedParams& params, const PagedStart& s)
      : p(params), unit(s.unit), end(s.end), total(s.total), ctas(s.ctas), b(s.b), h(0), qt(0), qts(0),
        item(s.request_unit) {
    if (unit >= end) return;
    r = paged_request(p, b);
    qts = paged_qtiles<NQ>(p, r);
    const int per_head = paged_head_units<NQ>(p, r);
    h = (int)((unit - item) / per_head);
    item += (long long)h * per_head;
    while (true) {
      const int n = max(1, paged_span<NQ>(p, r, qt).n);
      if (item + n > unit) break;
      item += n;
      ++qt;
    }
  }

  __device__ __forceinline__ bool next(PagedSegment& s) {
    if (unit >= end) return false;
    while (qt == qts) {  // on to the next head or request that has query rows
      qt = 0;
      if (++h == p.heads_kv || qts == 0) {
        h = 0;
        ++b;
        r = paged_request(p, b);
        qts = paged_qtiles<NQ>(p, r);
      }
    }
    s.b = b;
    s.h = h;
    s.qt = qt;
    s.r = r;
    s.span = paged_span<NQ>(p, r, qt);
    const int n = max(1, s.span.n);
    const int skip = (int)(unit - item);
    const int take = (int)min((long long)(n - skip), end - unit);
    s.tile = s.span.t0 + skip;
    s.n = s.span.n == 0 ? 0 : take;
    s.slot = -1;
    if (take < n) {
      s.slot = 2 * blockIdx.x + (skip > 0 ? 0 : 1);
      // CTA c has the units [c * total / ctas, (c + 1) * total / ctas).
      s.c0 = (int)(((item + 1) * ctas - 1) / total);
      s.c1 = (int)(((item + n) * ctas - 1) / total);
    }
    unit += take;
    item += n;
    ++qt;
    return true;
  }
};

// The CTA's range, and the request that it begins in. All threads call it.
template <int NQ>
__device__ __forceinline__ PagedStart paged_start(const PagedParams& p, long long* scan, int* found) {
  // Each thread sums a run of requests; the one whose run holds the first unit looks closer.
  const int per = (p.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(p.batch, (int)threadIdx.x * per), b1 = min(p.batch, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += (long long)paged_head_units<NQ>(p, paged_request(p, b)) * p.heads_kv;
  PagedStart s;
  const long long upto = block_scan<long long>(mine, scan, s.total);
  s.ctas = (int)min((long long)gridDim.x, max(s.total, 1LL));
  const long long c = min((int)blockIdx.x, s.ctas);
  s.unit = c * s.total / s.ctas;
  s.end = (int)blockIdx.x < s.ctas ? (c + 1) * s.total / s.ctas : s.unit;
  long long at = upto - mine;
  __syncthreads();  // scan is written again
  if (s.unit < s.end && at <= s.unit && s.unit < upto) {
    int b = b0;
    while (true) {
      const long long units = (long long)paged_head_units<NQ>(p, paged_request(p, b)) * p.heads_kv;
      if (at + units > s.unit) break;
      at += units;
      ++b;
    }
    *found = b;
    scan[0] = at;
  }
  __syncthreads();
  s.b = *found;
  s.request_unit = scan[0];
  return s;
}

__device__ __forceinline__ uint32_t e4m3x2_of_half2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return r;
}

__device__ __forceinline__ __half2 half2_of_e4m3x2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return *reinterpret_cast<__half2*>(&h);
}

// Sums over the warp, N values at a time, each lane ending with the sums of N / 32 (at least
// one) of them: v[0 .. max(1, N / 32)) for the columns from `column_of_lane` on.
template <int N>
__device__ __forceinline__ int warp_column_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int col = 0, n = N;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool upper = (lane & off) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float send = upper ? v[i] : v[i + n];
          const float keep = upper ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
        }
      }
      col += upper ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
  return col;
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(PagedCfg<T, D, NQ>::kThreads, PagedCfg<T, D, NQ>::kCtas)
    attn_paged_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const PagedParams p) {
  using C = PagedCfg<T, D, NQ>;
  constexpr int NS = C::kNS, NC = C::kNC;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = ptx::smem_u32(smem);
  if ((sbase & 1023u) != 0) {  // swizzled tiles need 1 KB alignment
    if (threadIdx.x == 0) report_error(p.status, p.host_flag, kStatusSmemAlign);
    if (threadIdx.x < 2) p.share[(2 * blockIdx.x + threadIdx.x) * kShareInts] = -1;
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = (int)(threadIdx.x & 31);
  constexpr int kWarpProd = C::kSoftWarps, kWarpMma = kWarpProd + 1, kWarpScale = kWarpProd + 2;
  auto bar = [&](int slot) -> uint32_t { return sbase + C::kBars + slot * 8; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kMisc + 4);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kMisc);

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(bar(C::kKvFull + s), 1);
      ptx::mbar_init(bar(C::kKvEmpty + s), 1);
    }
    ptx::mbar_init(bar(C::kQFull), C::kSoftWarps);
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(bar(C::kSFull + b), 1);
      ptx::mbar_init(bar(C::kSFree + b), C::kSoftWarps);
      ptx::mbar_init(bar(C::kPFull + b), C::kSoftWarps);
      ptx::mbar_init(bar(C::kPvDone + b), 1);
    }
    for (int s = 0; s < C::kScaleRing; ++s) {
      ptx::mbar_init(bar(C::kScFull + s), 1);
      ptx::mbar_init(bar(C::kScEmpty + s), C::kSoftWarps);
    }
    ptx::mbar_init(bar(C::kDrain), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kWarpMma) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_holder), C::kTmemCols);
    ptx::tmem_relinquish();
  }
  if (warp == kWarpProd && lane == 0) {
    ptx::prefetch_tmap(&tmK);
    ptx::prefetch_tmap(&tmV);
  }
  const PagedStart start = paged_start<NQ>(p, reinterpret_cast<long long*>(smem + C::kScan),
                                           reinterpret_cast<int*>(smem + C::kScan + 256));
  if (threadIdx.x < 2) p.share[(2 * blockIdx.x + threadIdx.x) * kShareInts] = -1;
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const Waiter W{abort_flag, p.status, p.timeout_ns, p.host_flag};
  // No role leaves its loop early: once a wait has run out, later ones are skipped, so that
  // every thread still meets its named barriers and the CTA ends soon.
  bool ok = true;
  auto wait = [&](int slot, uint32_t parity) {
    if (ok) ok = W.wait_warp(bar(slot), parity & 1u);
  };
  PagedWalk<NQ> walk(p, start);
  PagedSegment seg;

  if (warp < C::kSoftWarps) {
    // =========================================================== softmax ===
    const int wg = warp >> 2;
    const int t = (warp & 3) * 32 + lane;  // token of the tile; column of the head dim
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const int c_first = wg * NC;           // this warpgroup's query rows of the tile
    float* const col_m = reinterpret_cast<float*>(smem + C::kCol) + c_first;  // max - kPagedTop
    float* const col_q = col_m + NQ;       // q's scale
    float* const col_f = col_m + 2 * NQ;   // factor of a moved maximum; 1 / sum at the end
    int* const col_hi = reinterpret_cast<int*>(col_m + 3 * NQ);
    int* const col_lo = reinterpret_cast<int*>(col_m + 4 * NQ);
    float* const red = reinterpret_cast<float*>(smem + C::kRed) + wg * 4 * NC;
    const float4* const scales = reinterpret_cast<const float4*>(smem + C::kScales);
    const int page = t >> p.block_shift;
    int g = 0;  // tiles so far
    uint32_t fills = 0;  // ring fills of the segments before
    while (walk.next(seg)) {
      const int rows = min(NQ, seg.r.nq * p.group - seg.qt * NQ) - c_first;  // of this warpgroup; may be <= 0
      // ---- the query rows: scale each to (224, 448], split, store as the B operand ----
      ptx::named_bar_sync(1 + wg, 128);  // the last segment's reads of the column arrays are done
      constexpr int kPerRow = D / 16;    // threads (and 16-byte chunks of e4m3) per query row
      const int chunk = t % kPerRow;
#pragma unroll 1
      for (int c = t / kPerRow; c < NC; c += 128 / kPerRow) {
        const int row = seg.qt * NQ + c_first + c;
        const int i = row / p.group, hq = seg.h * p.group + row % p.group;
        uint32_t w[8];
        uint32_t top = 0;
        if (c < rows) {
          const uint4* src = reinterpret_cast<const uint4*>(
              static_cast<const T*>(p.q) + (long long)(seg.r.q0 + i) * p.q_st + (long long)hq * p.q_sh + chunk * 16);
          const uint4 a = __ldg(src), b = __ldg(src + 1);
          w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t m = w[k] & 0x7fff7fffu;
          const uint32_t bad = __vcmpgeu2(m, Elem<T>::kInf2);
          top = __vmaxu2(top, m & ~bad);
          w[k] |= bad & 0x7fff7fffu;  // infinities become NaN: the row's scores have no value
        }
        top = max(top & 0xffffu, top >> 16);
#pragma unroll
        for (int d = 1; d < kPerRow; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float s = append_scale(Elem<T>::to_float2(top).x);
        const float inv = 1.f / s;  // a power of two
        uint32_t term[C::kTerms][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float2 f = Elem<T>::to_float2(w[k]);
          f = make_float2(f.x * inv, f.y * inv);
#pragma unroll
          for (int j = 0; j < C::kTerms; ++j) {
            const uint32_t e = e4m3x2(f.x, f.y);
            const float2 back = e4m3x2_to_float2(e);
            f = make_float2(f.x - back.x, f.y - back.y);
            term[j][k >> 1] = (k & 1) ? term[j][k >> 1] | (e << 16) : e;
          }
        }
#pragma unroll
        for (int j = 0; j < C::kTerms; ++j)
          ptx::st_shared_v4(sbase + C::kQ + j * NQ * D + chunk * (NQ * 16) + (c_first + c) * 16, term[j][0],
                            term[j][1], term[j][2], term[j][3]);
        if (chunk == 0) {
          const int place = seg.r.len - seg.r.nq + min(i, seg.r.nq - 1);
          col_m[c] = kPagedUnset;
          col_q[c] = s;
          col_hi[c] = p.causal ? min(place + 1, seg.r.len) : seg.r.len;
          col_lo[c] = p.window >= 0 ? max(place - p.window, 0) : 0;
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::named_bar_sync(1 + wg, 128);
      if (seg.n > 0 && lane == 0) ptx::mbar_arrive(bar(C::kQFull));
      // Tiles within [lo_all, hi_all) are seen whole by every row of the tile.
      const int p_first = seg.r.len - seg.r.nq + seg.qt * NQ / p.group;
      const int p_last = seg.r.len - seg.r.nq + (min(seg.r.nq * p.group, (seg.qt + 1) * NQ) - 1) / p.group;
      const int hi_all = p.causal ? min(seg.r.len, p_first + 1) : seg.r.len;
      const int lo_all = p.window >= 0 ? max(0, p_last - p.window) : 0;
      float l[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) l[c] = 0.f;

#pragma unroll 1
      for (int j = 0; j < seg.n; ++j, ++g) {
        const int sb = g & 1;
        const int pos0 = (seg.tile + j) * kPagedTile, pos = pos0 + t;
        wait(C::kScFull + g % C::kScaleRing, (uint32_t)(g / C::kScaleRing));
        const float4 sc = scales[(g % C::kScaleRing) * 8 + page];  // a * scale_log2, log2 b, 1 / b
        wait(C::kSFull + sb, (uint32_t)(g >> 1));
        ptx::tc_fence_after();
        uint32_t s[NC];
#pragma unroll
        for (int c = 0; c < NC; c += 16) ptx::tmem_ld16(tmem + lane_off + (uint32_t)(sb * NQ + c_first + c), s + c);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < NC; c += 16) ptx::reg_fence16(s + c);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(bar(C::kScEmpty + g % C::kScaleRing));
          ptx::mbar_arrive(bar(C::kSFree + sb));
        }
        // y = x + log2 b, in place; -inf where the row does not see the token.
#pragma unroll
        for (int c = 0; c < NC; c += 4) {
          const float4 q4 = *reinterpret_cast<const float4*>(col_q + c);
          s[c] = __float_as_uint(fmaf(__uint_as_float(s[c]), sc.x * q4.x, sc.y));
          s[c + 1] = __float_as_uint(fmaf(__uint_as_float(s[c + 1]), sc.x * q4.y, sc.y));
          s[c + 2] = __float_as_uint(fmaf(__uint_as_float(s[c + 2]), sc.x * q4.z, sc.y));
          s[c + 3] = __float_as_uint(fmaf(__uint_as_float(s[c + 3]), sc.x * q4.w, sc.y));
        }
        if (pos0 < lo_all || pos0 + kPagedTile > hi_all) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (pos < col_lo[c] || pos >= col_hi[c]) s[c] = 0xff800000u;
        }
        float most = -INFINITY;
#pragma unroll
        for (int c = 0; c < NC; c += 4) {
          const float4 m4 = *reinterpret_cast<const float4*>(col_m + c);
          most = fmaxf(fmaxf(most, __uint_as_float(s[c]) - m4.x), __uint_as_float(s[c + 1]) - m4.y);
          most = fmaxf(fmaxf(most, __uint_as_float(s[c + 2]) - m4.z), __uint_as_float(s[c + 3]) - m4.w);
        }
        if (ptx::named_bar_or(1 + wg, 128, most > kPagedMost)) {
          // Move the maxima: over the warp, over the warps, then rescale the sums and O.
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float top = ptx::warp_max(__uint_as_float(s[c]));
            if (lane == (c & 31)) red[(warp & 3) * NC + c] = top;
          }
          ptx::named_bar_sync(1 + wg, 128);
          if (t < NC) {
            const float top = fmaxf(fmaxf(red[t], red[NC + t]), fmaxf(red[2 * NC + t], red[3 * NC + t])) - kPagedTop;
            const float old = col_m[t], now = fmaxf(old, top);
            col_f[t] = ptx::ex2(old - now);
            col_m[t] = now;
          }
          ptx::named_bar_sync(1 + wg, 128);
#pragma unroll
          for (int c = 0; c < NC; ++c) l[c] *= col_f[c];
          if (j > 0) {
            wait(C::kPvDone + (sb ^ 1), (uint32_t)((g - 1) >> 1));
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < C::kChunks * NC; c += 16) {
              const int cc = c % NC;
              const uint32_t at = tmem + lane_off + (uint32_t)(2 * NQ + (c / NC) * NQ + c_first + cc);
              uint32_t v[16];
              ptx::tmem_ld16(at, v);
              ptx::tmem_wait_ld();
              ptx::reg_fence16(v);
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * col_f[cc + k]);
              ptx::tmem_st16(at, v);
            }
            ptx::tmem_wait_st();
          }
        }
        // P buffer sb was read by P V of tile g - 2.
        if (g >= 2) wait(C::kPvDone + sb, (uint32_t)((g - 2) >> 1));
        const uint32_t dst = sbase + C::kP + sb * C::kTerms * C::kPTerm + t * 16 + c_first * 128;
#pragma unroll
        for (int c = 0; c < NC; c += 16) {
          uint32_t term[C::kTerms][4];
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const float4 m4 = *reinterpret_cast<const float4*>(col_m + c + k);
            float e[4];
            e[0] = ptx::ex2(__uint_as_float(s[c + k]) - m4.x);
            e[1] = ptx::ex2(__uint_as_float(s[c + k + 1]) - m4.y);
            e[2] = ptx::ex2(__uint_as_float(s[c + k + 2]) - m4.z);
            e[3] = ptx::ex2(__uint_as_float(s[c + k + 3]) - m4.w);
#pragma unroll
            for (int x = 0; x < 4; ++x) l[c + k + x] = fmaf(e[x], sc.z, l[c + k + x]);
            __half2 a = __floats2half2_rn(e[0], e[1]), b = __floats2half2_rn(e[2], e[3]);
#pragma unroll
            for (int j2 = 0; j2 < C::kTerms; ++j2) {
              const uint32_t ea = e4m3x2_of_half2(a), eb = e4m3x2_of_half2(b);
              term[j2][k >> 2] = ea | (eb << 16);
              if (j2 + 1 < C::kTerms) {
                a = __hsub2(a, half2_of_e4m3x2(ea));
                b = __hsub2(b, half2_of_e4m3x2(eb));
              }
            }
          }
#pragma unroll
          for (int j2 = 0; j2 < C::kTerms; ++j2)
            ptx::st_shared_v4(dst + c * 128 + j2 * C::kPTerm, term[j2][0], term[j2][1], term[j2][2], term[j2][3]);
        }
        // Tokens that no row sees: their V rows hold anything (NaN, an older tile), and 0 * NaN
        // would reach O. Clear them.
        if (pos0 < seg.span.lo || pos0 + kPagedTile > seg.span.hi) {
          const uint32_t fill = fills + (j + 1 < seg.n ? 2 * j + 2 : 2 * j + 1);  // V(j)'s place in the ring
          const int slot = (int)(fill % NS);
          wait(C::kKvFull + slot, fill / NS);
          if (wg == 0 && (pos < seg.span.lo || pos >= seg.span.hi)) {
#pragma unroll 1
            for (int k = 0; k < C::kChunks * C::kRow; k += 16)
              ptx::st_shared_v4(sbase + slot * C::kSlotBytes + (k / C::kRow) * (kPagedTile * C::kRow) + t * C::kRow +
                                    k % C::kRow, 0, 0, 0, 0);
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(C::kPFull + sb));
      }
      fills += 2 * seg.n;

      // ---- the segment's result ----
      {
        const int c = warp_column_sums<NC>(l);
        constexpr int kMine = NC / 32 > 1 ? NC / 32 : 1;
        if (NC >= 32 || (lane & (32 / NC - 1)) == 0)
#pragma unroll
          for (int k = 0; k < kMine; ++k) red[(warp & 3) * NC + c + k] = l[k];
      }
      ptx::named_bar_sync(1 + wg, 128);
      if (t < NC && t < rows) {
        const float sum = red[t] + red[NC + t] + red[2 * NC + t] + red[3 * NC + t];
        const float lse2 = sum == 0.f ? -INFINITY : col_m[t] + __log2f(sum);
        col_f[t] = sum == 0.f ? 0.f : 1.f / sum;
        const int row = seg.qt * NQ + c_first + t;
        if (seg.slot >= 0)
          p.part_lse[(long long)seg.slot * NQ + c_first + t] = lse2;
        else if (p.lse != nullptr)
          p.lse[(long long)(seg.h * p.group + row % p.group) * p.total_q + seg.r.q0 + row / p.group] =
              lse2 * 0.69314718055994531f;
      }
      if (seg.slot >= 0 && threadIdx.x == 0) {
        int* at = p.share + seg.slot * kShareInts;
        at[0] = seg.b;
        at[1] = seg.h;
        at[2] = seg.qt;
        at[3] = seg.c0;
        at[4] = seg.c1;
      }
      if (seg.n > 0) wait(C::kPvDone + ((g - 1) & 1), (uint32_t)((g - 1) >> 1));
      ptx::tc_fence_after();
      ptx::named_bar_sync(1 + wg, 128);
#pragma unroll 1
      for (int ch = 0; ch < C::kChunks; ++ch) {
        const int d = ch * 128 + t;
#pragma unroll 1
        for (int c = 0; c < NC; c += 16) {
          if (c >= rows) break;
          uint32_t v[16];
          ptx::tmem_ld16(tmem + lane_off + (uint32_t)(2 * NQ + ch * NQ + c_first + c), v);
          ptx::tmem_wait_ld();
          ptx::reg_fence16(v);
          const int row = seg.qt * NQ + c_first + c;
          int i = row / p.group, hq = row % p.group;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float inv = col_f[c + k];
            // A row that saw nothing has no O (its tiles may not have run): 0, whatever TMEM holds.
            const float val = inv == 0.f ? 0.f : __uint_as_float(v[k]) * inv;
            if (c + k < rows && d < D) {
              if (seg.slot >= 0)
                p.part_o[((long long)seg.slot * NQ + c_first + c + k) * D + d] = val;
              else
                static_cast<T*>(p.o)[(long long)(seg.r.q0 + i) * p.o_st + (long long)(seg.h * p.group + hq) * p.o_sh +
                                     d] = (T)val;
            }
            if (++hq == p.group) {
              hq = 0;
              ++i;
            }
          }
        }
      }
      ptx::tc_fence_before();
    }
  } else if (warp == kWarpProd) {
    // ========================================================== producer ===
    // Ring order per segment: K(0); then K(j + 1), V(j) for each j: the MMA warp's order.
    // Lane i loads page i of the tile; pages that no row sees are left out.
    const uint64_t policy = p.stream_once ? ptx::policy_evict_first() : ptx::policy_evict_last();
    const int pages = kPagedTile >> p.block_shift;
    uint32_t fills = 0;
    auto page_id = [&](int tile) -> int {  // -2: not loaded
      const int at = tile * kPagedTile + (lane << p.block_shift);
      if (lane >= pages || at >= seg.span.hi || at + (1 << p.block_shift) <= seg.span.lo) return -2;
      const int id = __ldg(p.block_table + (long long)seg.b * p.table_stride + (at >> p.block_shift));
      return id >= 0 && id < p.num_blocks ? id : -1;  // -1: outside the cache, reads as zeros
    };
    auto fill = [&](const CUtensorMap* map, int id) {
      const int slot = (int)(fills % NS);
      wait(C::kKvEmpty + slot, (fills / NS) ^ 1u);
      const uint32_t full = bar(C::kKvFull + slot);
      const unsigned loads = __ballot_sync(0xffffffffu, id > -2);
      if (ok) {
        if (lane == 0) ptx::mbar_arrive_expect_tx(full, (uint32_t)(__popc(loads) * D) << p.block_shift);
        __syncwarp();
        if (id > -2) {
#pragma unroll
          for (int ch = 0; ch < C::kChunks; ++ch)
            ptx::tma_load_4d(sbase + slot * C::kSlotBytes + ch * (kPagedTile * C::kRow) +
                                 ((uint32_t)(lane << p.block_shift) * C::kRow),
                             map, full, ch * 128, 0, seg.h, id, policy);
        }
        ++fills;
      }
      __syncwarp();
    };
    while (walk.next(seg)) {
      if (seg.n == 0) continue;
      int id = page_id(seg.tile);
      fill(&tmK, id);
#pragma unroll 1
      for (int j = 0; j < seg.n; ++j) {
        int next = -2;
        if (j + 1 < seg.n) {
          next = page_id(seg.tile + j + 1);
          fill(&tmK, next);
        }
        fill(&tmV, id);
        id = next;
      }
    }
    // Let every load land before the CTA exits.
    if (lane == 0) {
      const int last = (int)min(fills, (uint32_t)NS);
      for (int k = 0; k < last; ++k) {
        const uint32_t f = fills - 1 - k;
        drain_wait(bar(C::kKvFull + (int)(f % NS)), (f / NS) & 1u, p.timeout_ns, p.status, p.host_flag);
      }
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    // =============================================================== MMA ===
    constexpr uint32_t kDesc = (1u << 4) | ((uint32_t)(NQ >> 3) << 17) | ((uint32_t)(kPagedTile >> 4) << 24);
    constexpr uint32_t idS = kDesc;                              // e4m3, fp32 sums, both K-major
    constexpr uint32_t idPV = kDesc | (1u << 15) | (1u << 16);   // both MN-major
    uint32_t reads = 0;  // ring slots consumed
    int gs = 0, gp = 0;  // S and P V tiles issued
    auto acquire = [&]() -> int {
      const int slot = (int)(reads % NS);
      wait(C::kKvFull + slot, reads / NS);
      ++reads;
      return slot;
    };
    auto issue_S = [&]() {
      const int sb = gs & 1;
      if (gs >= 2) wait(C::kSFree + sb, (uint32_t)((gs >> 1) - 1));
      const int slot = acquire();
      ptx::tc_fence_after();
      if (ok) {
        uint32_t acc = 0;
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
          for (int ks = 0; ks < C::kRow / 32; ++ks) {
            const uint64_t a = ptx::smem_desc(sbase + slot * C::kSlotBytes + ch * (kPagedTile * C::kRow) + ks * 32, 16,
                                              8 * C::kRow, C::kSwizzle);
#pragma unroll
            for (int j = 0; j < C::kTerms; ++j) {
              const uint64_t b = ptx::smem_desc(
                  sbase + C::kQ + j * NQ * D + (ch * (C::kRow / 16) + 2 * ks) * (NQ * 16), NQ * 16, 128, 0);
              ptx::umma_ss_f8_warp(tmem + (uint32_t)(sb * NQ), a, b, idS, acc);
              acc = 1;
            }
          }
        ptx::tc_commit_warp(bar(C::kKvEmpty + slot));
        ptx::tc_commit_warp(bar(C::kSFull + sb));
      }
      ++gs;
    };
    auto issue_PV = [&](bool first) {
      const int sb = gp & 1;
      wait(C::kPFull + sb, (uint32_t)(gp >> 1));
      const int slot = acquire();
      ptx::tc_fence_after();
      if (ok) {
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
          for (int ks = 0; ks < kPagedTile / 32; ++ks) {
            // d = 64: the second 64 rows of M repeat the first (zero stride); nobody reads them.
            const uint64_t a = ptx::smem_desc(
                sbase + slot * C::kSlotBytes + ch * (kPagedTile * C::kRow) + ks * 32 * C::kRow, 0, 8 * C::kRow,
                C::kSwizzle);
#pragma unroll
            for (int j = 0; j < C::kTerms; ++j) {
              const uint64_t b = ptx::smem_desc(sbase + C::kP + (sb * C::kTerms + j) * C::kPTerm + ks * 32 * 16, 128, 2048, 0);
              ptx::umma_ss_f8_warp(tmem + (uint32_t)(2 * NQ + ch * NQ), a, b, idPV, first && ks == 0 && j == 0 ? 0u : 1u);
            }
          }
        ptx::tc_commit_warp(bar(C::kKvEmpty + slot));
        ptx::tc_commit_warp(bar(C::kPvDone + sb));
      }
      ++gp;
    };
    int n = 0;  // segments with tiles so far
    while (walk.next(seg)) {
      if (seg.n == 0) continue;
      wait(C::kQFull, (uint32_t)n++);
      issue_S();
#pragma unroll 1
      for (int j = 0; j < seg.n; ++j) {
        if (j + 1 < seg.n) issue_S();
        issue_PV(j == 0);
      }
    }
    ptx::tc_commit_warp(bar(C::kDrain));
    if (lane == 0) drain_wait(bar(C::kDrain), 0, p.timeout_ns, p.status, p.host_flag);
    __syncwarp();
  } else {
    // ============================================================ scales ===
    // Ahead of the softmax: per tile and page, a * sm_scale * log2 e, log2 b and 1 / b.
    const int pages = kPagedTile >> p.block_shift;
    float4* const scales = reinterpret_cast<float4*>(smem + C::kScales);
    int g = 0;
    while (walk.next(seg)) {
#pragma unroll 1
      for (int j = 0; j < seg.n; ++j, ++g) {
        const int at = (seg.tile + j) * kPagedTile + (lane << p.block_shift);
        // Pages that are not there: zero scores and values, and a V scale too small to move a maximum.
        float4 sc = make_float4(0.f, -100.f, 1.f / kPagedLeastScale, 0.f);
        if (lane < pages && at < seg.span.hi && at + (1 << p.block_shift) > seg.span.lo) {
          const int id = __ldg(p.block_table + (long long)seg.b * p.table_stride + (at >> p.block_shift));
          if (id >= 0 && id < p.num_blocks) {
            const float a = __ldg(p.k_scale + (long long)id * p.heads_kv + seg.h);
            const float b = fmaxf(__ldg(p.v_scale + (long long)id * p.heads_kv + seg.h), kPagedLeastScale);
            sc = make_float4(a * p.scale_log2, __log2f(b), 1.f / b, 0.f);
          }
        }
        wait(C::kScEmpty + g % C::kScaleRing, (uint32_t)(g / C::kScaleRing) ^ 1u);
        if (lane < pages) scales[(g % C::kScaleRing) * 8 + lane] = sc;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(C::kScFull + g % C::kScaleRing));
      }
    }
    if (p.zero_rest) {  // rows behind a request and before the next (or the first)
      for (int b = (int)blockIdx.x; b < p.batch; b += gridDim.x) {
        const PagedRequest r = paged_request(p, b);
        const int end = r.q0 + r.nq;
        const int next = b + 1 < p.batch ? paged_request(p, b + 1).q0 : p.total_q;
        const int heads = p.heads_kv * p.group;
        auto clear = [&](int from, int to) {
          for (long long x = lane; x < (long long)max(0, to - from) * heads * (D / 8); x += 32) {
            const int d = (int)(x % (D / 8)) * 8, hq = (int)(x / (D / 8) % heads), row = from + (int)(x / (D / 8) / heads);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (long long)row * p.o_st + (long long)hq * p.o_sh + d) =
                make_uint4(0, 0, 0, 0);
            if (p.lse != nullptr && d == 0) p.lse[(long long)hq * p.total_q + row] = 0.f;
          }
        };
        clear(end, next);
        if (b == 0) clear(0, r.q0);
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kTmemCols);
  }
  ptx::launch_dependents();
}

// Joins the parts of the items that several CTAs shared: o = sum_k w_k o_k / sum_k w_k with
// w_k = 2^(lse_k - max lse), in the CTAs' order. The CTAs c0 .. c1 of an item take its rows in
// turn, a warp per row where few parts meet and all warps a share of the parts where many do.
constexpr int kCombineThreads = 256;

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(kCombineThreads) attn_paged_combine_kernel(const PagedParams p) {
  constexpr int kWarps = kCombineThreads / 32, E = D / 32;
  __shared__ float part[kWarps][D];
  __shared__ float stat[kWarps][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::wait_for_previous_grid();
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int* at = p.share + (2 * blockIdx.x + side) * kShareInts;
    const int b = at[0];
    if (b < 0) continue;
    const int h = at[1], qt = at[2], c0 = at[3], c1 = at[4];
    const int k_parts = c1 - c0 + 1;
    const PagedRequest r = paged_request(p, b);
    const int rows = min(NQ, r.nq * p.group - qt * NQ);
    const bool alone = k_parts <= 4;  // a warp joins a row by itself
    const int lanes = alone ? kWarps : 1;
    for (int c = ((int)blockIdx.x - c0) * lanes + (alone ? warp : 0); c < rows; c += k_parts * lanes) {
      // Part k is CTA c0 + k's: the first left it behind, the others got it from before.
      auto slot = [&](int k) { return (long long)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * NQ + c; };
      const int first = alone ? 0 : warp, step = alone ? 1 : kWarps;
      float m = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int k = first + lane * step; k < k_parts; k += 32 * step) m = fmaxf(m, p.part_lse[slot(k)]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
      for (int k = first; k < k_parts; k += step) {
        const float w = ptx::ex2(p.part_lse[slot(k)] - base);
        const float* o = p.part_o + slot(k) * D + lane * E;
        sum += w;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(o + e);
          acc[e] = fmaf(w, v.x, acc[e]);
          acc[e + 1] = fmaf(w, v.y, acc[e + 1]);
        }
      }
      if (!alone) {
        if (lane == 0) {
          stat[warp][0] = m;
          stat[warp][1] = sum;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) part[warp][lane * E + e] = acc[e];
        __syncthreads();
        float all = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all = fmaxf(all, stat[w][0]);
        const float base_all = all == -INFINITY ? 0.f : all;
        if (warp == 0) {
          sum = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            // A warp without parts has max -inf: weight 0.
            const float f = ptx::ex2(stat[w][0] - base_all);
            sum += f * stat[w][1];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(f, part[w][lane * E + e], acc[e]);
          }
          m = all;
        }
        __syncthreads();
        if (warp != 0) continue;
      }
      const int row = qt * NQ + c;
      const int i = row / p.group, hq = h * p.group + row % p.group;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T* o = static_cast<T*>(p.o) + (long long)(r.q0 + i) * p.o_st + (long long)hq * p.o_sh + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(o + e) = DType<T>::pack(acc[e] * inv, acc[e + 1] * inv);
      if (p.lse != nullptr && lane == 0)
        p.lse[(long long)hq * p.total_q + r.q0 + i] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.69314718055994531f;
    }
  }
}

}  // namespace apex
