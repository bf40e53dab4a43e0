// Attention over a paged 8-bit K/V cache (the layout kv_cache_kernels.cuh writes) for sm_100a.
//
// For query rows q_i of one K/V head (the heads of its group and a request's new tokens
// together) and cached tokens j with codes k_j, v_j and block scales a_j, b_j:
//   x_ij = sm_scale * log2(e) * a_j * (q_i . k_j)          (base-2 scores)
//   o_i  = sum_j 2^x_ij b_j v_j / sum_j 2^x_ij
//
// The codes never leave 8 bits: both products run on tcgen05.mma kind::f8f6f4 with the cache
// tiles as the TMA wrote them to shared memory, so nothing converts the cache. What is not
// 8 bits wide is split into terms that add up to it:
//   * q, scaled per row by a power of two so that its largest magnitude lies in (224, 448]: two
//     terms of e4m3 for bf16 calls, and a third of e5m2 for fp16 ones. Its 8 or 11 significant bits
//     in pieces of 4, 4 and 3, exact but for what lies below 2^-10 (two terms) or 2^-17;
//   * the weight p'_ij = 2^(x_ij + log2 b_j - m_i) (the V scale goes into the exponent, one
//     addition per token), rounded to fp16: three terms of e5m2 for either type. Each is the nearest to
//     what the ones before it left, with a sign of its own, so that the 11 bits come in pieces of 3, 4
//     and 4: exact for weights from 2^-6 on, off by at most 2^-17 below. So a weight is off by 2^-11
//     of itself, or by 2^-30 of the row's largest.
// The weights need e5m2's exponents more than e4m3's bits. A row may have most of its weight on one
// token whose V is small, and its output is then the mean of many small weights: with two terms of
// e4m3, which end 2^-16 below the largest, 8192 tokens behind one of share 0.95 vanished from the
// output (and not from the sum); with a third of e5m2 they were off by 4 % where all were alike.
// The products of 32 tokens are exact to 2^-23 of their magnitudes, and their fp32 sums over the tiles are cut,
// not rounded: 131k tokens of one sign in one piece come out 2.6e-4 low, 524k 1.4e-3 (bf16's half step
// is 3.9e-3, fp16's 4.9e-4). An item that several CTAs share has shorter pieces.
//
// Up to 32 query rows per K/V head, tokens are the M side ("token-major"): S^T = K Q^T and O^T = V^T P,
// M = 128 tokens resp. 128 columns of the head dim, N = 16 or 32 query rows. A decode step has 1 to
// 16 query rows per K/V head; as the M side they would leave most of a 128-row tile empty. Thread t
// owns token t of a tile: its scales are per-thread scalars and its row of P is 16 contiguous bytes
// per 16 query rows. The price is that a row's maximum runs across threads; so the running
// maximum is only moved when some p' would pass 2^15.75 (one vote per tile), which is rare after
// a row's first tile.
// More rows, in tiles of 64 or 128, are the M side themselves ("query-major"): S = Q K^T, O = P V, a
// thread owns part of a row, and a maximum takes one exchange between warps. (Measured: 32 requests of
// 40 rows take 31.8 us in tiles of 64, 43.6 in two token-major tiles of 32, 38.4 in tiles of 128.)
//
// m_i tracks the maximum of x_ij + log2 b_j, kept 2^13 below p's top so that small weights stay
// above e5m2's floor: the largest weight of a row is held at 2^13 .. 2^15.75 (e5m2's largest is
// 57344 = 2^15.81). The row sum sum_j 2^(x_ij - m_i) = sum_j p'_ij / b_j is taken from the fp32 p', and
// scaled by 2^-13: with b = 2^-100 throughout (a context of zeros) it would overflow.
//
// Work: an item is (request, K/V head, query-row tile); its tiles of 128 tokens line up with all
// other items' in one sequence, which is cut into equal ranges, one per CTA, whatever the
// lengths. A CTA writes what it has of an item that it shares to the workspace (normalised
// rows and their base-2 logsumexp) and attn_paged_combine_kernel joins them in a fixed order.
// Lengths are read on the device only.
//
// Warps: 4 to 16 softmax (32 rows of TMEM each), then TMA producer, MMA issuer, scales and work
// list, and a fourth that token-major splits the next segment's query rows. The scales' warp alone walks the work list and publishes the segments
// in shared memory: a warp on its own takes some 4 cycles per dependent instruction, and all
// warps walking cost each of them about 2 us at the start and 1 us per segment.
//
// Bound: a decode step by the cache's bytes (48 requests of up to 8191 tokens, 410 MB: 76 us a call,
// 5.4 TB/s; some 7 us of them pass before the first scores are there, 4 in the joining kernel);
// calls with many new tokens by the softmax warps' issue (3 x 1024 tokens on 5k to 16k: 657 us a
// call, 663 TFLOP/s; schedulers busy 52 %, tensor pipe 34 %).
#pragma once

#include "attn_fwd_kernel.cuh"
#include "kv_cache_kernels.cuh"

namespace apex {

constexpr int kPagedTile = 128;      // cached tokens per tile
constexpr float kPagedTop = 13.0f;    // log2 of the weight that a row's maximum maps to
constexpr float kPagedMost = 15.75f;  // a weight above 2^this moves the maximum (57344 = 2^15.807)
constexpr float kPagedSumUnit = 1.f / 8192.f;  // 2^-kPagedTop: row sums are in these
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
  float* part_o;    // [2 * CTAs][NQ][D]: of CTA c's entries in `share`
  float* part_lse;  // [2 * CTAs][NQ]
  int* share;       // [2 * CTAs][kShareInts]
  int* status;
  int* host_flag;
  unsigned long long timeout_ns;
  long long table_stride;
  long long q_st, q_sh, o_st, o_sh;  // token, head strides (elements)
  int batch, heads_kv, group, total_q, max_q;
  unsigned group_magic;  // ceil(2^32 / group), for rows of a tile (0: group is 1)
  int num_blocks, block_shift, table_width;
  int causal, window, zero_rest;
  int one_tile;      // every request's rows of a K/V head fit one query tile; the cache is read once
  float scale_log2;  // sm_scale * log2(e)
};

// One entry per CTA for the item that reaches it from the CTA before (2c) and for the one
// that it leaves to the next (2c + 1): first query row of the request (-1: no entry), K/V head,
// rows of the tile, first token; first and last CTA, first head.
constexpr int kShareInts = 8;

template <typename T, int D, int NQ>
struct PagedCfg {
  static_assert(D == 64 || D == 128 || D == 256, "head dims 64, 128, 256");
  static constexpr int kRow = D < 128 ? D : 128;         // bytes of a token row in a column chunk
  static constexpr int kChunks = (D + 127) / 128;
  static constexpr uint32_t kSwizzle = kRow == 128 ? 2 : 4;
  static constexpr int kQTerms = std::is_same<T, __half>::value ? 3 : 2;  // of a query value
  static constexpr int kWTerms = 3;                                       // of a weight
  static constexpr bool kQueryMajor = NQ >= 64;
  // Columns of an S buffer.
  static constexpr int kSCols = kQueryMajor ? kPagedTile : NQ;
  static constexpr int kWG = kQueryMajor ? 4 : 1;        // softmax warpgroups
  // Query-major, d <= 128: two pairs of warpgroups take the tiles in turn, each pair with its own
  // maxima, sums and O, so that one's exponentials run while the other loads and converts.
  static constexpr int kPairs = kQueryMajor && D <= 128 ? 2 : 1;
  static constexpr int kLead = kPairs;                   // S runs this many tiles ahead of P V
  static constexpr int kSoftWarps = 4 * kWG;
  static constexpr int kTileWarps = kSoftWarps / kPairs; // softmax warps per tile
  static constexpr int kThreads = 128 * (kWG + 1);
  // Two CTAs per SM cover each other's latencies where their shared memory fits.
  static constexpr int kCtas = (D <= 128 && NQ <= 32) ? 2 : 1;
  static constexpr int kSlotBytes = kPagedTile * D;      // one K or V tile
  static constexpr int kPTerm = kPagedTile * NQ;         // one term of one P buffer
  static constexpr int kBudget = kCtas == 2 ? 115712 : 232448;
  static constexpr int kMiscBytes = 2240 + NQ * 60 + (kQueryMajor ? 14 * 128 * 4 : 0);  // what the plan below adds
  // Query-major M is 128 for 64-row tiles too. Where shared memory holds Q twice, rows 64 .. 127 of S
  // repeat the first 64 and their threads take half of the tokens: TMEM lanes belong to warps by
  // their quarter, so two of the SM's four schedulers would do nothing otherwise. Of O, rows 64 .. 127
  // are never read; the weights that they come from are what lies behind the 64 rows.
  static constexpr int kCopies =
      NQ == 64 && 2 * kQTerms * NQ * D + kWTerms * kPTerm + kMiscBytes + 3 * kSlotBytes <= kBudget ? 2 : 1;
  static constexpr int kQBytes = kQTerms * NQ * D * kCopies;  // one segment's query rows
  static constexpr int slots(int q_bufs, int p_bufs) {
    return (kBudget - q_bufs * kQBytes - p_bufs * kWTerms * kPTerm - kMiscBytes) / kSlotBytes;
  }
  static constexpr int kPBufs = slots(1, 2) >= 3 ? 2 : 1;
  // The next segment's query rows are split ahead of time, by a warp of their own, where that
  // leaves four ring slots; a query-major tile's are too many for one warp, and the softmax
  // warps split them between segments.
  static constexpr bool kSelfSplit = kQueryMajor;
  static constexpr int kQBufs = !kSelfSplit && slots(2, kPBufs) >= 4 ? 2 : 1;
  static constexpr int kNS = slots(kQBufs, kPBufs) > 12 ? 12 : slots(kQBufs, kPBufs);  // ring slots
  static_assert(kNS > kLead, "the ring needs K(j + kLead) beside V(j)");
  // Query-major: threads per row and tile, and the tokens of each.
  static constexpr int kParts = kWG / kPairs * kCopies;
  static constexpr int kTok = kPagedTile / kParts;
  // S values per thread at once: query rows, or tokens.
  static constexpr int kNC = kQueryMajor ? (kTok < 32 ? kTok : 32) : NQ;
  static constexpr int kScaleRing = 8;
  static constexpr int kSegRing = 4;
  // TMEM: S buffers at 0 and kSCols, O from 2 kSCols on (token-major: a block of NQ columns per 128 of
  // the head dim; query-major: the head dim, for each pair).
  static constexpr int kTmemUsed = 2 * kSCols + (kQueryMajor ? kPairs * D : kChunks * NQ);
  static constexpr int kTmemCols = kTmemUsed <= 64 ? 64 : (kTmemUsed <= 128 ? 128 : (kTmemUsed <= 256 ? 256 : 512));
  static_assert(kTmemUsed <= 512 && kCtas * kTmemCols <= 512, "TMEM plan");
  // shared-memory plan
  static constexpr int kQ = kNS * kSlotBytes;
  static constexpr int kP = kQ + kQBufs * kQBytes;
  static constexpr int kBars = kP + kPBufs * kWTerms * kPTerm;
  static constexpr int kKvFull = 0, kKvEmpty = kNS, kQFull = 2 * kNS, kQEmpty = kQFull + 2,
                       kColEmpty = kQEmpty + 2, kSFull = kColEmpty + 2, kSFree = kSFull + 2, kPFull = kSFree + 2, kPvDone = kPFull + 2, kScFull = kPvDone + 2,
                       kScEmpty = kScFull + kScaleRing, kSegFull = kScEmpty + kScaleRing,
                       kSegEmpty = kSegFull + kSegRing, kDrain = kSegEmpty + kSegRing, kNumBars = kDrain + 1;
  static constexpr int kScales = (kBars + kNumBars * 8 + 15) / 16 * 16;  // float4 [kScaleRing][8 pages]
  static constexpr int kCol = kScales + kScaleRing * 8 * 16;  // two of, per query row: -m, q scale, factor, hi, lo
  static constexpr int kRed = kCol + 2 * 5 * NQ * 4;          // token-major [4 warps + 1][NQ], query-major [14][128]
  static constexpr int kSegs = (kRed + (kQueryMajor ? 14 * 128 : 5 * NQ) * 4 + 15) / 16 * 16;       // int4 [kSegRing][kSegVecs]
  static constexpr int kBad = kSegs + kSegRing * 4 * 16;                 // unsigned [2][4]
  static constexpr int kScan = kBad + 32;                // long long [32], found request
  static constexpr int kMisc = kScan + 32 * 8 + 16;
  static constexpr int kBytes = kMisc + 16;
  static_assert(kBytes <= kBudget, "shared-memory plan");
  static_assert(!kQueryMajor || kBytes - kBars >= (128 - NQ) * 128, "rows behind the last weights");
};

// Inputs are read by plain loads. The kernel may start while the one that writes them still runs
// (it waits for that before it reads), and then they are not constant for its lifetime, as the
// non-coherent path takes them to be.
template <typename V>
__device__ __forceinline__ V read_input(const V* at) {
  return *at;
}

// The query rows of request b and where they stand.
struct PagedRequest {
  int q0, nq, len;  // first row, rows, cached tokens
};

__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int b) {
  PagedRequest r;
  if (p.cu_seqlens_q != nullptr) {
    r.q0 = min(max(read_input(p.cu_seqlens_q + b), 0), p.total_q);
    r.nq = min(max(read_input(p.cu_seqlens_q + b + 1), r.q0), p.total_q) - r.q0;
    r.nq = min(r.nq, p.max_q);
  } else {
    r.nq = p.max_q;
    r.q0 = b * r.nq;
  }
  r.len = min(max(read_input(p.seq_lens + b), 0), p.table_width << p.block_shift);
  return r;
}

// Row c (below 2^15) of a tile that begins at head `head0` of the group for query token `token0`:
// its query token, and its head in the group.
__device__ __forceinline__ void paged_row(const PagedParams& p, int token0, int head0, int c, int& token, int& head) {
  const unsigned x = (unsigned)(head0 + c);  // x * group < 2^32: the product with the magic is exact
  const int t = p.group_magic ? (int)__umulhi(x, p.group_magic) : (int)x;
  token = token0 + t;
  head = (int)x - t * p.group;
}

// Tokens [lo, hi) are what the rows of query tile qt see together; [t0, t0 + n) are their tiles.
struct PagedSpan {
  int lo, hi, t0, n;
  int i0, i1;  // first and last query token of the tile
};

template <int NQ>
__device__ __forceinline__ PagedSpan paged_span(const PagedParams& p, const PagedRequest& r, int qt) {
  int i0 = 0, i1 = r.nq - 1;
  if (!p.one_tile) {
    i0 = qt * NQ / p.group;
    i1 = (min(r.nq * p.group, (qt + 1) * NQ) - 1) / p.group;
  }
  const int first = r.len - r.nq + i0, last = r.len - r.nq + i1;  // positions
  PagedSpan s;
  s.i0 = i0;
  s.i1 = i1;
  s.hi = p.causal ? min(r.len, last + 1) : r.len;
  s.lo = p.window >= 0 ? max(0, first - p.window) : 0;
  s.t0 = s.lo / kPagedTile;
  s.n = s.hi > s.lo ? (s.hi + kPagedTile - 1) / kPagedTile - s.t0 : 0;
  return s;
}

template <int NQ>
__device__ __forceinline__ int paged_qtiles(const PagedParams& p, const PagedRequest& r) {
  return p.one_tile ? min(r.nq, 1) : (r.nq * p.group + NQ - 1) / NQ;
}

// A CTA that begins an item spends about as long on it as on this many tiles: units of an item
// are these and then its tiles, at least one (an item that sees nothing still has rows to
// write). Without them the CTAs that got short requests finished last: 48 requests of 129 to
// 8191 tokens take 102 us instead of 77, and three of 1024 new tokens each 695 instead of 665.
template <int NQ>
constexpr int kPagedItemUnits = NQ <= 32 ? 4 : 8;

// Units of one K/V head of a request.
template <int NQ>
__device__ __forceinline__ int paged_head_units(const PagedParams& p, const PagedRequest& r) {
  const int qts = paged_qtiles<NQ>(p, r);
  int units = 0;
  for (int qt = 0; qt < qts; ++qt) units += kPagedItemUnits<NQ> + max(1, paged_span<NQ>(p, r, qt).n);
  return units;
}

// A CTA's part of an item, as the walking warp publishes it.
struct PagedSegment {
  int b, h, q0, nq;              // request, K/V head, the request's first query row and rows
  int len, lo, hi, tile;         // cached tokens; tokens [lo, hi) are seen; first tile
  int n, slot, rows, token0;     // tiles (-1: no more segments); workspace entry, -1 if the item is whole
  int head0, lo_all, hi_all, pad;  // rows' first head; tokens [lo_all, hi_all) are seen by every row
};
constexpr int kSegVecs = sizeof(PagedSegment) / 16;
static_assert(sizeof(PagedSegment) == 64, "published as four 16-byte words");

// Where the walk begins: the CTA's range of units and the request that it begins in. The host
// refuses calls whose units might not fit 31 bits; offsets that overlap could name more, and then
// nothing is done.
struct PagedStart {
  int unit, end;     // the CTA's range
  int request_unit;  // first unit of request b
  int share;         // units per CTA, one more for each of the first `more`
  int b, more;

  __device__ __forceinline__ void cut(long long units) {
    const int total = units > 0x7fffffff ? 0 : (int)units;
    share = (int)((unsigned)total / gridDim.x);
    more = total - share * (int)gridDim.x;
    const int c = (int)blockIdx.x;
    unit = c * share + min(c, more);
    end = unit + share + (c < more ? 1 : 0);
  }
};

template <int NQ>
struct PagedWalk {
  const PagedParams& p;
  int unit, end, share, more;
  int b, h, qt, qts;
  int item;  // first unit of the item (b, h, qt)
  int tiles_begin = 0, tiles_end = 0;  // units of the tiles of the last segment's item
  PagedRequest r, ahead;  // of b, and of b + 1, read before it is needed

  __device__ __forceinline__ void look_ahead() {
    if (b + 1 < p.batch) ahead = paged_request(p, b + 1);
  }

  __device__ __forceinline__ PagedWalk(const PagedParams& params, const PagedStart& s)
      : p(params), unit(s.unit), end(s.end), share(s.share), more(s.more), b(s.b), h(0), qt(0), qts(0),
        item(s.request_unit) {
    if (unit >= end) return;
    r = paged_request(p, b);
    look_ahead();
    qts = paged_qtiles<NQ>(p, r);
    const int into = unit - item;
    if (p.heads_kv > 1 && into > 0) {
      const int per_head = paged_head_units<NQ>(p, r);
      h = (int)((unsigned)into / (unsigned)per_head);
      item += h * per_head;
    }
    while (qt + 1 < qts) {
      const int n = kPagedItemUnits<NQ> + max(1, paged_span<NQ>(p, r, qt).n);
      if (item + n > unit) break;
      item += n;
      ++qt;
    }
  }

  // The CTA whose range holds a unit.
  __device__ __forceinline__ int cta_of(int u) const {
    const int large = more * (share + 1);
    return u < large ? (int)((unsigned)u / (unsigned)(share + 1)) : more + (int)((unsigned)(u - large) / (unsigned)share);
  }

  // The next segment, or one of -1 tiles behind the last.
  __device__ __forceinline__ PagedSegment next() {
    PagedSegment s;
    s.n = -1;
    while (unit < end) {
      while (qt == qts) {  // on to the next head or request that has query rows
        qt = 0;
        if (++h == p.heads_kv || qts == 0) {
          h = 0;
          if (++b >= p.batch) return s;  // (units and requests always end together)
          r = ahead;
          look_ahead();
          qts = paged_qtiles<NQ>(p, r);
        }
      }
      const PagedSpan span = paged_span<NQ>(p, r, qt);
      const int n = max(1, span.n);
      const int first = item + kPagedItemUnits<NQ>, last = first + n;  // the tiles' units
      const int from = max(unit, first), to = min(end, last);
      const int row0 = qt * NQ;
      unit = min(end, last);
      item = last;
      ++qt;
      if (from >= to) continue;  // the range ends before the item's first tile
      s.b = b;
      s.h = h;
      s.q0 = r.q0;
      s.nq = r.nq;
      s.len = r.len;
      s.lo = span.lo;
      s.hi = span.hi;
      s.tile = span.t0 + (from - first);
      s.n = span.n == 0 ? 0 : to - from;
      s.rows = min(NQ, r.nq * p.group - row0);
      s.token0 = span.i0;
      s.head0 = row0 - span.i0 * p.group;
      const int place = r.len - r.nq;
      s.hi_all = p.causal ? min(r.len, place + span.i0 + 1) : r.len;
      s.lo_all = p.window >= 0 ? max(0, place + span.i1 - p.window) : 0;
      s.slot = -1;
      if (to - from < n) s.slot = 2 * (int)blockIdx.x + (from > first ? 0 : 1);
      tiles_begin = first;
      tiles_end = last;
      return s;
    }
    return s;
  }

  // Leaves the joining kernel what it needs to know of a segment that is part of an item. (After
  // the segment is published: nobody waits for this.)
  __device__ __forceinline__ void share_out(const PagedSegment& s) const {
    if (s.n < 0 || s.slot < 0 || (threadIdx.x & 31) != 0) return;
    int4* at = reinterpret_cast<int4*>(p.share + s.slot * kShareInts);
    at[0] = make_int4(s.q0, s.h, s.rows, s.token0);
    at[1] = make_int4(cta_of(tiles_begin), cta_of(tiles_end - 1), s.head0, 0);
  }
};

constexpr int kPagedWarpBatch = 128;  // requests that one warp looks over by itself

// The CTA's range, and the request that it begins in: by one warp, for batches up to
// kPagedWarpBatch.
template <int NQ>
__device__ __forceinline__ PagedStart paged_start_warp(const PagedParams& p) {
  constexpr int kRounds = kPagedWarpBatch / 32;
  const int lane = (int)(threadIdx.x & 31);
  PagedStart s;
  int upto[kRounds], mine[kRounds], total = 0;
  long long whole = 0;  // the total, which `total` may not hold
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    mine[i] = 0;
    if (32 * i < p.batch) {
      const int b = 32 * i + lane;
      if (b < p.batch) mine[i] = paged_head_units<NQ>(p, paged_request(p, b)) * p.heads_kv;
    }
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    upto[i] = mine[i];
    if (32 * i < p.batch) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto[i], d);
        if (lane >= d) upto[i] += up;
      }
      upto[i] += total;
      total = __shfl_sync(0xffffffffu, upto[i], 31);
      whole += __reduce_add_sync(0xffffffffu, (unsigned)mine[i] & 0xffffu);
      whole += (long long)__reduce_add_sync(0xffffffffu, (unsigned)mine[i] >> 16) << 16;
    }
  }
  s.cut(whole);
  s.b = 0;
  s.request_unit = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (32 * i < p.batch) {
      const unsigned has = __ballot_sync(0xffffffffu, upto[i] - mine[i] <= s.unit && s.unit < upto[i]);
      if (has != 0) {
        s.b = 32 * i + __ffs(has) - 1;
        s.request_unit = __shfl_sync(0xffffffffu, upto[i] - mine[i], __ffs(has) - 1);
      }
    }
  }
  return s;
}

// The same by the whole CTA: each thread sums a run of requests, and the one whose run holds
// the first unit looks closer.
template <int NQ>
__device__ __forceinline__ PagedStart paged_start_cta(const PagedParams& p, long long* scan, int* found) {
  PagedStart s;
  const int per = (p.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(p.batch, (int)threadIdx.x * per), b1 = min(p.batch, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += paged_head_units<NQ>(p, paged_request(p, b)) * p.heads_kv;
  long long total;
  const long long upto = block_scan<long long>(mine, scan, total);
  s.cut(total);
  long long at = upto - mine;
  __syncthreads();  // scan is written again
  if (s.unit < s.end && at <= s.unit && s.unit < upto) {
    int b = b0;
    while (b + 1 < b1) {
      const int units = paged_head_units<NQ>(p, paged_request(p, b)) * p.heads_kv;
      if (at + units > s.unit) break;
      at += units;
      ++b;
    }
    *found = b;
    scan[0] = at;
  }
  __syncthreads();
  s.b = *found;
  s.request_unit = (int)scan[0];
  return s;
}

// Four fp16 values to e5m2, a.x in the lowest byte.
__device__ __forceinline__ uint32_t e5m2x4_of_half2(__half2 a, __half2 b) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e5m2x2.f16x2 lo, %1;\n\t"
      "cvt.rn.satfinite.e5m2x2.f16x2 hi, %2;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "r"(*reinterpret_cast<uint32_t*>(&a)), "r"(*reinterpret_cast<uint32_t*>(&b)));
  return r;
}

// Four fp16 values to e4m3 (a.x in the lowest byte) and back. One asm block each, so that the
// halves are converted in place instead of being moved and merged.
__device__ __forceinline__ uint32_t e4m3x4_of_half2(__half2 a, __half2 b) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 lo, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 hi, %2;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "r"(*reinterpret_cast<uint32_t*>(&a)), "r"(*reinterpret_cast<uint32_t*>(&b)));
  return r;
}

__device__ __forceinline__ void half2_of_e4m3x4(uint32_t v, __half2& a, __half2& b) {
  uint32_t x, y;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "mov.b32 {lo, hi}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=r"(x), "=r"(y)
      : "r"(v));
  a = *reinterpret_cast<__half2*>(&x);
  b = *reinterpret_cast<__half2*>(&y);
}

// e5m2 is fp16's upper byte.
__device__ __forceinline__ void half2_of_e5m2x4(uint32_t v, __half2& a, __half2& b) {
  const uint32_t x = __byte_perm(v, 0, 0x1404), y = __byte_perm(v, 0, 0x3424);
  a = *reinterpret_cast<const __half2*>(&x);
  b = *reinterpret_cast<const __half2*>(&y);
}

// Splits four weights (fp16, below 57344) into terms of e5m2 that add up to them.
template <int K>
__device__ __forceinline__ void split_weights(__half2 a, __half2 b, uint32_t (&term)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) {
    term[i] = e5m2x4_of_half2(a, b);
    if (i + 1 < K) {
      __half2 ra, rb;
      half2_of_e5m2x4(term[i], ra, rb);
      a = __hsub2(a, ra);
      b = __hsub2(b, rb);
    }
  }
}

// Splits four query values (fp16) into K terms that add up to them: e4m3, and of three the last e5m2, whose
// smallest values lie 2^7 below e4m3's (a third piece has three bits left, as many as it holds).
template <int K>
__device__ __forceinline__ void split_query(__half2 a, __half2 b, uint32_t (&term)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) {
    if (i == 2) {
      term[i] = e5m2x4_of_half2(a, b);
      continue;
    }
    term[i] = e4m3x4_of_half2(a, b);
    if (i + 1 < K) {
      __half2 ra, rb;
      half2_of_e4m3x4(term[i], ra, rb);
      a = __hsub2(a, ra);
      b = __hsub2(b, rb);
    }
  }
}

// Sums N (at most 32) values per lane over the warp; each lane ends with the sum of one in
// v[0] and gets its index (lanes that differ in the lowest bit share one if N is 16).
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

// Splits a segment's query rows: each is scaled by a power of two to (224, 448], split into
// 8-bit terms and stored as the B operand of S^T, [term][16-byte chunk of the head dim][row]; the
// rows' column arrays are set up. Warp `w` of `warps` takes its share of the rows.
template <typename T, int D, int NQ, int kAhead>
__device__ __forceinline__ void split_query_rows(const PagedParams& p, const PagedSegment& seg, uint8_t* smem,
                                                 int n, int w, int warps) {
  using C = PagedCfg<T, D, NQ>;
  constexpr int kPerRow = D / 16;      // lanes per query row, 16 values each
  constexpr int kStep = 32 / kPerRow;  // rows per warp and step; kAhead steps' loads are under way
  const int lane = (int)(threadIdx.x & 31), chunk = lane % kPerRow;
  float* const col_nm = reinterpret_cast<float*>(smem + C::kCol) + (n & 1) * 5 * NQ;
  const uint32_t dst = ptx::smem_u32(smem) + C::kQ + (n % C::kQBufs) * C::kQBytes;
  // Row c's place: token-major [16-byte chunk of the head dim][row], query-major rows of up to 128
  // bytes, swizzled as the TMA writes K.
  auto place_of = [&](int c) -> uint32_t {
    if constexpr (!C::kQueryMajor) return dst + chunk * (NQ * 16) + c * 16;
    constexpr int kUnits = C::kRow / 16;
    const uint32_t off = (uint32_t)(c * C::kRow + chunk % kUnits * 16);
    return dst + chunk / kUnits * (C::kCopies * NQ * C::kRow) + (off ^ (((off >> 7) & (kUnits - 1)) << 4));
  };
  const T* const q = static_cast<const T*>(p.q) + (long long)seg.q0 * p.q_st +
                     (long long)(seg.h * p.group) * p.q_sh + chunk * 16;
  uint4 na[kAhead], nb[kAhead];
  auto load = [&](int c, uint4& a, uint4& b) {
    a = b = make_uint4(0, 0, 0, 0);
    if (c < seg.rows) {
      int token, head;
      paged_row(p, seg.token0, seg.head0, c, token, head);
      const uint4* src = reinterpret_cast<const uint4*>(q + token * p.q_st + head * p.q_sh);
      a = read_input(src);
      b = read_input(src + 1);
    }
  };
  const int first = w * kStep + lane / kPerRow, step = warps * kStep;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(first + i * step, na[i], nb[i]);
#pragma unroll 1
  for (int c = first; c < NQ; c += step) {
    uint32_t x[8] = {na[0].x, na[0].y, na[0].z, na[0].w, nb[0].x, nb[0].y, nb[0].z, nb[0].w};
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) na[i] = na[i + 1], nb[i] = nb[i + 1];
    load(c + kAhead * step, na[kAhead - 1], nb[kAhead - 1]);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = x[k] & 0x7fff7fffu;
      const uint32_t bad = __vcmpgeu2(m, Elem<T>::kInf2);
      top = __vmaxu2(top, m & ~bad);
      x[k] |= bad & 0x7fff7fffu;  // infinities become NaN: the row's scores have no value
    }
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
    for (int d = 1; d < kPerRow; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float s = append_scale(Elem<T>::to_float2(top).x);
    const float inv = 1.f / s;  // a power of two
    uint32_t term[C::kQTerms][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // Scaled values fit fp16 exactly (11 bits; below 2^-13 fewer, far under e4m3's floor).
      const float2 f = __fmul2_rn(Elem<T>::to_float2(x[2 * k]), make_float2(inv, inv));
      const float2 g = __fmul2_rn(Elem<T>::to_float2(x[2 * k + 1]), make_float2(inv, inv));
      __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(g.x, g.y);
      uint32_t four[C::kQTerms];
      split_query(a, b, four);
#pragma unroll
      for (int j = 0; j < C::kQTerms; ++j) term[j][k] = four[j];
    }
#pragma unroll
    for (int j = 0; j < C::kQTerms; ++j) {
      const uint32_t at = place_of(c) + j * C::kCopies * NQ * D;
      ptx::st_shared_v4(at, term[j][0], term[j][1], term[j][2], term[j][3]);
      if (C::kCopies == 2) ptx::st_shared_v4(at + NQ * C::kRow, term[j][0], term[j][1], term[j][2], term[j][3]);
    }
    if (C::kQueryMajor) {
      if (chunk == 0) col_nm[NQ + c] = s;
    } else if (chunk == 0) {
      int token, head;
      paged_row(p, seg.token0, seg.head0, c, token, head);
      const int place = seg.len - seg.nq + min(token, seg.nq - 1);
      col_nm[c] = 0.f;
      col_nm[NQ + c] = s;
      col_nm[2 * NQ + c] = -1.f;
      reinterpret_cast<int*>(col_nm)[3 * NQ + c] = p.causal ? min(place + 1, seg.len) : seg.len;
      reinterpret_cast<int*>(col_nm)[4 * NQ + c] = p.window >= 0 ? max(place - p.window, 0) : 0;
    }
  }
  ptx::fence_proxy_async_smem();
  __syncwarp();
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
    ptx::wait_for_previous_grid();
    if (threadIdx.x == 0) report_error(p.status, p.host_flag, kStatusSmemAlign);
    if (threadIdx.x < 2) p.share[(2 * blockIdx.x + threadIdx.x) * kShareInts] = -1;
    return;
  }
  // All CTAs of this launch are on the device at once, so the joining kernel's may take the
  // places that they leave, and wait there for the last.
  ptx::launch_dependents();
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = (int)(threadIdx.x & 31);
  constexpr int kWarpProd = C::kSoftWarps, kWarpMma = kWarpProd + 1, kWarpScale = kWarpProd + 2, kWarpQ = kWarpProd + 3;
  auto bar = [&](int slot) -> uint32_t { return sbase + C::kBars + slot * 8; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kMisc + 4);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kMisc);

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(bar(C::kKvFull + s), 1);
      ptx::mbar_init(bar(C::kKvEmpty + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(bar(C::kQFull + b), 1);
      ptx::mbar_init(bar(C::kQEmpty + b), 1);
      ptx::mbar_init(bar(C::kColEmpty + b), C::kSoftWarps);
      ptx::mbar_init(bar(C::kSFull + b), 1);
      ptx::mbar_init(bar(C::kSFree + b), C::kTileWarps);
      ptx::mbar_init(bar(C::kPFull + b), C::kTileWarps);
      ptx::mbar_init(bar(C::kPvDone + b), 1);
    }
    for (int s = 0; s < C::kScaleRing; ++s) {
      ptx::mbar_init(bar(C::kScFull + s), 1);
      ptx::mbar_init(bar(C::kScEmpty + s), C::kTileWarps);
    }
    for (int s = 0; s < C::kSegRing; ++s) {
      ptx::mbar_init(bar(C::kSegFull + s), 1);
      ptx::mbar_init(bar(C::kSegEmpty + s), C::kSoftWarps + 3);  // softmax, producer, MMA, query rows
    }
    ptx::mbar_init(bar(C::kDrain), 1);
    *abort_flag = 0;
    for (int k = 0; k < 8; ++k) reinterpret_cast<unsigned*>(smem + C::kBad)[k] = 0;
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
  // Launched while the kernel before may still run: up to here nothing of it was touched.
  ptx::wait_for_previous_grid();
  PagedStart start{};
  if (p.batch > kPagedWarpBatch)
    start = paged_start_cta<NQ>(p, reinterpret_cast<long long*>(smem + C::kScan),
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
  // Readers of the segment ring: every warp but the walking one (the scales').
  int seg_reads = 0;
  auto next_segment = [&](PagedSegment& seg) -> bool {
    const int at = seg_reads % C::kSegRing;
    wait(C::kSegFull + at, (uint32_t)(seg_reads / C::kSegRing));
    ++seg_reads;
    const int4* src = reinterpret_cast<const int4*>(smem + C::kSegs) + at * kSegVecs;
    int4 v[kSegVecs];
#pragma unroll
    for (int k = 0; k < kSegVecs; ++k) v[k] = src[k];
    seg = PagedSegment{v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w,
                       v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(C::kSegEmpty + at));
    return ok && seg.n >= 0;  // after a failed wait the ring may hold anything
  };
  PagedSegment seg{};

  if (warp < C::kSoftWarps) {
    // =========================================================== softmax ===
    const int wg = warp >> 2;
    const int t = (warp & 3) * 32 + lane;  // token of the tile; column of the head dim
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const int c_first = wg * NC;           // this warpgroup's query rows of the tile
    // The warps' maxima or sums of each query row (token-major), and by how much a row's maximum
    // moves. That has a place of its own: a warp may still read it while another, with no barrier
    // between, writes its sums at the segment's end or the maxima of the next move.
    float* const red = reinterpret_cast<float*>(smem + C::kRed) + wg * 5 * NC;
    float* const moved = red + 4 * NC;
    const float4* const scales = reinterpret_cast<const float4*>(smem + C::kScales);
    const int page = t >> p.block_shift;
    int g = 0;  // tiles so far
    uint32_t fills = 0;  // ring fills of the segments before
    auto split = [&](const PagedSegment& s, int n) {
      // All of a warp's loads at once: 32 / (D / 16) rows per step.
      constexpr int kSteps = NQ * (D / 16) / (32 * C::kSoftWarps);
      split_query_rows<T, D, NQ, (kSteps > 1 ? kSteps : 1)>(p, s, smem, n, warp, C::kSoftWarps);
      ptx::named_bar_sync(15, 32 * C::kSoftWarps);
      if (threadIdx.x == 0) ptx::mbar_arrive(bar(C::kQFull + (n & 1)));
    };
    // One answer for all softmax warps, or those that go on would miss the others at a barrier.
    auto next_for_all = [&](PagedSegment& s) {
      const bool more = next_segment(s);
      return !ptx::named_bar_or(15, 32 * C::kSoftWarps, !more);
    };
    // Before P V of tile j, the V rows that would carry NaN to rows that do not see their token
    // (0 * NaN): those of tokens that no row sees hold anything (NaN, an older tile) and are
    // cleared. Where some rows see a token and others do not, a V row with NaN in it is cleared
    // too, and the rows that see it get a weight of NaN instead: `poison(token)` writes this
    // thread's. Thread t of a tile's first warpgroup takes token t.
    unsigned* const bad_tokens = reinterpret_cast<unsigned*>(smem + C::kBad);  // [2 tiles][128 bits]
    auto clear_unseen = [&](int j, int tile_barrier, auto&& poison) {
      const int pos0 = (seg.tile + j) * kPagedTile, pos = pos0 + t;
      const bool uneven = (pos0 < seg.lo_all && seg.lo < seg.lo_all) ||
                          (pos0 + kPagedTile > seg.hi_all && seg.hi_all < seg.hi);
      if (!uneven && pos0 >= seg.lo && pos0 + kPagedTile <= seg.hi) return;
      const uint32_t fill = fills + min(seg.n, j + 1 + C::kLead) + j;  // V(j)'s place in the ring
      const int slot = (int)(fill % NS);
      wait(C::kKvFull + slot, fill / NS);
      unsigned* const bad = bad_tokens + (g & 1) * 4;
      const uint32_t row = sbase + slot * C::kSlotBytes + t * C::kRow;
      auto at = [&](int k) { return row + (k / C::kRow) * (kPagedTile * C::kRow) + k % C::kRow; };
      if ((wg & 1) == 0) {
        const bool unseen = pos < seg.lo || pos >= seg.hi;
        bool nan = false;
        if (uneven && !unseen) {
#pragma unroll 1
          for (int k = 0; k < D; k += 16) {
            const uint4 v = ptx::ld_shared_v4(at(k));
            // A byte of 7f or ff: its low seven bits carry when 1 is added.
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) nan |= (((w[x] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
          }
          if (nan) atomicOr(bad + (t >> 5), 1u << (t & 31));
        }
        if (unseen || nan) {
#pragma unroll 1
          for (int k = 0; k < D; k += 16) ptx::st_shared_v4(at(k), 0, 0, 0, 0);
        }
      }
      if (!uneven) return;
      ptx::named_bar_sync(tile_barrier, 32 * C::kTileWarps);
      if ((bad[0] | bad[1] | bad[2] | bad[3]) != 0) {
#pragma unroll 1
        for (int x = 0; x < kPagedTile; ++x)
          if (bad[x >> 5] >> (x & 31) & 1) poison(x);
        ptx::named_bar_sync(tile_barrier, 32 * C::kTileWarps);
        if ((wg & 1) == 0 && t < 4) bad[t] = 0;  // before this pair's next barrier
      }
    };
    bool more = next_for_all(seg);
    if constexpr (C::kQueryMajor) {
      // Thread: row `row` of the tile, tokens tok0 .. tok0 + kTok - 1 of the tiles of its pair; the warps
      // of a pair that share rows (one TMEM quarter's, or two with the same rows) agree on their maxima.
      constexpr int kWGs = C::kWG / C::kPairs;     // warpgroups per pair
      constexpr int kTok = C::kTok, kParts = C::kParts, kQuarters = 4 / C::kCopies;
      const int quarter = warp & 3, pair = wg / kWGs, rows_of = quarter % kQuarters;
      const int row = rows_of * 32 + lane, copy = quarter / kQuarters;
      const int tok0 = (wg % kWGs * C::kCopies + copy) * kTok;
      const int vote = 1 + pair * 4 + rows_of;     // barrier of the pair's warps that share the rows
      // What part k of a row's threads in pair q wrote to an exchange array at [wg * 128 + t].
      auto part_at = [&](int q, int k) { return (q * kWGs + k / C::kCopies) * 128 + k % C::kCopies * NQ + row; };
      // Exchange: maxima [2 tiles][kWG][128], sums [kWG][128], references [pairs][128].
      float* const exchange = reinterpret_cast<float*>(smem + C::kRed);
#pragma unroll 1
      for (int n = 0; more; ++n) {
        if (n == 0) split(seg, 0);
        const float qs = reinterpret_cast<const float*>(smem + C::kCol)[(n & 1) * 5 * NQ + NQ + row];
        int token, head;
        paged_row(p, seg.token0, seg.head0, row, token, head);
        const int place = seg.len - seg.nq + min(token, seg.nq - 1);
        const int hi = p.causal ? min(place + 1, seg.len) : seg.len;
        const int lo = p.window >= 0 ? max(place - p.window, 0) : 0;
        float nm = 0.f, l = 0.f;  // kPagedTop - max; the row's sum over this thread's tokens
        bool set = false, force = true;
        // Rows past the tile's last: nobody reads their S, weights or O.
        const bool idle = rows_of * 32 >= seg.rows;
#pragma unroll 1
        for (int j = 0; j < seg.n; ++j, ++g) {
          const int sb = g & 1;
          if (C::kPairs == 2 && sb != pair) continue;
          const int pos0 = (seg.tile + j) * kPagedTile;
          const bool masked = pos0 < seg.lo_all || pos0 + kPagedTile > seg.hi_all;
          wait(C::kScFull + g % C::kScaleRing, (uint32_t)(g / C::kScaleRing));
          const float4* const sc = scales + (g % C::kScaleRing) * 8;
          wait(C::kSFull + sb, (uint32_t)(g >> 1));
          ptx::tc_fence_after();
          float2 d[NC / 2];
          auto load = [&](int c0) {  // NC tokens' scores
            const uint32_t at = tmem + lane_off + (uint32_t)(sb * C::kSCols + c0);
#pragma unroll
            for (int c = 0; c < NC; c += 16) ptx::tmem_ld16(at + c, reinterpret_cast<uint32_t*>(d) + c);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < NC; c += 16) ptx::reg_fence16(reinterpret_cast<uint32_t*>(d) + c);
          };
          // d = x + log2 b - m; -inf where the row does not see the token.
          auto scaled = [&](int c0) {
#pragma unroll
            for (int half = 0; half < NC / 16; ++half) {
              const float4 s = sc[(c0 + 16 * half) >> p.block_shift];
              const float a = s.x * qs, b = s.y + nm;
              const float2 a2 = make_float2(a, a), b2 = make_float2(b, b);
#pragma unroll
              for (int c = 8 * half; c < 8 * half + 8; ++c) d[c] = __ffma2_rn(d[c], a2, b2);
            }
            if (masked) {
#pragma unroll
              for (int c = 0; c < NC; ++c) {
                const int pos = pos0 + c0 + c;
                if (pos < lo || pos >= hi) (c & 1 ? d[c / 2].y : d[c / 2].x) = -INFINITY;
              }
            }
          };
          // The P buffer was read by an earlier tile's P V.
          auto wait_p_buffer = [&]() {
            if (g >= C::kPBufs) wait(C::kPvDone + ((g - C::kPBufs) & 1), (uint32_t)((g - C::kPBufs) >> 1));
          };
          // S is read: the MMA warp may write the buffer again.
          auto release = [&]() {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(C::kSFree + sb));
          };
          if (idle) wait_p_buffer();  // (clear_unseen counts on it)
          if (!idle) {
            float most = -INFINITY;
#pragma unroll 1
            for (int c0 = 0; c0 < kTok; c0 += NC) {
              load(tok0 + c0);
              if (kTok == NC) release();
              scaled(tok0 + c0);
#pragma unroll
              for (int c = 0; c < NC / 2; ++c) most = ptx::fmax3(most, d[c].x, d[c].y);
            }
            const bool left = pos0 < seg.lo_all;
            const bool move = force || left ? true : ptx::named_bar_or(vote, 32 * kParts, most > kPagedMost);
            force = left;
            if (move) {
              float* const tops = exchange + ((g / C::kPairs) & 1) * C::kWG * 128;
              tops[wg * 128 + t] = most;
              ptx::named_bar_sync(vote, 32 * kParts);
              float top = most;
#pragma unroll
              for (int k = 0; k < kParts; ++k) top = fmaxf(top, tops[part_at(pair, k)]);
              // By how much the maximum moves: up only, but freely the first time.
              const bool some = top != -INFINITY;
              const float by = some ? (set ? fmaxf(top - kPagedTop, 0.f) : top - kPagedTop) : 0.f;
              const float f = set ? ptx::ex2(-by) : 0.f;
              set = set || some;
              nm -= by;
              l *= f;
              if (kTok == NC) {  // d is still here; else it is loaded again below
                const float2 by2 = make_float2(-by, -by);
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) d[c] = __fadd2_rn(d[c], by2);
              }
              if (j >= C::kPairs && copy == 0) {
                wait(C::kPvDone + ((g - C::kPairs) & 1), (uint32_t)((g - C::kPairs) >> 1));
                ptx::tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D / kWGs; c += 16) {
                  const uint32_t at = tmem + lane_off + (uint32_t)(2 * C::kSCols + pair * D + wg % kWGs * (D / kWGs) + c);
                  uint32_t v[16];
                  ptx::tmem_ld16(at, v);
                  ptx::tmem_wait_ld();
                  ptx::reg_fence16(v);
#pragma unroll
                  for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                  ptx::tmem_st16(at, v);
                }
                ptx::tmem_wait_st();
              }
            }
            wait_p_buffer();
            const uint32_t dst = sbase + C::kP + (C::kPBufs == 2 ? sb : 0) * C::kWTerms * C::kPTerm + row * 128;
#pragma unroll 1
            for (int c0 = 0; c0 < kTok; c0 += NC) {
              if (kTok > NC) {
                load(tok0 + c0);
                if (c0 + NC == kTok) release();
                scaled(tok0 + c0);
              }
#pragma unroll
              for (int half = 0; half < NC / 16; ++half) {
                const int c16 = tok0 + c0 + 16 * half;
                uint32_t term[C::kWTerms][4];
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int x = 8 * half + 2 * k;
                  const float2 e0 = make_float2(ptx::ex2(d[x].x), ptx::ex2(d[x].y));
                  const float2 e1 = make_float2(ptx::ex2(d[x + 1].x), ptx::ex2(d[x + 1].y));
                  sum = __fadd2_rn(sum, __fadd2_rn(e0, e1));
                  __half2 a = __floats2half2_rn(e0.x, e0.y), b = __floats2half2_rn(e1.x, e1.y);
                  uint32_t four[C::kWTerms];
                  split_weights(a, b, four);
#pragma unroll
                  for (int i = 0; i < C::kWTerms; ++i) term[i][k] = four[i];
                }
                l = fmaf(sum.x + sum.y, sc[c16 >> p.block_shift].z, l);
                const uint32_t unit = (uint32_t)((c16 >> 4) ^ (row & 7)) << 4;
#pragma unroll
                for (int i = 0; i < C::kWTerms; ++i)
                  ptx::st_shared_v4(dst + unit + i * C::kPTerm, term[i][0], term[i][1], term[i][2], term[i][3]);
              }
            }
          }
          if (idle) release();
          clear_unseen(j, 13 + pair, [&](int x) {
            const int pos = pos0 + x;
            if (!idle && x >= tok0 && x < tok0 + kTok && pos >= lo && pos < hi)
              ptx::st_shared_u8(sbase + C::kP + (C::kPBufs == 2 ? sb : 0) * C::kWTerms * C::kPTerm + row * 128 +
                                    (((x >> 4) ^ (row & 7)) << 4) + (x & 15), 0x7fu);
          });
          ptx::fence_proxy_async_smem();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(bar(C::kScEmpty + g % C::kScaleRing));
            ptx::mbar_arrive(bar(C::kPFull + sb));
          }
        }
        fills += 2 * seg.n;
        // The next segment's scores are under way while this one's result is written. (Q's buffer is
        // free: every S of this segment is here once all warps meet.)
        PagedSegment then;
        more = next_for_all(then);
        if (more) split(then, n + 1);

        // ---- the segment's result: this thread's row, a quarter of its columns ----
        float* const sums = exchange + 2 * C::kWG * 128;
        float* const refs = sums + C::kWG * 128;
        sums[wg * 128 + t] = l;
        if (wg % kWGs == 0) refs[pair * 128 + t] = set ? nm : INFINITY;
        ptx::named_bar_sync(9 + rows_of, 32 * C::kWG * C::kCopies);
        float ref = refs[row];
#pragma unroll
        for (int k = 1; k < C::kPairs; ++k) ref = fminf(ref, refs[k * 128 + row]);
        // o = (sum_k f_k O_k) / (sum_k f_k l_k) over the pairs, f_k = 2^(m_k - max m).
        float f[C::kPairs], sum = 0.f;
#pragma unroll
        for (int k = 0; k < C::kPairs; ++k) {
          const float mine = refs[k * 128 + row];
          f[k] = mine == INFINITY ? 0.f : ptx::ex2(ref - mine);
          float s = 0.f;
#pragma unroll
          for (int x = 0; x < kParts; ++x) s += sums[part_at(k, x)];
          sum = fmaf(f[k], s, sum);
        }
        const float inv = sum == 0.f ? 0.f : kPagedSumUnit / sum;
#pragma unroll
        for (int k = 0; k < C::kPairs; ++k) f[k] *= inv;
        const bool real = copy == 0 && row < seg.rows;
        if (wg == 0 && real) {
          const float lse2 = sum == 0.f ? -INFINITY : __log2f(sum) + (kPagedTop - ref);
          if (seg.slot >= 0)
            p.part_lse[(long long)seg.slot * NQ + t] = lse2;
          else if (p.lse != nullptr)
            p.lse[(long long)(seg.h * p.group + head) * p.total_q + seg.q0 + token] = lse2 * 0.69314718055994531f;
        }
#pragma unroll
        for (int k = 1; k <= C::kPairs; ++k)
          if (seg.n >= k) wait(C::kPvDone + ((g - k) & 1), (uint32_t)((g - k) >> 1));
        ptx::tc_fence_after();
        T* const o = static_cast<T*>(p.o) + (seg.q0 + token) * p.o_st + (seg.h * p.group + head) * p.o_sh;
        float* const part = p.part_o + ((long long)seg.slot * NQ + t) * D;
#pragma unroll 1
        for (int c = wg * (D / C::kWG); c < (wg + 1) * (D / C::kWG); c += 16) {
          float out[16];
#pragma unroll
          for (int k = 0; k < C::kPairs; ++k) {
            uint32_t v[16];
            ptx::tmem_ld16(tmem + lane_off + (uint32_t)(2 * C::kSCols + k * D + c), v);
            ptx::tmem_wait_ld();
            ptx::reg_fence16(v);
            // f = 0: the pair has nothing of this row, and TMEM may hold anything.
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const float y = f[k] == 0.f ? 0.f : __uint_as_float(v[x]) * f[k];
              out[x] = k == 0 ? y : out[x] + y;
            }
          }
          if (!real) continue;
          if (seg.slot >= 0) {
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              *reinterpret_cast<float4*>(part + c + k) = make_float4(out[k], out[k + 1], out[k + 2], out[k + 3]);
          } else {
            uint32_t pk[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) pk[k] = DType<T>::pack(out[2 * k], out[2 * k + 1]);
            *reinterpret_cast<uint4*>(o + c) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            *reinterpret_cast<uint4*>(o + c + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
          }
        }
        // Every warp has read its part of O before anyone's weights let the next P V write it.
        ptx::tc_fence_before();
        ptx::named_bar_sync(15, 32 * C::kSoftWarps);
        seg = then;
      }
    } else {
      // The first rows are split here in any case: these warps have nothing else to do yet.
#pragma unroll 1
      for (int n = 0; more; ++n) {
        const int rows = seg.rows - c_first;  // of this warpgroup; may be <= 0
        float* const col_nm = reinterpret_cast<float*>(smem + C::kCol) + (n & 1) * 5 * NQ + c_first;  // kPagedTop - max
        const float* const col_q = col_nm + NQ;  // q's scale
        float* const col_f = col_nm + 2 * NQ;    // factor of a moved maximum, -1 before the first; 1 / sum at the end
        const int* const col_hi = reinterpret_cast<const int*>(col_nm + 3 * NQ);  // tokens [lo, hi) are seen
        const int* const col_lo = reinterpret_cast<const int*>(col_nm + 4 * NQ);
        if (n == 0) split(seg, 0);
        wait(C::kQFull + (n & 1), (uint32_t)(n >> 1));
        float2 l[NC / 2];
#pragma unroll
        for (int c = 0; c < NC / 2; ++c) l[c] = make_float2(0.f, 0.f);
        bool force = true;  // a row's maximum may not be set: first tile, or behind one left of a row's window

#pragma unroll 1
        for (int j = 0; j < seg.n; ++j, ++g) {
          const int sb = g & 1;
          const int pos0 = (seg.tile + j) * kPagedTile, pos = pos0 + t;
          wait(C::kScFull + g % C::kScaleRing, (uint32_t)(g / C::kScaleRing));
          const float4 sc = scales[(g % C::kScaleRing) * 8 + page];  // a * scale_log2, log2 b, 2^-13 / b
          wait(C::kSFull + sb, (uint32_t)(g >> 1));
          ptx::tc_fence_after();
          float2 d[NC / 2];
#pragma unroll
          for (int c = 0; c < NC; c += 16)
            ptx::tmem_ld16(tmem + lane_off + (uint32_t)(sb * NQ + c_first + c), reinterpret_cast<uint32_t*>(d) + c);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < NC; c += 16) ptx::reg_fence16(reinterpret_cast<uint32_t*>(d) + c);
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(bar(C::kScEmpty + g % C::kScaleRing));
            ptx::mbar_arrive(bar(C::kSFree + sb));
          }
          // d = x + log2 b - m; -inf where the row does not see the token.
          const float2 a2 = make_float2(sc.x, sc.x), b2 = make_float2(sc.y, sc.y), i2 = make_float2(sc.z, sc.z);
          float most = -INFINITY;
#pragma unroll
          for (int c = 0; c < NC / 2; c += 2) {
            const float4 q4 = *reinterpret_cast<const float4*>(col_q + 2 * c);
            const float4 n4 = *reinterpret_cast<const float4*>(col_nm + 2 * c);
            d[c] = __ffma2_rn(d[c], __fmul2_rn(a2, make_float2(q4.x, q4.y)), __fadd2_rn(b2, make_float2(n4.x, n4.y)));
            d[c + 1] =
                __ffma2_rn(d[c + 1], __fmul2_rn(a2, make_float2(q4.z, q4.w)), __fadd2_rn(b2, make_float2(n4.z, n4.w)));
            most = ptx::fmax3(most, d[c].x, d[c].y);
            most = ptx::fmax3(most, d[c + 1].x, d[c + 1].y);
          }
          const bool masked = pos0 < seg.lo_all || pos0 + kPagedTile > seg.hi_all;
          if (masked) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
              if (pos < col_lo[c] || pos >= col_hi[c]) (c & 1 ? d[c / 2].y : d[c / 2].x) = -INFINITY;
            // What nobody sees has no say in where the maxima move: not one bit of the result is its.
            most = -INFINITY;
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) most = ptx::fmax3(most, d[c].x, d[c].y);
          }
          const bool left = pos0 < seg.lo_all;
          const bool move = force || left ? true : ptx::named_bar_or(1 + wg, 128, most > kPagedMost);
          force = left;
          if (move) {
            // Move the maxima: over the warp, over the warps; then rescale the sums and O.
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const float top = ptx::warp_max(c & 1 ? d[c / 2].y : d[c / 2].x);
              if (lane == c) red[(warp & 3) * NC + c] = top;
            }
            ptx::named_bar_sync(1 + wg, 128);
            if (t < NC) {
              const float top = fmaxf(fmaxf(red[t], red[NC + t]), fmaxf(red[2 * NC + t], red[3 * NC + t]));
              // By how much the maximum moves: up only, but freely the first time.
              const bool set = col_f[t] >= 0.f;
              const float by = top == -INFINITY ? 0.f : (set ? fmaxf(top - kPagedTop, 0.f) : top - kPagedTop);
              if (set || top != -INFINITY) col_f[t] = set ? ptx::ex2(-by) : 0.f;
              col_nm[t] -= by;
              moved[t] = by;
            }
            ptx::named_bar_sync(1 + wg, 128);
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) {
              const float2 by = *reinterpret_cast<const float2*>(moved + 2 * c);
              d[c] = make_float2(d[c].x - by.x, d[c].y - by.y);
              l[c] = __fmul2_rn(l[c], *reinterpret_cast<const float2*>(col_f + 2 * c));
            }
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
          const uint32_t dst = sbase + C::kP + sb * C::kWTerms * C::kPTerm + t * 16 + c_first * 128;
#pragma unroll
          for (int c = 0; c < NC; c += 16) {
            uint32_t term[C::kWTerms][4];
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const int x = (c + k) / 2;
              const float2 e0 = make_float2(ptx::ex2(d[x].x), ptx::ex2(d[x].y));
              const float2 e1 = make_float2(ptx::ex2(d[x + 1].x), ptx::ex2(d[x + 1].y));
              l[x] = __ffma2_rn(e0, i2, l[x]);
              l[x + 1] = __ffma2_rn(e1, i2, l[x + 1]);
              __half2 a = __floats2half2_rn(e0.x, e0.y), b = __floats2half2_rn(e1.x, e1.y);
              uint32_t four[C::kWTerms];
              split_weights(a, b, four);
#pragma unroll
              for (int j2 = 0; j2 < C::kWTerms; ++j2) term[j2][k >> 2] = four[j2];
            }
#pragma unroll
            for (int j2 = 0; j2 < C::kWTerms; ++j2)
              ptx::st_shared_v4(dst + c * 128 + j2 * C::kPTerm, term[j2][0], term[j2][1], term[j2][2], term[j2][3]);
          }
          clear_unseen(j, 1 + wg, [&](int x) {  // columns 16-byte chunk by chunk, tokens within
            if (x != t) return;
            for (int c = 0; c < NC; ++c)
              if (pos >= col_lo[c] && pos < col_hi[c]) ptx::st_shared_u8(dst + (c >> 4) * 2048 + (c & 15), 0x7fu);
          });
          ptx::fence_proxy_async_smem();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(C::kPFull + sb));
        }
        fills += 2 * seg.n;

        // ---- the segment's result ----
        {
          float sums[NC];
#pragma unroll
          for (int c = 0; c < NC / 2; ++c) sums[2 * c] = l[c].x, sums[2 * c + 1] = l[c].y;
          const int c = warp_column_sums<NC>(sums);
          if (NC == 32 || (lane & 1) == 0) red[(warp & 3) * NC + c] = sums[0];
        }
        ptx::named_bar_sync(1 + wg, 128);
        if (t < NC && t < rows) {
          const float sum = red[t] + red[NC + t] + red[2 * NC + t] + red[3 * NC + t];
          const float lse2 = sum == 0.f ? -INFINITY : __log2f(sum) + (kPagedTop - col_nm[t]);
          col_f[t] = sum == 0.f ? 0.f : kPagedSumUnit / sum;
          if (seg.slot >= 0) {
            p.part_lse[(long long)seg.slot * NQ + c_first + t] = lse2;
          } else if (p.lse != nullptr) {
            int token, head;
            paged_row(p, seg.token0, seg.head0, c_first + t, token, head);
            p.lse[(long long)(seg.h * p.group + head) * p.total_q + seg.q0 + token] = lse2 * 0.69314718055994531f;
          }
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
            int token, head;
            paged_row(p, seg.token0, seg.head0, c_first + c, token, head);
            T* o = static_cast<T*>(p.o) + (seg.q0 + token) * p.o_st + (seg.h * p.group + head) * p.o_sh + d;
            float* part = p.part_o + ((long long)seg.slot * NQ + c_first + c) * D + d;
            const long long wrap = p.o_st - (p.group - 1) * p.o_sh;  // from a token's last head to the next's first
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (c + k >= rows) break;
              const float inv = col_f[c + k];
              // A row that saw nothing has no O (its tiles may not have run): 0, whatever TMEM holds.
              const float val = inv == 0.f ? 0.f : __uint_as_float(v[k]) * inv;
              if (d < D) {
                if (seg.slot >= 0) part[k * D] = val;
                else *o = (T)val;
              }
              const bool last = ++head == p.group;
              o += last ? wrap : p.o_sh;
              head = last ? 0 : head;
            }
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(C::kColEmpty + (n & 1)));
        more = next_for_all(seg);
      }
    }
  } else if (warp == kWarpProd) {
    // ========================================================== producer ===
    // Ring order per segment: K(0 .. kLead - 1); then K(j + kLead), V(j) for each j: the MMA warp's.
    // Lane i copies page i of a tile; pages that no row sees are left out.
    const uint64_t policy = p.one_tile ? ptx::policy_evict_first() : ptx::policy_evict_last();
    const int pages = kPagedTile >> p.block_shift;
    uint32_t fills = 0;
    // Block ids of four tiles at a time, one batch ahead: lane 8 i + k holds page k of the i-th.
    // -2: not loaded; -1: outside the cache, reads as zeros.
    auto page_ids = [&](const PagedSegment& s, int tile) -> int {
      const int at = (tile + (lane >> 3)) * kPagedTile + ((lane & 7) << p.block_shift);
      if ((lane & 7) >= pages || at >= s.hi || at + (1 << p.block_shift) <= s.lo) return -2;
      const int id = read_input(p.block_table + (long long)s.b * p.table_stride + (at >> p.block_shift));
      return id >= 0 && id < p.num_blocks ? id : -1;
    };
    // The next K tile, V tile or both, from the block ids in lanes 0 .. pages - 1 and V's in lanes
    // 16 on. One wait, one announcement and one run of copies for both, where the ring is long enough
    // for the next K not to wait for a free V place: apart, a fill of four blocks took this warp
    // 1150 cycles, and the card's memory brings one in 700. (Measured with five slots: 83 -> 77 us
    // for 48 ragged requests; with three, 32 requests of 40 rows at d = 256, it would be 48 -> 52.)
    auto fill = [&](bool k, bool v, int ids) {  // `seg`'s head
      const bool second = lane >= 16;
      const uint32_t mine = fills + (k && v && second ? 1 : 0);
      const int slot = (int)(mine % NS);
      wait(C::kKvEmpty + slot, (mine / NS) ^ 1u);
      const uint32_t full = bar(C::kKvFull + slot);
      const unsigned boxes = __ballot_sync(0xffffffffu, ids > -2);
      if (ok) {
        if (lane == 0 ? k : lane == 16 && v)
          ptx::mbar_arrive_expect_tx(full, (uint32_t)(__popc(second ? boxes >> 16 : boxes & 0xffffu) * D) << p.block_shift);
        __syncwarp();
        if (ids > -2) {
          const CUtensorMap* const map = second ? &tmV : &tmK;
          const uint32_t dst = sbase + slot * C::kSlotBytes + ((uint32_t)((lane & 7) << p.block_shift) * C::kRow);
#pragma unroll
          for (int ch = 0; ch < C::kChunks; ++ch)
            ptx::tma_load_4d(dst + ch * (kPagedTile * C::kRow), map, full, ch * 128, 0, seg.h, ids, policy);
        }
        fills += (k ? 1 : 0) + (v ? 1 : 0);
      }
      __syncwarp();
    };
    // The next segment and its first block ids are looked up while the ring is full of this one.
    bool more = next_segment(seg);
    int ids = -2, ahead = -2;
    if (more) {
      ids = page_ids(seg, seg.tile);
      ahead = page_ids(seg, seg.tile + 4);
    }
    while (more) {
      PagedSegment then;
      int then_ids = -2, then_ahead = -2;
      auto look = [&]() {
        more = next_segment(then);
        if (more) {
          then_ids = page_ids(then, then.tile);
          then_ahead = page_ids(then, then.tile + 4);
        }
      };
      auto pick = [&](int j) {  // tile j's ids, page k in lane k
        const int id = __shfl_sync(0xffffffffu, ids, ((j & 3) << 3) + (lane & 7));
        return lane < 8 ? id : -2;
      };
      // Tiles' ids in fill order: K runs kLead tiles ahead of V.
      if (seg.n == 0) look();
      int behind[C::kLead];
#pragma unroll
      for (int k = 0; k < C::kLead; ++k) {
        behind[k] = k < seg.n ? pick(k) : -2;
        if (k < seg.n) fill(true, false, behind[k]);
      }
#pragma unroll 1
      for (int j = 0; j < seg.n; ++j) {
        const int ahead_tile = j + C::kLead;
        int next = -2;
        if (ahead_tile < seg.n) {
          if ((ahead_tile & 3) == 0) {
            ids = ahead;
            ahead = page_ids(seg, seg.tile + ahead_tile + 4);
          }
          next = pick(ahead_tile);
        }
        const int v_ids = __shfl_sync(0xffffffffu, behind[0], lane & 7);  // to lanes 16 .. 23
        const bool k = ahead_tile < seg.n;
        if (k && NS < 5) fill(true, false, next);
        fill(k && NS >= 5, true, lane < 8 && NS >= 5 ? next : lane >= 16 && lane < 24 ? v_ids : -2);
#pragma unroll
        for (int k = 0; k + 1 < C::kLead; ++k) behind[k] = behind[k + 1];
        behind[C::kLead - 1] = next;
        if (j == 0) look();
      }
      seg = then;
      ids = then_ids;
      ahead = then_ahead;
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
    // 8 bits, fp32 sums, M = 128. S: both operands K-major. P V: V is always MN-major; the weights
    // are MN-major as the B operand (token-major), K-major as the A operand (query-major).
    constexpr uint32_t kDesc = (1u << 4) | ((uint32_t)(128 >> 4) << 24);
    constexpr uint32_t idS = kDesc | ((uint32_t)(C::kSCols >> 3) << 17);
    // The operand that is split (query-major A, token-major B) is e5m2 where it is a weight, or the third
    // term of q.
    constexpr uint32_t kE5m2 = 1u << (C::kQueryMajor ? 7 : 10);
    constexpr uint32_t idPV = kE5m2 | (C::kQueryMajor ? kDesc | (1u << 16) | ((uint32_t)(D >> 3) << 17)
                                                      : kDesc | (1u << 15) | (1u << 16) | ((uint32_t)(NQ >> 3) << 17));
    int gs = 0, gp = 0;  // S and P V tiles issued
    auto acquire = [&](uint32_t fill) -> int {
      const int slot = (int)(fill % NS);
      wait(C::kKvFull + slot, fill / NS);
      return slot;
    };
    int n = 0;  // segments so far
    auto issue_S = [&](uint32_t fill, bool last) {
      const int sb = gs & 1;
      if (gs >= 2) wait(C::kSFree + sb, (uint32_t)((gs >> 1) - 1));
      const int slot = acquire(fill);
      ptx::tc_fence_after();
      if (ok) {
        uint32_t acc = 0;
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
          for (int ks = 0; ks < C::kRow / 32; ++ks) {
            const uint64_t k = ptx::smem_desc(sbase + slot * C::kSlotBytes + ch * (kPagedTile * C::kRow) + ks * 32, 16,
                                              8 * C::kRow, C::kSwizzle);
#pragma unroll
            for (int j = 0; j < C::kQTerms; ++j) {
              const uint32_t rows = sbase + C::kQ + (n % C::kQBufs) * C::kQBytes + j * C::kCopies * NQ * D;
              const uint32_t dS = tmem + (uint32_t)(sb * C::kSCols);
              if constexpr (C::kQueryMajor) {
                const uint64_t q = ptx::smem_desc(rows + ch * (C::kCopies * NQ * C::kRow) + ks * 32, 16,
                                                  8 * C::kRow, C::kSwizzle);
                ptx::umma_ss_f8_warp(dS, q, k, j == 2 ? idS | kE5m2 : idS, acc);
              } else {
                const uint64_t q = ptx::smem_desc(rows + (ch * (C::kRow / 16) + 2 * ks) * (NQ * 16), NQ * 16, 128, 0);
                ptx::umma_ss_f8_warp(dS, k, q, j == 2 ? idS | kE5m2 : idS, acc);
              }
              acc = 1;
            }
          }
        ptx::tc_commit_warp(bar(C::kKvEmpty + slot));
        ptx::tc_commit_warp(bar(C::kSFull + sb));
        if (!C::kQueryMajor && last) ptx::tc_commit_warp(bar(C::kQEmpty + n % C::kQBufs));
      }
      ++gs;
    };
    auto issue_PV = [&](uint32_t fill, bool first) {
      const int sb = gp & 1;
      wait(C::kPFull + sb, (uint32_t)(gp >> 1));
      const int slot = acquire(fill);
      ptx::tc_fence_after();
      if (ok) {
        const uint32_t weights = sbase + C::kP + (C::kPBufs == 2 ? sb : 0) * C::kWTerms * C::kPTerm;
        const uint32_t dO = tmem + (uint32_t)(2 * C::kSCols + (C::kPairs == 2 ? sb * D : 0));
        if constexpr (C::kQueryMajor) {
#pragma unroll
          for (int ks = 0; ks < kPagedTile / 32; ++ks) {
            const uint64_t v = ptx::smem_desc(sbase + slot * C::kSlotBytes + ks * 32 * C::kRow, kPagedTile * C::kRow,
                                              8 * C::kRow, C::kSwizzle);
#pragma unroll
            for (int j = 0; j < C::kWTerms; ++j) {
              const uint64_t w = ptx::smem_desc(weights + j * C::kPTerm + ks * 32, 16, 1024, 2);
              ptx::umma_ss_f8_warp(dO, w, v, idPV, first && ks == 0 && j == 0 ? 0u : 1u);
            }
          }
        } else {
#pragma unroll
          for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
            for (int ks = 0; ks < kPagedTile / 32; ++ks) {
              // d = 64: the second 64 rows of M repeat the first (zero stride); nobody reads them.
              const uint64_t v = ptx::smem_desc(
                  sbase + slot * C::kSlotBytes + ch * (kPagedTile * C::kRow) + ks * 32 * C::kRow, 0, 8 * C::kRow,
                  C::kSwizzle);
#pragma unroll
              for (int j = 0; j < C::kWTerms; ++j) {
                const uint64_t w = ptx::smem_desc(weights + j * C::kPTerm + ks * 32 * 16, 128, 2048, 0);
                ptx::umma_ss_f8_warp(dO + (uint32_t)(ch * NQ), v, w, idPV, first && ks == 0 && j == 0 ? 0u : 1u);
              }
            }
        }
        ptx::tc_commit_warp(bar(C::kKvEmpty + slot));
        ptx::tc_commit_warp(bar(C::kPvDone + sb));
      }
      ++gp;
    };
    uint32_t fills = 0;  // of the segments before
    for (; next_segment(seg); ++n) {
      // Places in the ring as the producer fills it.
      auto k_at = [&](int j) { return fills + j + max(0, j - C::kLead); };
      auto v_at = [&](int j) { return fills + j + min(seg.n, j + 1 + C::kLead); };
      wait(C::kQFull + (n & 1), (uint32_t)(n >> 1));
      if (!C::kQueryMajor && seg.n == 0 && lane == 0) ptx::mbar_arrive(bar(C::kQEmpty + n % C::kQBufs));
#pragma unroll 1
      for (int j = 0; j < min(seg.n, C::kLead); ++j) issue_S(k_at(j), j + 1 == seg.n);
#pragma unroll 1
      for (int j = 0; j < seg.n; ++j) {
        const int next = j + C::kLead;
        if (next < seg.n) issue_S(k_at(next), next + 1 == seg.n);
        issue_PV(v_at(j), j < C::kPairs);
      }
      fills += 2 * seg.n;
    }
    ptx::tc_commit_warp(bar(C::kDrain));
    if (lane == 0) drain_wait(bar(C::kDrain), 0, p.timeout_ns, p.status, p.host_flag);
    __syncwarp();
  } else if (warp == kWarpScale) {
    // ============================================================ scales ===
    // Ahead of the softmax: per tile and page, a * sm_scale * log2 e, log2 b and 2^-13 / b.
    // Four tiles' loads at a time: lane 8 i + k looks after page k of the i-th.
    const int pages = kPagedTile >> p.block_shift;
    float4* const scales = reinterpret_cast<float4*>(smem + C::kScales);
    if (p.batch <= kPagedWarpBatch) start = paged_start_warp<NQ>(p);
    PagedWalk<NQ> walk(p, start);
    int published = 0;
    auto publish = [&](const PagedSegment& x) {
      const int at = published % C::kSegRing;
      wait(C::kSegEmpty + at, (uint32_t)(published / C::kSegRing) ^ 1u);
      ++published;
      int4* dst = reinterpret_cast<int4*>(smem + C::kSegs) + at * kSegVecs;
      if (lane == 0) {
        dst[0] = make_int4(x.b, x.h, x.q0, x.nq);
        dst[1] = make_int4(x.len, x.lo, x.hi, x.tile);
        dst[2] = make_int4(x.n, x.slot, x.rows, x.token0);
        dst[3] = make_int4(x.head0, x.lo_all, x.hi_all, 0);
        ptx::mbar_arrive(bar(C::kSegFull + at));
      }
      __syncwarp();
    };
    int g = 0;
    seg = walk.next();
    publish(seg);
    walk.share_out(seg);
    while (seg.n >= 0) {
      // One segment ahead of its scales, so that the other roles can look ahead too.
      const PagedSegment then = walk.next();
      publish(then);
      walk.share_out(then);
#pragma unroll 1
      for (int j0 = 0; j0 < seg.n; j0 += 4) {
        const int j = j0 + (lane >> 3), page = lane & 7;
        const int at = (seg.tile + j) * kPagedTile + (page << p.block_shift);
        // Pages that are not there: zero scores and values, and a V scale too small to move a maximum.
        float4 sc = make_float4(0.f, -100.f, kPagedSumUnit / kPagedLeastScale, 0.f);
        if (j < seg.n && page < pages && at < seg.hi && at + (1 << p.block_shift) > seg.lo) {
          const int id = read_input(p.block_table + (long long)seg.b * p.table_stride + (at >> p.block_shift));
          if (id >= 0 && id < p.num_blocks) {
            const float a = read_input(p.k_scale + (long long)id * p.heads_kv + seg.h);
            const float given = read_input(p.v_scale + (long long)id * p.heads_kv + seg.h);
            const float b = fmaxf(given, kPagedLeastScale);
            // A scale of NaN goes on in the exponent, which is masked; b is not, and stays a number.
            sc = make_float4(a * p.scale_log2, given != given ? given : __log2f(b), kPagedSumUnit / b, 0.f);
          }
        }
        const int take = min(4, seg.n - j0);
#pragma unroll 1
        for (int i = 0; i < take; ++i, ++g) {
          wait(C::kScEmpty + g % C::kScaleRing, (uint32_t)(g / C::kScaleRing) ^ 1u);
          if ((lane >> 3) == i) scales[(g % C::kScaleRing) * 8 + page] = sc;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(C::kScFull + g % C::kScaleRing));
        }
      }
      seg = then;
      if (!ok) break;
    }
    if (p.zero_rest) {
      // Rows of o outside every request. Those in front of the first and behind the last (a padded
      // step has them) are shared out over the CTAs: cleared by one warp, 64 rows of 32 heads of 128
      // take 120 us; by all, 4096 rows take 2 to 7. Others, which only offsets that leave rows out have,
      // go by request.
      const int heads = p.heads_kv * p.group;
      auto clear = [&](int from, int to, int step) {
#pragma unroll 1
        for (long long row = from; row < to; row += step) {
          T* const o = static_cast<T*>(p.o) + row * p.o_st;
#pragma unroll 1
          for (int x = lane; x < heads * (D / 8); x += 32) {
            const int hq = x / (D / 8), d = x % (D / 8) * 8;
            *reinterpret_cast<uint4*>(o + hq * p.o_sh + d) = make_uint4(0, 0, 0, 0);
            if (p.lse != nullptr && d == 0) p.lse[(long long)hq * p.total_q + row] = 0.f;
          }
        }
      };
      const PagedRequest last = paged_request(p, p.batch - 1);
      clear((int)blockIdx.x, paged_request(p, 0).q0, (int)gridDim.x);
      clear(last.q0 + last.nq + (int)blockIdx.x, p.total_q, (int)gridDim.x);
      for (int b = (int)blockIdx.x; b + 1 < p.batch; b += gridDim.x) {
        const PagedRequest r = paged_request(p, b);
        clear(r.q0 + r.nq, paged_request(p, b + 1).q0, 1);
      }
    }
  } else if (warp == kWarpQ) {
    // ======================================================== query rows ===
    // Ahead of the softmax, from the second segment on.
    for (int n = 0; next_segment(seg); ++n) {
      if (n == 0 || C::kSelfSplit) continue;
      if (n >= C::kQBufs) wait(C::kQEmpty + n % C::kQBufs, (uint32_t)(n / C::kQBufs - 1));
      if (n >= 2) wait(C::kColEmpty + (n & 1), (uint32_t)((n >> 1) - 1));
      split_query_rows<T, D, NQ, 4>(p, seg, smem, n, 0, 1);
      if (lane == 0) ptx::mbar_arrive(bar(C::kQFull + (n & 1)));
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the parts of the items that several CTAs shared: o = sum_k w_k o_k / sum_k w_k with
// w_k = 2^(lse_k - max lse), in the CTAs' order. The CTAs c0 .. c1 of an item share its rows out.
// Bound: latency (three dependent loads). Few parts: a thread takes four columns of a row, so
// that all its loads are under way at once. Many: a CTA takes a row, each warp a share of the
// parts.
constexpr int kCombineThreads = 256;
constexpr int kCombineFew = 4;

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(kCombineThreads) attn_paged_combine_kernel(const PagedParams p) {
  constexpr int kWarps = kCombineThreads / 32, E = D / 32;
  __shared__ float part[kWarps][D];
  __shared__ float stat[kWarps][2];
  ptx::launch_dependents();
  ptx::wait_for_previous_grid();
  const int4* const share = reinterpret_cast<const int4*>(p.share + 2 * blockIdx.x * kShareInts);
  const int4 entry[4] = {share[0], share[1], share[2], share[3]};
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int4 item = side ? entry[2] : entry[0], ctas = side ? entry[3] : entry[1];
    if (item.x < 0) continue;
    const int h = item.y, rows = item.z, c0 = ctas.x, k_parts = ctas.y - ctas.x + 1;
    // Part k is CTA c0 + k's: the first left it behind, the others got it from before.
    auto slot = [&](int k, int c) { return (long long)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * NQ + c; };
    auto out = [&](int c, int d, long long& lse_at) {
      int i, hq;
      paged_row(p, item.w, ctas.z, c, i, hq);
      i += item.x;
      hq += h * p.group;
      lse_at = (long long)hq * p.total_q + i;
      return static_cast<T*>(p.o) + i * p.o_st + hq * p.o_sh + d;
    };
    auto put_lse = [&](long long at, float m, float sum) {
      if (p.lse != nullptr) p.lse[at] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.69314718055994531f;
    };
    if (k_parts <= kCombineFew) {
      constexpr int kQuads = D / 4;  // threads per row
      for (int x = ((int)blockIdx.x - c0) * kCombineThreads + (int)threadIdx.x; x < rows * kQuads;
           x += k_parts * kCombineThreads) {
        const int c = x / kQuads, d = x % kQuads * 4;
        float lse[kCombineFew], m = -INFINITY, sum = 0.f;
        float4 o[kCombineFew];
#pragma unroll
        for (int k = 0; k < kCombineFew; ++k) {
          lse[k] = -INFINITY;
          if (k < k_parts) {
            lse[k] = p.part_lse[slot(k, c)];
            o[k] = *reinterpret_cast<const float4*>(p.part_o + slot(k, c) * D + d);
          }
        }
#pragma unroll
        for (int k = 0; k < kCombineFew; ++k) m = fmaxf(m, lse[k]);
        const float base = m == -INFINITY ? 0.f : m;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kCombineFew; ++k) {
          if (k < k_parts) {
            const float w = ptx::ex2(lse[k] - base);
            sum += w;
            acc = make_float4(fmaf(w, o[k].x, acc.x), fmaf(w, o[k].y, acc.y), fmaf(w, o[k].z, acc.z),
                              fmaf(w, o[k].w, acc.w));
          }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        long long lse_at;
        T* to = out(c, d, lse_at);
        *reinterpret_cast<uint2*>(to) = make_uint2(DType<T>::pack(acc.x * inv, acc.y * inv),
                                                   DType<T>::pack(acc.z * inv, acc.w * inv));
        if (d == 0) put_lse(lse_at, m, sum);
      }
      continue;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c = (int)blockIdx.x - c0; c < rows; c += k_parts) {
      float m = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int k = warp + lane * kWarps; k < k_parts; k += 32 * kWarps) m = fmaxf(m, p.part_lse[slot(k, c)]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
      for (int k = warp; k < k_parts; k += kWarps) {
        const float w = ptx::ex2(p.part_lse[slot(k, c)] - base);
        const float* o = p.part_o + slot(k, c) * D + lane * E;
        sum += w;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(o + e);
          acc[e] = fmaf(w, v.x, acc[e]);
          acc[e + 1] = fmaf(w, v.y, acc[e + 1]);
        }
      }
      if (lane == 0) {
        stat[warp][0] = m;
        stat[warp][1] = sum;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) part[warp][lane * E + e] = acc[e];
      __syncthreads();
      if (threadIdx.x < D / 2) {
        float all = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all = fmaxf(all, stat[w][0]);
        const float base_all = all == -INFINITY ? 0.f : all;
        const int d = 2 * threadIdx.x;
        float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ptx::ex2(stat[w][0] - base_all);  // a warp without parts has -inf: 0
          total = fmaf(f, stat[w][1], total);
          x = fmaf(f, part[w][d], x);
          y = fmaf(f, part[w][d + 1], y);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        long long lse_at;
        *reinterpret_cast<uint32_t*>(out(c, d, lse_at)) = DType<T>::pack(x * inv, y * inv);
        if (d == 0) put_lse(lse_at, all, total);
      }
      __syncthreads();
    }
  }
}

}  // namespace apex
