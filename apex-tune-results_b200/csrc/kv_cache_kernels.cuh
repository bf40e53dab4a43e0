// Kernels that keep a paged 8-bit K/V cache: block bookkeeping (kv_plan, kv_release) and the
// write of new tokens (kv_append). The attention that reads the cache is in
// attn_paged_kernel.cuh.
//
// The cache holds e4m3 codes [num_blocks, H_kv, block, D] and one fp32 scale per (block,
// K/V head); a value is code * scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace apex {

// ------------------------------------------------------------------ bookkeeping --
constexpr int kPlanMaxBatch = 8192;  // the prefix sums of a call live in one CTA's shared memory

struct PlanParams {
  int* block_table;  // [batch, table_width], row stride table_stride
  long long table_stride;
  const int* seq_lens;  // tokens each request holds before the call
  const int* new_lens;  // plan: tokens to place; release: non-zero where the request is finished
  int* free_blocks;     // stack of free block ids, the top at free_count - 1
  const int* free_count;
  long long* slots;  // plan: [max_new] slot of each new token, -1 where it has none
  int* cu_seqlens;   // plan: [batch + 1] offsets of the requests' new tokens
  int* seq_lens_out;
  int* free_count_out;
  int* placed;  // plan: [batch] 1 where the request got its blocks
  int batch, table_width, free_capacity, block_shift, max_new;
};

// Inclusive sum over the CTA's threads; `total` is the sum of all. `warp_sums` holds one
// value per warp; the barriers also order its reuse.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* warp_sums, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  V s = lane < warps ? warp_sums[lane] : V(0);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += up;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const V before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
  return warp > 0 ? v + before : v;
}

// The last index i of the nondecreasing a[0 .. n) with a[i] <= x (a[0] <= x).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;  // a[lo] <= x < a[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One scheduling step: request b (holding len_b tokens in ceil(len_b / block) blocks) gets
// need_b = ceil((len_b + new_b) / block) - ceil(len_b / block) blocks, popped from the stack
// in request order: entry e of all needs together (base_b <= e < base_b + need_b, base the
// exclusive prefix sum) is free_blocks[count - 1 - e]. A request is placed if its blocks fit
// its table row, its tokens the slot array, and the stack holds what it and all before it
// need; one that is not placed keeps its length and gets slots of -1.
//
// Bound: latency (a few KB move). Every CTA computes the prefix sums of all requests by
// itself (two block scans over at most 8192 lengths that sit in the L2), so no CTA waits for
// another and one launch does; then table entries and slots are spread over all threads, each
// finding its request by bisection in shared memory. CTA 0 writes the per-request results.
__global__ void __launch_bounds__(1024) kv_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;              // [batch + 1]
  int* base = cu + p.batch + 1;     // [batch]
  int* len = base + p.batch;        // [batch], -1 - len where the request is not placed
  __shared__ long long sums64[32];
  __shared__ int popped_s;
  const int block = 1 << p.block_shift;
  const int count = min(max(__ldg(p.free_count), 0), p.free_capacity);
  const bool writer = blockIdx.x == 0;
  if (threadIdx.x == 0) popped_s = 0;
  long long cu_carry = 0;
  int base_carry = 0;  // saturates above free_capacity, where no request is placed any more
  int popped = 0;
  for (int b0 = 0; b0 < p.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const bool in = b < p.batch;
    const int held = in ? max(__ldg(p.seq_lens + b), 0) : 0;
    const int fresh = in ? max(__ldg(p.new_lens + b), 0) : 0;
    long long total64;
    const long long end = cu_carry + block_scan<long long>(fresh, sums64, total64);
    const long long after = (long long)held + fresh;
    const int have = (int)(((long long)held + block - 1) >> p.block_shift);
    const long long want = (after + block - 1) >> p.block_shift;
    const bool fits = want <= p.table_width && end <= p.max_new;
    // A need above the whole stack counts as one above it, so that the sums stay in range.
    const int need = fits ? (int)min(want - have, (long long)p.free_capacity + 1) : 0;
    long long total_need;
    const long long need_end = (long long)base_carry + block_scan<long long>(need, sums64, total_need);
    const bool placed = fits && (need == 0 || need_end <= count);
    if (in) {
      const long long begin = end - fresh;
      cu[b] = (int)min(begin, (long long)0x7fffffff);
      base[b] = (int)min(need_end - need, (long long)0x7fffffff);
      len[b] = placed ? held : -1 - held;
      if (placed && need > 0) popped = max(popped, (int)need_end);
      if (writer) {
        p.cu_seqlens[b] = cu[b];
        p.seq_lens_out[b] = placed ? held + fresh : held;
        p.placed[b] = placed ? 1 : 0;
      }
    }
    cu_carry += total64;
    base_carry = (int)min((long long)base_carry + total_need, (long long)p.free_capacity + 1);
  }
  __syncthreads();
  if (popped > 0) atomicMax(&popped_s, popped);
  if (threadIdx.x == 0) {
    cu[p.batch] = (int)min(cu_carry, (long long)0x7fffffff);
    if (writer) p.cu_seqlens[p.batch] = cu[p.batch];
  }
  __syncthreads();
  popped = popped_s;
  if (writer && threadIdx.x == 0) *p.free_count_out = count - popped;
  const int stride = gridDim.x * blockDim.x;
  const int me = blockIdx.x * blockDim.x + threadIdx.x;
  for (int e = me; e < popped; e += stride) {
    const int b = last_not_above(base, p.batch, e);
    const int have = (len[b] + block - 1) >> p.block_shift;  // placed: len[b] >= 0
    p.block_table[(long long)b * p.table_stride + have + (e - base[b])] = p.free_blocks[count - 1 - e];
  }
  const int tokens = min(cu[p.batch], p.max_new);
  for (int t = me; t < p.max_new; t += stride) {
    long long slot = -1;
    if (t < tokens) {
      const int b = last_not_above(cu, p.batch, t);
      const int held = len[b];
      if (held >= 0) {
        const int at = held + (t - cu[b]);
        const int j = at >> p.block_shift;
        const int have = (held + block - 1) >> p.block_shift;
        // Blocks from `have` on are the ones handed out above (by any CTA): read the stack.
        const int id = j < have ? p.block_table[(long long)b * p.table_stride + j]
                                : p.free_blocks[count - 1 - (base[b] + (j - have))];
        slot = ((long long)id << p.block_shift) + (at & (block - 1));
      }
    }
    p.slots[t] = slot;
  }
}

// Gives the blocks of finished requests back: they go on the stack in request order, each
// request's in table order, and the request's length becomes 0. Same plan as kv_plan_kernel.
__global__ void __launch_bounds__(1024) kv_release_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* base = plan_smem;  // [batch]
  __shared__ long long sums64[32];
  const int block = 1 << p.block_shift;
  const int count = min(max(__ldg(p.free_count), 0), p.free_capacity);
  const bool writer = blockIdx.x == 0;
  int carry = 0;
  const int room = p.free_capacity - count;
  for (int b0 = 0; b0 < p.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const bool in = b < p.batch;
    const int held = in ? max(__ldg(p.seq_lens + b), 0) : 0;
    const bool done = in && __ldg(p.new_lens + b) != 0;
    const int gone = done ? (int)min(((long long)held + block - 1) >> p.block_shift, (long long)p.table_width) : 0;
    long long total;
    const long long end = carry + block_scan<long long>(gone, sums64, total);
    if (in) {
      base[b] = (int)min(end - gone, (long long)0x7fffffff);
      if (writer) p.seq_lens_out[b] = done ? 0 : held;
    }
    carry = (int)min(carry + total, (long long)0x7fffffff);
  }
  __syncthreads();
  const int back = min(carry, room);  // a stack that would overflow keeps what it has room for
  if (writer && threadIdx.x == 0) *p.free_count_out = count + back;
  for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < back; e += gridDim.x * blockDim.x) {
    const int b = last_not_above(base, p.batch, e);
    p.free_blocks[count + e] = p.block_table[(long long)b * p.table_stride + (e - base[b])];
  }
}

// ----------------------------------------------------------------------- append --
constexpr int kAppendWarps = 4;
constexpr int kMinScaleExponent = -100;

struct AppendParams {
  const void* x[2];            // new K and V, 16-bit [total, H_kv, D]
  unsigned char* codes[2];     // cache
  float* scale[2];             // [num_blocks, H_kv]
  const long long* slots;      // [total]
  long long x_st[2], x_sh[2];  // token and head strides (elements)
  long long c_sb[2], c_sh[2], c_st[2];  // block, head and token strides of the cache (bytes)
  long long num_slots;         // num_blocks * block
  int total, heads, block_shift, window;  // window: at most 32 tokens
};

// The smallest power of two, at least 2^-100, whose 448-fold is at least `amax` (>= 0,
// finite). 448 = 1.75 * 2^8, so the exponent follows from amax's own and its mantissa.
__device__ __forceinline__ float append_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, kMinScaleExponent);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four fp32 values to e4m3, a.x in the lowest byte; nearest even, at most 448, NaN stays.
__device__ __forceinline__ uint32_t e4m3x4(float2 a, float2 b) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr uint32_t kInf2 = 0x7f807f80u;
  static __device__ __forceinline__ float2 to_float2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};
template <>
struct Elem<__half> {
  static constexpr uint32_t kInf2 = 0x7c007c00u;
  static __device__ __forceinline__ float2 to_float2(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
};

// Quantises new tokens into their slots. A run is a maximal sequence of tokens with
// consecutive slots inside one block; it starts at offset o of the block and makes the scale
//   s = 2^e, e the smallest integer >= -100 with max |x| <= 448 * 2^e  (over the run, one head),
//   raised to the block's old scale if o > 0 (its tokens 0 .. o-1 stay),
// then writes code = e4m3(x / s). Where s grew, the codes of tokens 0 .. o-1 are divided by
// the growth. With powers of two both divisions are exact, so the only rounding is the one to
// e4m3, and requantising changes no code that stays in e4m3's normal range; a scale of
// amax/448 would round every code anew each time a block's range grows, and e4m3 being a
// floating format it would not make the others more exact. Values that are not finite leave
// the scale alone and are stored as NaN.
//
// A warp takes the runs that start in its CTA's window of tokens, for one head of K or V: a lane
// looks at one token of the window each, so that finding the runs is one load. A run of up to
// 2048 values (16 tokens of 128) stays in registers between the pass for the maximum and the
// one for the codes; a longer one is read again, from the L2.
// Bound: DRAM for prompts (2 bytes read, 1 written per value): 25k tokens of 8 heads of 128 in
// 31 us a call, 5.0 TB/s of 6.6. Of that 29.5 on the device, where it took 36 with 80 registers and
// three quarters of the warps, and 30.4 with eight warps per CTA. Latency for a decode step: 4.9 us a call.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kAppendWarps, 8) kv_append_kernel(const AppendParams p) {
  constexpr int kPerRow = D / 8;   // 8 values (16 bytes of input) per lane and step
  constexpr int kAhead = 8;        // steps in registers at once
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.y * kAppendWarps + warp;
  if (unit >= 2 * p.heads) return;
  const int kv = unit >= p.heads, h = unit - kv * p.heads;
  const int block = 1 << p.block_shift;
  const int t0 = blockIdx.x * p.window;
  // Lane i looks at token t0 + i, beyond the window too. It follows the token before it if its
  // slot does and no block begins there; a run begins where one in the window does not follow.
  const bool real = t0 + lane < p.total;
  const long long mine = real ? __ldg(p.slots + t0 + lane) : -1;
  long long prev = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) prev = t0 > 0 ? __ldg(p.slots + t0 - 1) : -2;
  const unsigned follows =
      __ballot_sync(0xffffffffu, real && mine == prev + 1 && (mine & (block - 1)) != 0 && prev >= 0);
  const unsigned in_cache = __ballot_sync(0xffffffffu, lane < p.window && mine >= 0 && mine < p.num_slots);
  for (unsigned runs = in_cache & ~follows; runs != 0; runs &= runs - 1) {
    const int first = __ffs(runs) - 1;
    const int t = t0 + first;
    const long long slot = __shfl_sync(0xffffffffu, mine, first);
    const int o = (int)(slot & (block - 1));
    // Its length, at most to the block's end: the bits of `follows` behind it, and if they reach
    // the last lane, the tokens behind.
    const unsigned after = first < 31 ? ~(follows >> (first + 1)) : 1u;  // 0 bits: tokens that follow
    int n = after != 0 ? __ffs(after) : 32;
    n = min(n, 32 - first);
    if (first + n == 32) {
      const int most = min(block - o, p.total - t);
      for (int i = n; i < most; i += 32) {
        const unsigned ends =
            __ballot_sync(0xffffffffu, i + lane >= most || __ldg(p.slots + t + i + lane) != slot + i + lane);
        n = i + (ends != 0 ? __ffs(ends) - 1 : 32);
        if (ends != 0) break;
      }
    }
    // This lane's chunks: i = 32 k + lane, 8 values each; 32 chunks are kRows rows.
    constexpr int kRows = 32 / kPerRow;
    const int chunks = n * kPerRow;
    const int row = lane / kPerRow, col = lane % kPerRow * 8;
    const T* x = static_cast<const T*>(p.x[kv]) + (t + row) * p.x_st[kv] + h * p.x_sh[kv] + col;
    const long long x_step = kRows * p.x_st[kv];
    uint4 v[kAhead];
    auto load = [&](int base) {
      const T* at = x + base / 32 * x_step;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        v[k] = make_uint4(0, 0, 0, 0);
        if (base + 32 * k + lane < chunks) v[k] = __ldg(reinterpret_cast<const uint4*>(at + k * x_step));
      }
    };
    // Largest magnitude, compared as bits; what is not finite has the largest bits, and then
    // (never in a sound model) a second look leaves it out.
    uint32_t top = 0;
    for (int base = 0; base < chunks; base += 32 * kAhead) {
      load(base);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        top = __vmaxu2(top, __vmaxu2(v[k].x & 0x7fff7fffu, v[k].y & 0x7fff7fffu));
        top = __vmaxu2(top, __vmaxu2(v[k].z & 0x7fff7fffu, v[k].w & 0x7fff7fffu));
      }
    }
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    const bool all_finite = top < (Elem<T>::kInf2 & 0xffffu);
    if (!all_finite) {
      top = 0;
#pragma unroll 1
      for (int i = lane; i < chunks; i += 32) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(x + i / 32 * x_step));
        const uint32_t u[4] = {w.x & 0x7fff7fffu, w.y & 0x7fff7fffu, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __vmaxu2(top, u[e] & ~__vcmpgeu2(u[e], Elem<T>::kInf2));
      }
      top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    }
    const float wanted = append_scale(Elem<T>::to_float2(top).x);
    float* scale = p.scale[kv] + (slot >> p.block_shift) * p.heads + h;
    const float before = o > 0 ? *scale : 0.f;
    const float s = o > 0 ? fmaxf(before, wanted) : wanted;
    __syncwarp();
    if (lane == 0) *scale = s;  // every lane has read it
    unsigned char* dst = p.codes[kv] + (slot >> p.block_shift) * p.c_sb[kv] + (long long)h * p.c_sh[kv];
    if (o > 0 && s != before) {
      const float shrink = before / s;
#pragma unroll 4
      for (int i = lane; i < o * (D / 16); i += 32) {
        uint4* at = reinterpret_cast<uint4*>(dst + (i / (D / 16)) * p.c_st[kv] + (i % (D / 16)) * 16);
        uint4 c = *at;
        uint32_t* w = &c.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 lo = e4m3x2_to_float2(w[k] & 0xffffu), hi = e4m3x2_to_float2(w[k] >> 16);
          w[k] = e4m3x4(make_float2(lo.x * shrink, lo.y * shrink), make_float2(hi.x * shrink, hi.y * shrink));
        }
        *at = c;
      }
    }
    // x / s: by the exact reciprocal when s is a power of two (always, unless the old scale
    // came from elsewhere).
    const bool plain = all_finite && (__float_as_uint(s) & 0x7fffffu) == 0;
    const float inv = 1.f / s;
    unsigned char* to = dst + (o + row) * p.c_st[kv] + col;
    const long long to_step = kRows * p.c_st[kv];
    auto write = [&](auto&& quotient) {
      for (int base = 0; base < chunks; base += 32 * kAhead) {
        if (chunks > 32 * kAhead) load(base);
        unsigned char* at = to + base / 32 * to_step;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (base + 32 * k + lane < chunks) {
            const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
            float2 f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = quotient(Elem<T>::to_float2(w[e]));
            *reinterpret_cast<uint2*>(at + k * to_step) = make_uint2(e4m3x4(f[0], f[1]), e4m3x4(f[2], f[3]));
          }
        }
      }
    };
    if (plain) {
      write([&](float2 f) { return __fmul2_rn(f, make_float2(inv, inv)); });
    } else {
      auto one = [&](float q) { return isfinite(q) ? q / s : __int_as_float(0x7fffffff); };
      write([&](float2 f) { return make_float2(one(f.x), one(f.y)); });
    }
  }
}

}  // namespace apex
