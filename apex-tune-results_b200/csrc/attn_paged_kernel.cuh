// Attention over a paged 8-bit K/V cache (the layout kv_cache_kernels.cuh writes).
#pragma once

#include "attn_fwd_kernel.cuh"
#include "kv_cache_kernels.cuh"

namespace apex {

struct PagedParams {
  const void* q;  // [total_q, H, D]
  void* o;
  float* lse;  // nullable, [H, total_q]
  const unsigned char* k_codes;
  const unsigned char* v_codes;
  const float* k_scale;  // [num_blocks, H_kv]
  const float* v_scale;
  const int* block_table;  // [batch, table_width], row stride table_stride
  const int* seq_lens;     // [batch] tokens in the cache
  const int* cu_seqlens_q; // [batch + 1]; null: total_q / batch query tokens each
  long long table_stride;
  long long q_st, q_sh, o_st, o_sh;                      // token, head strides (elements)
  long long k_sb, k_sh, k_st, v_sb, v_sh, v_st;          // block, head, token strides (bytes)
  int batch, heads_q, heads_kv, group, total_q, max_q;
  int num_blocks, block_shift, table_width;
  int causal, window, zero_rest;
  float scale_log2;  // sm_scale * log2(e)
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
    r.nq = p.total_q / p.batch;
    r.q0 = b * r.nq;
  }
  const long long room = (long long)p.table_width << p.block_shift;
  r.len = (int)min((long long)max(__ldg(p.seq_lens + b), 0), room);
  return r;
}

// One CTA per (query token of a request, query head): its warps take keys in turn, one key
// per warp at a time with the head dim spread over the lanes, each with a running maximum
// and sum, and are merged at the end.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_paged_simple_kernel(const PagedParams p) {
  constexpr int E = D / 32;  // consecutive columns per lane
  const int b = blockIdx.z, i = blockIdx.x, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedRequest r = paged_request(p, b);
  if (p.zero_rest && i == 0) {  // rows outside every request: before the first, behind this one
    const int next = b + 1 < p.batch ? paged_request(p, b + 1).q0 : p.total_q;
    for (int row = b == 0 ? 0 : r.q0 + r.nq; row < next; ++row) {
      if (row >= r.q0 && row < r.q0 + r.nq) continue;
      for (int d = threadIdx.x; d < D; d += 128)
        static_cast<T*>(p.o)[(long long)row * p.o_st + (long long)h * p.o_sh + d] = (T)0.f;
      if (p.lse != nullptr && threadIdx.x == 0) p.lse[(long long)h * p.total_q + row] = 0.f;
    }
  }
  if (i >= r.nq) return;
  const int hkv = h / p.group;
  const T* q = static_cast<const T*>(p.q) + (long long)(r.q0 + i) * p.q_st + (long long)h * p.q_sh + lane * E;
  float qf[E];
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = (float)q[e];
  const int place = r.len - r.nq + i;
  const int hi = p.causal ? min(place + 1, r.len) : r.len;
  const int lo = p.window >= 0 ? max(place - p.window, 0) : 0;
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int j = lo + warp; j < hi; j += 4) {
    const int id = __ldg(p.block_table + (long long)b * p.table_stride + (j >> p.block_shift));
    const int row = j & ((1 << p.block_shift) - 1);
    const bool real = id >= 0 && id < p.num_blocks;  // others read as zeros
    const float ks = real ? __ldg(p.k_scale + (long long)id * p.heads_kv + hkv) : 0.f;
    const float vs = real ? __ldg(p.v_scale + (long long)id * p.heads_kv + hkv) : 0.f;
    const unsigned char* k = p.k_codes + (long long)id * p.k_sb + (long long)hkv * p.k_sh + (long long)row * p.k_st;
    const unsigned char* v = p.v_codes + (long long)id * p.v_sb + (long long)hkv * p.v_sh + (long long)row * p.v_st;
    float s = 0.f;
    if (real) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 kk = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(k + lane * E + e));
        s += qf[e] * kk.x + qf[e + 1] * kk.y;
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= ks * p.scale_log2;
    const float top = fmaxf(m, s);
    const float w = exp2f(s - top), old = exp2f(m - top);
    l = l * old + w;
    m = top;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 vv = real ? e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(v + lane * E + e)) : make_float2(0.f, 0.f);
      acc[e] = acc[e] * old + w * vs * vv.x;
      acc[e + 1] = acc[e + 1] * old + w * vs * vv.y;
    }
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float sum = 0.f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - top);
    sum += sl[w] * f[w];
  }
  T* o = static_cast<T*>(p.o) + (long long)(r.q0 + i) * p.o_st + (long long)h * p.o_sh;
  for (int d = threadIdx.x; d < D; d += 128) {
    const float x = so[0][d] * f[0] + so[1][d] * f[1] + so[2][d] * f[2] + so[3][d] * f[3];
    o[d] = (T)(sum == 0.f ? 0.f : x / sum);
  }
  if (p.lse != nullptr && threadIdx.x == 0)
    p.lse[(long long)h * p.total_q + r.q0 + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace apex
