// Host side of the paged 8-bit K/V cache operators: argument validation and launches behind
// the C ABI declared in include/apex_attn.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "apex_attn.h"
#include "attn_paged_kernel.cuh"
#include "kv_cache_kernels.cuh"
#include "runtime.h"

namespace {

using apex::host::aligned16;
using apex::host::device_of;
using apex::host::DeviceGuard;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int launched() {
  if (cudaGetLastError() != cudaSuccess) return APEX_ATTN_ERR_LAUNCH;
  return APEX_ATTN_OK;
}

// 16, 32, 64 or 128 -> its logarithm; -1 otherwise.
int block_shift_of(int block_size) {
  for (int s = 4; s <= 7; ++s)
    if (block_size == 1 << s) return s;
  return -1;
}

// Every pointer of a call lives on the device of the first; nulls are skipped.
int common_device(const void* const* ptrs, int n) {
  const int dev = device_of(ptrs[0]);
  if (dev < 0) return -1;
  for (int i = 1; i < n; ++i)
    if (ptrs[i] != nullptr && device_of(ptrs[i]) != dev) return -1;
  return dev;
}

// Whether the rows of `row` elements that a strided array is written in do not overlap: taken from
// the smallest stride up, each steps over all that the dimensions below it reach.
template <int N>
bool rows_distinct(long long row, const long long (&size)[N], const long long (&stride)[N]) {
  __int128 reach = row;
  unsigned left = (1u << N) - 1;
  for (int n = 0; n < N; ++n) {
    int least = -1;
    for (int i = 0; i < N; ++i)
      if ((left >> i & 1) && (least < 0 || stride[i] < stride[least])) least = i;
    left &= ~(1u << least);
    if (size[least] <= 1) continue;
    if (stride[least] < reach) return false;
    reach += (__int128)(size[least] - 1) * stride[least];
  }
  return true;
}

// The device of a call: the one that the caller knows to own every pointer, else looked up.
int device_of_call(int known, const void* const* ptrs, int n) {
  if (known != 0) return known > 0 && known <= apex::host::kMaxDevices ? known - 1 : -1;
  return common_device(ptrs, n);
}

// Raises a kernel's dynamic shared-memory limit once per device.
template <typename K>
int allow_smem(K kern, int bytes, std::atomic<unsigned long long>& done, int dev) {
  const unsigned long long bit = 1ull << dev;
  if (done.load(std::memory_order_acquire) & bit) return APEX_ATTN_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return APEX_ATTN_ERR_LAUNCH;
  }
  done.fetch_or(bit, std::memory_order_release);
  return APEX_ATTN_OK;
}
static_assert(apex::host::kMaxDevices <= 64, "one bit per device");

// ------------------------------------------------------------------ bookkeeping --
constexpr int kPlanSmem = (3 * apex::kPlanMaxBatch + 1) * (int)sizeof(int);
std::atomic<unsigned long long> g_plan_smem{0}, g_release_smem{0};

int plan(const apex_attn_kv_plan_args* a, bool release, void* stream) {
  if (!a || !a->block_table || !a->seq_lens || !a->free_blocks || !a->free_count || !a->seq_lens_out ||
      !a->free_count_out)
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (release ? !a->finished : (!a->new_lens || !a->slots || !a->cu_seqlens || !a->placed))
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->table_width <= 0 || a->free_capacity <= 0 || (!release && a->max_new_tokens <= 0))
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  const int shift = block_shift_of(a->block_size);
  if (shift < 0) return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (a->batch > apex::kPlanMaxBatch || (long long)a->table_width * a->block_size > INT_MAX ||
      a->free_capacity > (1 << 30) || a->max_new_tokens > (1 << 30))
    return APEX_ATTN_ERR_TOO_LARGE;
  if (a->table_stride < a->table_width) return APEX_ATTN_ERR_BAD_LAYOUT;
  const void* ptrs[] = {a->block_table, a->seq_lens,     a->free_blocks, a->free_count,
                        a->seq_lens_out, a->free_count_out, release ? a->finished : a->new_lens,
                        release ? nullptr : a->slots, release ? nullptr : a->cu_seqlens,
                        release ? nullptr : a->placed};
  for (const void* ptr : ptrs)
    if (!aligned(ptr, 4)) return APEX_ATTN_ERR_BAD_LAYOUT;
  if (!release && !aligned(a->slots, 8)) return APEX_ATTN_ERR_BAD_LAYOUT;
  // The CTAs read all inputs independently of one another's writes.
  if (a->seq_lens_out == a->seq_lens || a->free_count_out == a->free_count) return APEX_ATTN_ERR_INVALID_ARGUMENT;

  const int dev = device_of_call(a->known_device, ptrs, 10);
  if (dev < 0) return APEX_ATTN_ERR_NO_DEVICE;
  DeviceGuard guard(dev);
  apex::host::Device d;
  int rc = apex::host::acquire(dev, &d);
  if (rc != APEX_ATTN_OK) return rc;
  rc = release ? allow_smem(apex::kv_release_kernel, kPlanSmem, g_release_smem, dev)
               : allow_smem(apex::kv_plan_kernel, kPlanSmem, g_plan_smem, dev);
  if (rc != APEX_ATTN_OK) return rc;

  apex::PlanParams p{};
  p.block_table = a->block_table;
  p.table_stride = a->table_stride;
  p.seq_lens = a->seq_lens;
  p.new_lens = release ? a->finished : a->new_lens;
  p.free_blocks = a->free_blocks;
  p.free_count = a->free_count;
  p.slots = a->slots;
  p.cu_seqlens = a->cu_seqlens;
  p.seq_lens_out = a->seq_lens_out;
  p.free_count_out = a->free_count_out;
  p.placed = a->placed;
  p.batch = a->batch;
  p.table_width = a->table_width;
  p.free_capacity = a->free_capacity;
  p.block_shift = shift;
  p.max_new = a->max_new_tokens;
  const int threads = a->batch <= 256 ? 256 : 1024;
  const long long entries = release ? (long long)a->batch * 4 : std::max(a->max_new_tokens, a->batch);
  const int grid = (int)std::min<long long>((entries + threads - 1) / threads, d.num_sms);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (release)
    apex::kv_release_kernel<<<grid, threads, a->batch * (int)sizeof(int), s>>>(p);
  else
    apex::kv_plan_kernel<<<grid, threads, (3 * a->batch + 1) * (int)sizeof(int), s>>>(p);
  return launched();
}

// ----------------------------------------------------------------------- append --
template <typename T>
void launch_append(const apex::AppendParams& p, int head_dim, dim3 grid, cudaStream_t s) {
  constexpr int kThreads = 32 * apex::kAppendWarps;
  switch (head_dim) {
    case 64: apex::kv_append_kernel<T, 64><<<grid, kThreads, 0, s>>>(p); break;
    case 128: apex::kv_append_kernel<T, 128><<<grid, kThreads, 0, s>>>(p); break;
    default: apex::kv_append_kernel<T, 256><<<grid, kThreads, 0, s>>>(p);
  }
}

int append(const apex_attn_kv_append_args* a, void* stream) {
  if (!a || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->slots)
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (a->total <= 0 || a->heads_kv <= 0 || a->num_blocks <= 0) return APEX_ATTN_ERR_INVALID_ARGUMENT;
  const int shift = block_shift_of(a->block_size);
  if (shift < 0) return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (!apex_attn_supports_head_dim(a->head_dim)) return APEX_ATTN_ERR_UNSUPPORTED_HEAD_DIM;
  if (a->dtype != APEX_ATTN_BF16 && a->dtype != APEX_ATTN_FP16) return APEX_ATTN_ERR_UNSUPPORTED_DTYPE;
  if (a->total > (1 << 30) || a->heads_kv > 65535) return APEX_ATTN_ERR_TOO_LARGE;
  for (int i = 0; i < 4; ++i)
    if (a->strides[i] < 0 || (a->strides[i] & 7) != 0 || a->strides[i] >= (1LL << 38)) return APEX_ATTN_ERR_BAD_LAYOUT;
  for (int i = 4; i < 10; ++i)
    if (a->strides[i] < 0 || (a->strides[i] & 15) != 0 || a->strides[i] >= (1LL << 38)) return APEX_ATTN_ERR_BAD_LAYOUT;
  if (a->strides[6] < a->head_dim || a->strides[9] < a->head_dim) return APEX_ATTN_ERR_BAD_LAYOUT;
  for (int i = 4; i < 10; i += 3)
    if (!rows_distinct<3>(a->head_dim, {a->num_blocks, a->heads_kv, a->block_size},
                          {a->strides[i], a->strides[i + 1], a->strides[i + 2]}))
      return APEX_ATTN_ERR_BAD_LAYOUT;
  if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_cache) || !aligned16(a->v_cache) ||
      !aligned(a->k_scale, 4) || !aligned(a->v_scale, 4) || !aligned(a->slots, 8))
    return APEX_ATTN_ERR_BAD_LAYOUT;

  const void* ptrs[] = {a->k, a->v, a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->slots};
  const int dev = device_of_call(a->known_device, ptrs, 7);
  if (dev < 0) return APEX_ATTN_ERR_NO_DEVICE;
  DeviceGuard guard(dev);
  apex::host::Device d;
  int rc = apex::host::acquire(dev, &d);
  if (rc != APEX_ATTN_OK) return rc;

  apex::AppendParams p{};
  p.x[0] = a->k;
  p.x[1] = a->v;
  p.codes[0] = static_cast<unsigned char*>(a->k_cache);
  p.codes[1] = static_cast<unsigned char*>(a->v_cache);
  p.scale[0] = a->k_scale;
  p.scale[1] = a->v_scale;
  p.slots = a->slots;
  for (int i = 0; i < 2; ++i) {
    p.x_st[i] = a->strides[2 * i];
    p.x_sh[i] = a->strides[2 * i + 1];
    p.c_sb[i] = a->strides[4 + 3 * i];
    p.c_sh[i] = a->strides[5 + 3 * i];
    p.c_st[i] = a->strides[6 + 3 * i];
  }
  p.num_slots = (long long)a->num_blocks * a->block_size;
  p.total = a->total;
  p.heads = a->heads_kv;
  p.block_shift = shift;
  // A window of one token while that makes at most 32 CTAs per SM (decode: every token is a run of
  // its own); else windows that a run mostly fills.
  const int groups = (2 * a->heads_kv + apex::kAppendWarps - 1) / apex::kAppendWarps;
  const bool few = (long long)a->total * groups <= 32LL * d.num_sms;
  p.window = few ? 1 : std::min(a->block_size, 32);
  const dim3 grid((unsigned)((a->total + p.window - 1) / p.window), (unsigned)groups);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == APEX_ATTN_BF16) launch_append<__nv_bfloat16>(p, a->head_dim, grid, s);
  else launch_append<__half>(p, a->head_dim, grid, s);
  return launched();
}

// -------------------------------------------------------------------- attention --
constexpr int kMaxSms = 160;  // the workspace holds what this many SMs' CTAs may write

// Query rows per tile, the smallest that holds all rows of a request's K/V head: 16 or 32 with
// tokens as the M side of the products, 64 with the query rows (half the shared memory for rows
// and weights, so more of the cache under way), else 128.
int query_tile(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

struct Workspace {
  size_t share, lse, o, bytes;  // offsets and size
};

Workspace workspace_plan(int query_rows, int head_dim) {
  const size_t parts = 2 * 2 * kMaxSms;  // two per CTA, at most two CTAs per SM
  Workspace w;
  w.share = 0;
  w.lse = parts * apex::kShareInts * sizeof(int);
  w.o = w.lse + parts * query_rows * sizeof(float);
  w.bytes = w.o + parts * query_rows * head_dim * sizeof(float);
  return w;
}

size_t workspace_bytes(int heads_q, int heads_kv, int max_seqlen_q, int head_dim) {
  if (heads_q <= 0 || heads_kv <= 0 || max_seqlen_q <= 0 || head_dim <= 0) return 0;
  const long long rows = (long long)((heads_q + heads_kv - 1) / heads_kv) * max_seqlen_q;
  return workspace_plan(query_tile((int)std::min(rows, 1LL << 30)), head_dim).bytes;
}

// 4-D map over the cache [num_blocks, H_kv, block, D], dims ordered (D, block, H_kv, blocks); a
// box is one block of one head, up to 128 columns, swizzled by its row size.
int encode_cache(CUtensorMap* m, const void* ptr, const apex_attn_paged_args& a, const long long* st) {
  const cuuint64_t sh = a.heads_kv > 1 ? st[1] : (cuuint64_t)a.block_size * st[2];
  const cuuint64_t sb = a.num_blocks > 1 ? st[0] : (cuuint64_t)a.heads_kv * sh;
  const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.block_size, (cuuint64_t)a.heads_kv,
                              (cuuint64_t)a.num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)st[2], sh, sb};
  const cuuint32_t box[4] = {(cuuint32_t)std::min(a.head_dim, 128), (cuuint32_t)a.block_size, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = apex::host::tensor_map_encoder()(
      m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, strides, box, estr,
      CU_TENSOR_MAP_INTERLEAVE_NONE, a.head_dim >= 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
      // Rows that do not follow one another: fetching 256 bytes for one would read a neighbour's.
      st[2] >= 256 && st[2] > a.head_dim ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? APEX_ATTN_OK : APEX_ATTN_ERR_TENSOR_MAP;
}

template <typename T, int D, int NQ>
int launch_paged(const apex::PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int dev, int num_sms,
                 cudaStream_t s) {
  using C = apex::PagedCfg<T, D, NQ>;
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(apex::attn_paged_kernel<T, D, NQ>, C::kBytes, done, dev);
  if (rc != APEX_ATTN_OK) return rc;
  const int grid = C::kCtas * std::min(num_sms, kMaxSms);
  // Both may be set up while the last CTAs of the kernel before them run; they wait for its end
  // before they read or write anything (measured: one short request 14.4 -> 11.9 us a call, 48 requests
  // 80 -> 77; calls of 3 x 1024 new tokens lose 1 %).
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kBytes;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, apex::attn_paged_kernel<T, D, NQ>, mk, mv, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return APEX_ATTN_ERR_LAUNCH;
  }
  cfg.blockDim = dim3(apex::kCombineThreads);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, apex::attn_paged_combine_kernel<T, D, NQ>, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return APEX_ATTN_ERR_LAUNCH;
  }
  return APEX_ATTN_OK;
}

template <typename T, int D>
int launch_tile(int tile, const apex::PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int dev,
                int num_sms, cudaStream_t s) {
  switch (tile) {
    case 16: return launch_paged<T, D, 16>(p, mk, mv, dev, num_sms, s);
    case 32: return launch_paged<T, D, 32>(p, mk, mv, dev, num_sms, s);
    case 64: return launch_paged<T, D, 64>(p, mk, mv, dev, num_sms, s);
    default: return launch_paged<T, D, 128>(p, mk, mv, dev, num_sms, s);
  }
}

template <typename T>
int launch_dim(int head_dim, int tile, const apex::PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv,
               int dev, int num_sms, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_tile<T, 64>(tile, p, mk, mv, dev, num_sms, s);
    case 128: return launch_tile<T, 128>(tile, p, mk, mv, dev, num_sms, s);
    default: return launch_tile<T, 256>(tile, p, mk, mv, dev, num_sms, s);
  }
}

int forward_paged(const apex_attn_paged_args* a, void* workspace, size_t bytes, void* stream) {
  // ---- argument validation (no CUDA calls) ----
  if (!a || !a->q || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->block_table || !a->seq_lens ||
      !a->o || !workspace)
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->heads_q % a->heads_kv != 0 || a->total_q <= 0 ||
      a->max_seqlen_q <= 0 || a->num_blocks <= 0 || a->table_width <= 0)
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (!a->cu_seqlens_q && (a->total_q % a->batch != 0 || a->total_q / a->batch != a->max_seqlen_q))
    return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (a->window_left < -1 || (a->window_left >= 0 && !a->causal)) return APEX_ATTN_ERR_INVALID_ARGUMENT;
  const int shift = block_shift_of(a->block_size);
  if (shift < 0) return APEX_ATTN_ERR_INVALID_ARGUMENT;
  if (!apex_attn_supports_head_dim(a->head_dim)) return APEX_ATTN_ERR_UNSUPPORTED_HEAD_DIM;
  if (a->dtype != APEX_ATTN_BF16 && a->dtype != APEX_ATTN_FP16) return APEX_ATTN_ERR_UNSUPPORTED_DTYPE;
  if (!std::isfinite(a->sm_scale) || !(a->sm_scale > 0.f)) return APEX_ATTN_ERR_BAD_SCALE;
  if (a->total_q > (1 << 30) || a->batch > 65535 || a->heads_q > 32767 ||
      (long long)a->max_seqlen_q * a->heads_q > (1 << 30) || (long long)a->table_width * a->block_size > (1 << 30))
    return APEX_ATTN_ERR_TOO_LARGE;
  for (int i = 0; i < 4; ++i)
    if (a->strides[i] < 0 || (a->strides[i] & 7) != 0 || a->strides[i] >= (1LL << 38)) return APEX_ATTN_ERR_BAD_LAYOUT;
  for (int i = 4; i < 10; ++i)
    if (a->strides[i] < 0 || (a->strides[i] & 15) != 0 || a->strides[i] >= (1LL << 38)) return APEX_ATTN_ERR_BAD_LAYOUT;
  if (a->strides[1] < a->head_dim || a->strides[3] < a->head_dim || a->strides[6] < a->head_dim ||
      a->strides[9] < a->head_dim || a->table_stride < a->table_width ||
      !rows_distinct<2>(a->head_dim, {a->total_q, a->heads_q}, {a->strides[2], a->strides[3]}))
    return APEX_ATTN_ERR_BAD_LAYOUT;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->o) || !aligned16(workspace))
    return APEX_ATTN_ERR_BAD_LAYOUT;
  if (!aligned(a->k_scale, 4) || !aligned(a->v_scale, 4) || !aligned(a->block_table, 4) || !aligned(a->seq_lens, 4) ||
      !aligned(a->cu_seqlens_q, 4) || !aligned(a->lse, 4))
    return APEX_ATTN_ERR_BAD_LAYOUT;
  if (bytes < workspace_bytes(a->heads_q, a->heads_kv, a->max_seqlen_q, a->head_dim))
    return APEX_ATTN_ERR_INVALID_ARGUMENT;

  // ---- device ----
  const void* ptrs[] = {a->q,           a->k_cache,  a->v_cache,      a->k_scale, a->v_scale,
                        a->block_table, a->seq_lens, a->cu_seqlens_q, a->o,       a->lse, workspace};
  const int dev = device_of_call(a->known_device, ptrs, 11);
  if (dev < 0) return APEX_ATTN_ERR_NO_DEVICE;
  DeviceGuard guard(dev);
  apex::host::Device d;
  int rc = apex::host::acquire(dev, &d);
  if (rc != APEX_ATTN_OK) return rc;

  const long long* st = a->strides;
  CUtensorMap mk, mv;
  if ((rc = encode_cache(&mk, a->k_cache, *a, st + 4)) || (rc = encode_cache(&mv, a->v_cache, *a, st + 7))) return rc;

  const int group = a->heads_q / a->heads_kv;
  const int tile = query_tile(group * a->max_seqlen_q);
  // The kernel counts its work in 31 bits: K/V heads x query tiles x (tiles of the cache and the
  // fixed cost of an item).
  const long long items = (long long)a->heads_kv * ((long long)a->total_q * group / tile + a->batch);
  const long long units = (long long)a->table_width * a->block_size / apex::kPagedTile + 1 + apex::kPagedItemUnits<128>;
  if (items * units > INT_MAX) return APEX_ATTN_ERR_TOO_LARGE;
  const Workspace w = workspace_plan(tile, a->head_dim);
  char* ws = static_cast<char*>(workspace);
  apex::PagedParams p{};
  p.q = a->q;
  p.o = a->o;
  p.lse = a->lse;
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.block_table = a->block_table;
  p.seq_lens = a->seq_lens;
  p.cu_seqlens_q = a->cu_seqlens_q;
  p.share = reinterpret_cast<int*>(ws + w.share);
  p.part_lse = reinterpret_cast<float*>(ws + w.lse);
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  p.status = d.status;
  p.host_flag = d.host_flag_dev;
  p.timeout_ns = apex::host::wait_timeout_ns();
  p.table_stride = a->table_stride;
  p.q_st = st[0];
  p.q_sh = st[1];
  p.o_st = st[2];
  p.o_sh = st[3];
  p.batch = a->batch;
  p.heads_kv = a->heads_kv;
  p.group = group;
  p.group_magic = group > 1 ? (unsigned)(((1ull << 32) + group - 1) / group) : 0;
  p.total_q = a->total_q;
  p.max_q = a->max_seqlen_q;
  p.num_blocks = a->num_blocks;
  p.block_shift = shift;
  p.table_width = a->table_width;
  p.causal = a->causal ? 1 : 0;
  // A window that reaches past every table hides nothing.
  p.window = a->window_left < a->table_width * a->block_size ? a->window_left : -1;
  p.zero_rest = a->zero_rest && a->cu_seqlens_q ? 1 : 0;
  p.one_tile = group * a->max_seqlen_q <= tile ? 1 : 0;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->dtype == APEX_ATTN_BF16 ? launch_dim<__nv_bfloat16>(a->head_dim, tile, p, mk, mv, dev, d.num_sms, s)
                                    : launch_dim<__half>(a->head_dim, tile, p, mk, mv, dev, d.num_sms, s);
}

}  // namespace

extern "C" {

int apex_attn_kv_plan(const apex_attn_kv_plan_args* args, void* stream) { return plan(args, false, stream); }

int apex_attn_kv_release(const apex_attn_kv_plan_args* args, void* stream) { return plan(args, true, stream); }

int apex_attn_kv_append(const apex_attn_kv_append_args* args, void* stream) { return append(args, stream); }

size_t apex_attn_fwd_paged_workspace_bytes(int heads_q, int heads_kv, int max_seqlen_q, int head_dim) {
  return workspace_bytes(heads_q, heads_kv, max_seqlen_q, head_dim);
}

int apex_attn_fwd_paged(const apex_attn_paged_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  return forward_paged(args, workspace, workspace_bytes, stream);
}

}  // extern "C"
