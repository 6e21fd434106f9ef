// The 8-bit paged key/value cache: page planning and the cache write.
//
// A page holds 64 tokens of every KV head; its K and V are e4m3 codes with
// one power-of-two scale per (page, head) each.  plan_pages_kernel turns
// request lengths into block tables, slots and positions; append_kv_kernel
// rounds a step's keys and values into the pages.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "launch.h"

namespace ls {
namespace {

constexpr int kPage = LS_PAGE_TOKENS;

// ---------------------------------------------------------------------------
// Planning
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 512;

__device__ __forceinline__ int32_t saturate32(int64_t x) {
  return static_cast<int32_t>(x > 0x7FFFFFFF ? 0x7FFFFFFF : x);
}

// Request b holds ctx tokens and gets n: blocks before the step, new blocks,
// blocks the step writes (the half-filled one included).
struct PlanRow {
  int64_t ctx, n, had, need, written;
  bool bad;
};

__device__ __forceinline__ PlanRow plan_row(const PlanArgs& a, int b) {
  PlanRow r;
  r.ctx = __ldg(a.context_lens + b);
  r.n = __ldg(a.new_lens + b);
  r.bad = r.ctx < 0 || r.n < 0;
  r.ctx = max(r.ctx, int64_t{0});
  r.n = max(r.n, int64_t{0});
  const int64_t m = a.max_blocks;
  const int64_t total = (r.ctx + r.n + kPage - 1) / kPage;
  r.bad = r.bad || total > m;
  r.had = min((r.ctx + kPage - 1) / kPage, m);
  r.need = min(total, m) - r.had;
  r.written = r.n > 0 ? total - r.ctx / kPage : 0;
  return r;
}

// Every CTA computes the prefix sums over the requests by itself (shared
// memory, one block scan), so one launch does the whole step and no CTA waits
// for another; then the tokens are dealt to the threads, which find their
// request by binary search.  The thread of a new block's first token writes
// its block-table entry; a token in the half-filled old block reads that
// block's entry, which nobody writes.  Integer sums only: the result does not
// depend on the launch shape.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* cu_q = plan_smem;                  // [batch + 1]
  int32_t* cu_need = plan_smem + a.batch + 1;  // [batch + 1]
  __shared__ int64_t warp_sum[3][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool lead = blockIdx.x == 0;

  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t own[3] = {0, 0, 0};
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const PlanRow r = plan_row(a, b);
    own[0] += r.n;
    own[1] += r.need;
    own[2] += r.written;
    bad = bad || r.bad;
  }
  int64_t run[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int64_t x = own[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[i][warp] = x;
    run[i] = x - own[i];
  }
  __syncthreads();
  int64_t total[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) run[i] += warp_sum[i][w];
      total[i] += warp_sum[i][w];
    }
  for (int b = b0; b < b1; ++b) {
    const PlanRow r = plan_row(a, b);
    cu_q[b] = saturate32(run[0]);
    cu_need[b] = saturate32(run[1]);
    if (lead) {
      a.cu_seqlens_q[b] = saturate32(run[0]);
      a.cu_blocks[b] = saturate32(run[2]);
      a.seq_lens[b] = saturate32(r.ctx + r.n);
    }
    run[0] += r.n;
    run[1] += r.need;
    run[2] += r.written;
  }
  const int64_t head_in = __ldg(a.free_head);
  const int64_t head = min(max(head_in, int64_t{0}), static_cast<int64_t>(a.num_free));
  if (tid == 0) {
    cu_q[a.batch] = saturate32(total[0]);
    cu_need[a.batch] = saturate32(total[1]);
    if (lead) {
      a.cu_seqlens_q[a.batch] = saturate32(total[0]);
      a.cu_blocks[a.batch] = saturate32(total[2]);
      *a.free_head_out =
          static_cast<int32_t>(min(head + total[1], static_cast<int64_t>(a.num_free)));
      if (total[0] > a.total_new) report(a.status, LS_DEVERR_SEQLENS);
      if (head != head_in || head + total[1] > a.num_free) report(a.status, LS_DEVERR_PAGES);
    }
  }
  if (lead && bad) report(a.status, LS_DEVERR_SEQLENS);
  __syncthreads();

  const int64_t tokens = min(total[0], a.total_new);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid; i < a.total_new;
       i += stride) {
    int64_t slot = -1, pos = 0;
    if (i < tokens) {
      // Last request whose first token is at or before i (empty requests
      // share their successor's offset and are passed over).
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu_q[mid] <= i) lo = mid; else hi = mid - 1;
      }
      const int64_t ctx = max(__ldg(a.context_lens + lo), 0);
      pos = ctx + (i - cu_q[lo]);
      const int64_t block = pos / kPage;
      if (block < a.max_blocks) {
        const int64_t had = (ctx + kPage - 1) / kPage;
        int32_t* entry = a.block_table + static_cast<int64_t>(lo) * a.max_blocks + block;
        int32_t page;
        if (block < had) {
          page = *entry;
        } else {
          const int64_t at = head + cu_need[lo] + (block - had);
          page = at < a.num_free ? __ldg(a.free_pages + at) : -1;
          if (pos % kPage == 0) *entry = page;
        }
        if (page >= 0) slot = static_cast<int64_t>(page) * kPage + pos % kPage;
      }
    }
    a.slots[i] = slot;
    a.positions[i] = pos;
  }
}

// ---------------------------------------------------------------------------
// Cache write
// ---------------------------------------------------------------------------

constexpr int kAppendThreads = 256;
constexpr int kMinExp = -40, kMaxExp = 48;

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of the smallest power of two s with amax <= 448 s, clamped.
// 448 = 1.75 * 2^8, so the fraction is compared with that of 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kMinExp), kMaxExp);
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  const __half2_raw h =
      __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(__half2(h));
}

// Eight codes times `ratio`, rounded to e4m3 again.
__device__ __forceinline__ uint2 rescale8(uint2 w, float ratio) {
  const float2 a = e4m3x2_to_float2(w.x), b = e4m3x2_to_float2(w.x >> 16);
  const float2 c = e4m3x2_to_float2(w.y), d = e4m3x2_to_float2(w.y >> 16);
  return make_uint2(e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio),
                    e4m3x4(c.x * ratio, c.y * ratio, d.x * ratio, d.y * ratio));
}

// One CTA = one (block the step writes, KV head, K or V), which it owns alone:
// rows r0 .. r1 of the page are new, rows before r0 hold older tokens.  One
// pass: the new rows stay in registers between the maximum and the rounding.
// When the page's scale grows, its older codes are rescaled by the ratio
// (exact but for e4m3 subnormals, since scales are powers of two); rows
// behind r1 are left as they were.
__global__ void __launch_bounds__(kAppendThreads) append_kv_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float red[kAppendThreads / 32];
  const int g = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int64_t item = blockIdx.x;
  if (item >= __ldg(a.cu_blocks + a.batch)) return;
  const int b = find_sequence(a.cu_blocks, a.batch, item);
  const int64_t ctx = __ldg(a.context_lens + b);
  const int64_t seq = __ldg(a.seq_lens + b);
  const int64_t q0 = __ldg(a.cu_seqlens_q + b);
  const int64_t block = ctx / kPage + (item - __ldg(a.cu_blocks + b));
  const int64_t p0 = max(ctx, block * kPage), p1 = min(seq, (block + 1) * kPage);
  const int64_t t0 = q0 + (p0 - ctx);
  if (ctx < 0 || p1 <= p0 || t0 < 0 || t0 + (p1 - p0) > a.total_new) {
    // lengths that disagree with the packed rows: nothing is written
    if (threadIdx.x == 0) report(a.status, LS_DEVERR_SEQLENS);
    return;
  }
  const int64_t slot = __ldg(a.slots + t0);
  if (slot < 0) return;  // a token without a page
  const int64_t page = slot / kPage;
  if (page >= a.num_pages) {
    if (threadIdx.x == 0) report(a.status, LS_DEVERR_PAGE_INDEX);
    return;
  }
  const int r0 = static_cast<int>(p0 - block * kPage), r1 = static_cast<int>(p1 - block * kPage);
  const uint16_t* src = (is_v ? a.v : a.k) + g * 128;
  const int64_t row_stride = is_v ? a.v_stride : a.k_stride;
  uint8_t* codes = (is_v ? a.v_pages : a.k_pages) +
                   (page * a.num_groups + g) * static_cast<int64_t>(kPage * 128);
  float* scale = (is_v ? a.v_scale : a.k_scale) + page * a.num_groups + g;

  // 16 threads of 8 values per row, 16 rows per pass.
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  uint4 raw[4];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r + 16 * i;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row >= r0 && row < r1)
      raw[i] = __ldg(reinterpret_cast<const uint4*>(src + (t0 + (row - r0)) * row_stride) + c);
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // fmaxf passes over NaN: it is stored as NaN and leaves the scale alone
      amax = fmaxf(amax, fabsf(__uint_as_float(w[j] << 16)));
      amax = fmaxf(amax, fabsf(__uint_as_float(w[j] & 0xFFFF0000u)));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const float held = r0 > 0 ? *scale : 0.f;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) amax = fmaxf(amax, red[i]);
  float to = pow2(scale_exponent(amax));
  if (r0 > 0) {
    to = fminf(fmaxf(to, held), pow2(kMaxExp));
    if (to != held) {
      const float ratio = held / to;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r + 16 * i;
        if (row < r0) {
          uint2* w = reinterpret_cast<uint2*>(codes + row * 128) + c;
          *w = rescale8(*w, ratio);
        }
      }
    }
  }
  const float inv = 1.f / to;  // exact: a power of two
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r + 16 * i;
    if (row >= r0 && row < r1) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16) * inv;
        f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u) * inv;
      }
      reinterpret_cast<uint2*>(codes + row * 128)[c] =
          make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
    }
  }
  if (threadIdx.x == 0) *scale = to;
}

}  // namespace

cudaError_t launch_plan_pages(const PlanArgs& args, cudaStream_t stream) {
  const size_t smem = 2 * sizeof(int32_t) * (static_cast<size_t>(args.batch) + 1);
  if (smem > 40 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(
        plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
  }
  const int64_t want = (args.total_new + kPlanThreads - 1) / kPlanThreads;
  const unsigned grid = static_cast<unsigned>(want < 1 ? 1 : want > 148 * 2 ? 148 * 2 : want);
  plan_pages_kernel<<<grid, kPlanThreads, smem, stream>>>(args);
  return cudaGetLastError();
}

cudaError_t launch_append_kv(const AppendArgs& args, cudaStream_t stream) {
  // A request of n tokens writes at most n blocks and at most n / 64 + 2.
  const int64_t ragged = args.total_new / kPage + 2 * static_cast<int64_t>(args.batch);
  const int64_t blocks = args.total_new < ragged ? args.total_new : ragged;
  if (blocks == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(args.num_groups), 2);
  append_kv_kernel<<<grid, kAppendThreads, 0, stream>>>(args);
  return cudaGetLastError();
}

}  // namespace ls
