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

constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / 32;

__device__ __forceinline__ int32_t saturate32(int64_t x) {
  return static_cast<int32_t>(x > 0x7FFFFFFF ? 0x7FFFFFFF : x);
}

// Request b holds ctx tokens and gets n: blocks before the step, new blocks,
// blocks the step writes (the half-filled one included).  Lengths beyond 2^30
// are cut there: no table holds them.
struct PlanRow {
  int64_t ctx, n;
  int had, need, written;
  bool bad;
  __device__ __forceinline__ uint64_t blocks() const {
    return static_cast<uint64_t>(static_cast<uint32_t>(need)) << 32 |
           static_cast<uint32_t>(written);
  }
};

__device__ __forceinline__ PlanRow plan_row(const PlanArgs& a, int b) {
  PlanRow r;
  const int ctx = load_input(a.context_lens + b), n = load_input(a.new_lens + b);
  const int c = min(max(ctx, 0), 1 << 30), m = min(max(n, 0), 1 << 30);
  const int total = static_cast<int>((static_cast<uint32_t>(c) + m + kPage - 1) / kPage);
  r.ctx = c;
  r.n = m;
  r.bad = c != ctx || m != n || total > a.max_blocks;
  r.had = min((c + kPage - 1) / kPage, a.max_blocks);
  r.need = min(total, a.max_blocks) - r.had;
  r.written = m > 0 ? total - c / kPage : 0;
  return r;
}

// Every CTA computes the prefix sums over the requests by itself (shared
// memory, one block scan), so one launch does the whole step and no CTA waits
// for another; then the tokens are dealt to the threads, which find their
// request by binary search.  The thread of a new block's first token writes
// its block-table entry; a token in the half-filled old block reads that
// block's entry, which nobody writes.  Integer sums only: the result does not
// depend on the launch shape.  Latency bound, a chain of round trips (lengths,
// page, stores): 2.6 us of device time for 8 decode tokens, 4.1 for 1024, 8.3
// for the 727K tokens of 64 prompts (11.6 MB of results, 1.8 us at the copy
// rate; up to four CTAs per SM, as two took 9.1 and ten 10.8, since each repeats
// the sums; four neighbouring tokens a thread with 16-byte stores took 8.9, and
// 3.9 instead of 2.6 for small steps).
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* cu_q = plan_smem;                  // [batch + 1]
  int32_t* cu_need = plan_smem + a.batch + 1;  // [batch + 1]
  __shared__ int64_t warp_tok[kPlanWarps + 1];
  __shared__ uint64_t warp_blk[kPlanWarps + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool lead = blockIdx.x == 0;
  allow_next_launch();
  wait_for_inputs();

  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  // Two running sums: new tokens, and pages taken and written (32 bits each;
  // both stay below the tokens' sum, which is reported when it is too large).
  int64_t tok = 0;
  uint64_t blk = 0;
  bool bad = false;
  PlanRow r{};
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    r = plan_row(a, b);
    tok += r.n;
    blk += r.blocks();
    bad = bad || r.bad;
  }
  int64_t tok_run = tok;
  uint64_t blk_run = blk;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, tok_run, o);
    const uint64_t y = __shfl_up_sync(0xffffffffu, blk_run, o);
    if (lane >= o) {
      tok_run += x;
      blk_run += y;
    }
  }
  if (lane == 31) {
    warp_tok[warp] = tok_run;
    warp_blk[warp] = blk_run;
  }
  tok_run -= tok;
  blk_run -= blk;
  __syncthreads();
  if (warp == 0) {  // the warps' sums to sums of the warps before, and the total
    int64_t x = lane < kPlanWarps ? warp_tok[lane] : 0;
    uint64_t y = lane < kPlanWarps ? warp_blk[lane] : 0;
    const int64_t x0 = x;
    const uint64_t y0 = y;
#pragma unroll
    for (int o = 1; o < kPlanWarps; o <<= 1) {
      const int64_t xs = __shfl_up_sync(0xffffffffu, x, o);
      const uint64_t ys = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += xs;
        y += ys;
      }
    }
    if (lane < kPlanWarps) {
      warp_tok[lane] = x - x0;
      warp_blk[lane] = y - y0;
    }
    if (lane == kPlanWarps - 1) {
      warp_tok[kPlanWarps] = x;
      warp_blk[kPlanWarps] = y;
    }
  }
  __syncthreads();
  tok_run += warp_tok[warp];
  blk_run += warp_blk[warp];
  const int64_t tok_all = warp_tok[kPlanWarps];
  const uint64_t blk_all = warp_blk[kPlanWarps];
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    if (b1 - b0 > 1) r = plan_row(a, b);
    cu_q[b] = saturate32(tok_run);
    cu_need[b] = static_cast<int32_t>(blk_run >> 32);
    if (lead) {
      a.cu_seqlens_q[b] = saturate32(tok_run);
      a.cu_blocks[b] = static_cast<int32_t>(blk_run);
      a.seq_lens[b] = saturate32(r.ctx + r.n);
    }
    tok_run += r.n;
    blk_run += r.blocks();
  }
  const int64_t head_in = load_input(a.free_head);
  const int64_t head = min(max(head_in, int64_t{0}), static_cast<int64_t>(a.num_free));
  if (tid == 0) {
    const int64_t taken = static_cast<int64_t>(blk_all >> 32);
    cu_q[a.batch] = saturate32(tok_all);
    cu_need[a.batch] = static_cast<int32_t>(taken);
    if (lead) {
      a.cu_seqlens_q[a.batch] = saturate32(tok_all);
      a.cu_blocks[a.batch] = static_cast<int32_t>(blk_all);
      *a.free_head_out = static_cast<int32_t>(min(head + taken, static_cast<int64_t>(a.num_free)));
      if (tok_all > a.total_new) report(a.status, LS_DEVERR_SEQLENS);
      if (head != head_in || head + taken > a.num_free) report(a.status, LS_DEVERR_PAGES);
    }
  }
  if (lead && bad) report(a.status, LS_DEVERR_SEQLENS);
  __syncthreads();

  const int total_new = static_cast<int>(a.total_new);
  const int tokens = static_cast<int>(min(tok_all, a.total_new));
  for (uint32_t at = blockIdx.x * kPlanThreads + tid; at < static_cast<uint32_t>(total_new);
       at += gridDim.x * kPlanThreads) {
    const int i = static_cast<int>(at);
    int64_t slot = -1;
    int pos = 0;
    if (i < tokens) {
      // Last request whose first token is at or before i (empty requests share
      // their successor's offset and are passed over).
      int b = 0, top = a.batch - 1;
      while (b < top) {
        const int mid = (b + top + 1) >> 1;
        if (cu_q[mid] <= i) b = mid; else top = mid - 1;
      }
      const int ctx = min(max(load_input(a.context_lens + b), 0), 1 << 30);
      pos = ctx + (i - cu_q[b]);
      const int block = pos / kPage, had = (ctx + kPage - 1) / kPage;
      if (block < a.max_blocks) {
        int32_t* entry = a.block_table + static_cast<int64_t>(b) * a.max_blocks + block;
        int32_t page;
        if (block < had) {
          page = *entry;
        } else {
          const int64_t from = head + cu_need[b] + (block - had);
          page = from < a.num_free ? load_input(a.free_pages + from) : -1;
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

// What a CTA needs of the block it writes.
struct BlockRows {
  int64_t t0;      // packed row of its first new token
  int r0, r1;      // new rows of the page; rows before r0 hold older tokens
  enum { kNone, kFound, kBad } state;
};

// Finds the request of block `item` and the rows to write, by one warp.  The
// requests are probed 32 at a time with everything that is needed of them, so
// the usual call costs one round trip: up to 32 requests, or a decode step,
// where request b writes block b.  Other batches narrow the window first, 32
// ways a step.
__device__ __forceinline__ BlockRows find_block(const AppendArgs& a, int64_t item, int lane) {
  int lo = 0, n = a.batch;  // the request is one of [lo, lo + n)
  if (n > 32) {
    lo = static_cast<int>(min(max(item - 16, int64_t{0}), static_cast<int64_t>(n - 32)));
    n = 32;
  }
  const int total = load_input(a.cu_blocks + a.batch);
  for (int round = 0; round < 2; ++round) {
    const int b = lo + lane;
    int first = 0x7FFFFFFF, ctx = 0, seq = 0, q0 = 0;
    if (lane < n) {
      first = load_input(a.cu_blocks + b);
      ctx = load_input(a.context_lens + b);
      seq = load_input(a.seq_lens + b);
      q0 = load_input(a.cu_seqlens_q + b);
    }
    const int behind = load_input(a.cu_blocks + lo + n);
    const uint32_t at = __ballot_sync(0xffffffffu, lane < n && first <= item);
    if (item >= total) return {0, 0, 0, BlockRows::kNone};
    if (at != 0 && item < behind) {
      // the last of them: empty requests share their successor's offset
      const int src = 31 - __clz(at);
      first = __shfl_sync(0xffffffffu, first, src);
      ctx = __shfl_sync(0xffffffffu, ctx, src);
      seq = __shfl_sync(0xffffffffu, seq, src);
      q0 = __shfl_sync(0xffffffffu, q0, src);
      const int64_t block = ctx / kPage + (item - first);
      const int64_t p0 = max(static_cast<int64_t>(ctx), block * kPage);
      const int64_t p1 = min(static_cast<int64_t>(seq), (block + 1) * kPage);
      BlockRows r;
      r.t0 = q0 + (p0 - ctx);
      r.r0 = static_cast<int>(p0 - block * kPage);
      r.r1 = static_cast<int>(p1 - block * kPage);
      const bool ok = ctx >= 0 && q0 >= 0 && p1 > p0 && r.t0 + (p1 - p0) <= a.total_new;
      r.state = ok ? BlockRows::kFound : BlockRows::kBad;
      return r;
    }
    // Not in this window: narrow the side that holds it.
    int from = at != 0 ? lo + n : 0, to = at != 0 ? a.batch : lo;
    if (from >= to) break;
    while (to - from > 32) {
      const int step = (to - from + 31) / 32, probe = from + lane * step;
      const uint32_t before =
          __ballot_sync(0xffffffffu, probe < to && load_input(a.cu_blocks + probe) <= item);
      const int pick = before == 0 ? 0 : 31 - __clz(before);
      from += pick * step;
      to = min(from + step, to);
    }
    lo = from;
    n = to - from;
  }
  return {0, 0, 0, BlockRows::kBad};  // offsets that are no prefix sums
}

// One CTA = one (block the step writes, KV head), which it owns alone: half of
// its threads write K, half V.  Rows r0 .. r1 of the page are new, rows before
// r0 hold older tokens.  One pass: the new rows stay in registers between the
// maximum and the rounding.  When the page's scale grows, its older codes are
// rescaled by the ratio (exact but for e4m3 subnormals, since scales are powers
// of two); rows behind r1 are left as they were.  16 threads of 8 values per
// row; kThreads (per half) is 128 for pages that fill up and 32 for steps of a
// token or two, where the rest of a larger block would only wait.  Bound by HBM
// when pages fill up: a prompt of 131072 tokens, 134 MB read and 67 MB written,
// takes 35 us, 5.8 TB/s, 0.88 of the measured copy rate.  A step of one token a
// request is a chain of round trips (lengths, slot, scale): 2.2 us of device
// time for 8 requests, 2.8 for 512 (10.9 with a binary search for the request).
template <int kThreads>
__global__ void __launch_bounds__(2 * kThreads, kThreads == 128 ? 3 : 16) append_kv_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kWarps = kThreads / 32, kRows = kThreads / 16, kPasses = kPage / kRows;
  constexpr int kHeld = kPasses < 8 ? kPasses : kThreads == 32 ? 2 : 8;  // passes held in registers
  __shared__ float red[2][kWarps];
  const int lane = threadIdx.x & 31;
  const int g = blockIdx.y;
  const int is_v = threadIdx.x / kThreads;
  const int64_t item = blockIdx.x;
  allow_next_launch();
  wait_for_inputs();
  const BlockRows rows = find_block(a, item, lane);
  if (rows.state != BlockRows::kFound) {
    // lengths that disagree with the packed rows: nothing is written
    if (rows.state == BlockRows::kBad && threadIdx.x == 0) report(a.status, LS_DEVERR_SEQLENS);
    return;
  }
  const int64_t slot = load_input(a.slots + rows.t0);
  const int r0 = rows.r0, r1 = rows.r1;
  const uint16_t* src = (is_v ? a.v : a.k) + g * 128;
  const int64_t row_stride = is_v ? a.v_stride : a.k_stride;
  const int c = threadIdx.x & 15, r = (threadIdx.x % kThreads) >> 4;
  const auto load = [&](int row) {
    if (row >= r1) return make_uint4(0, 0, 0, 0);
    return load_input(
        reinterpret_cast<const uint4*>(src + (rows.t0 + (row - r0)) * row_stride) + c);
  };
  // Rows r0 + r, r0 + r + kRows, ...: the first passes stay in registers, the
  // others (kThreads == 32, more than 4 new rows) are read again.
  const int passes = (r1 - r0 + kRows - 1) / kRows;
  uint4 raw[kHeld];
  float amax = 0.f;
  const auto track = [&](const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // fmaxf passes over NaN: it is stored as NaN and leaves the scale alone
      amax = fmaxf(amax, fabsf(__uint_as_float(w[j] << 16)));
      amax = fmaxf(amax, fabsf(__uint_as_float(w[j] & 0xFFFF0000u)));
    }
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) raw[i] = load(r0 + r + i * kRows);
#pragma unroll
  for (int i = 0; i < kHeld; ++i) track(raw[i]);
  for (int i = kHeld; i < passes; ++i) track(load(r0 + r + i * kRows));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (slot < 0) return;  // a token without a page
  const int64_t page = slot / kPage;
  if (page >= a.num_pages) {
    if (threadIdx.x == 0) report(a.status, LS_DEVERR_PAGE_INDEX);
    return;
  }
  uint8_t* codes = (is_v ? a.v_pages : a.k_pages) +
                   (page * a.num_groups + g) * static_cast<int64_t>(kPage * 128);
  float* scale = (is_v ? a.v_scale : a.k_scale) + page * a.num_groups + g;
  const float held = r0 > 0 ? *scale : 0.f;
  if (kWarps > 1) {
    if (lane == 0) red[is_v][(threadIdx.x % kThreads) >> 5] = amax;
    __syncthreads();  // also: every thread has read the old scale
#pragma unroll
    for (int i = 0; i < kWarps; ++i) amax = fmaxf(amax, red[is_v][i]);
  } else {
    __syncwarp();
  }
  float to = pow2(scale_exponent(amax));
  if (r0 > 0) {
    to = fminf(fmaxf(to, held), pow2(kMaxExp));
    if (to != held) {
      const float ratio = held / to;
      for (int row = r; row < r0; row += kRows) {
        uint2* w = reinterpret_cast<uint2*>(codes + row * 128) + c;
        *w = rescale8(*w, ratio);
      }
    }
  }
  const float inv = 1.f / to;  // exact: a power of two
  const auto store = [&](int row, const uint4& x) {
    if (row >= r1) return;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16) * inv;
      f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u) * inv;
    }
    reinterpret_cast<uint2*>(codes + row * 128)[c] =
        make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) store(r0 + r + i * kRows, raw[i]);
  for (int i = kHeld; i < passes; ++i) store(r0 + r + i * kRows, load(r0 + r + i * kRows));
  if (threadIdx.x % kThreads == 0) *scale = to;
}

}  // namespace

cudaError_t launch_plan_pages(const PlanArgs& args, cudaStream_t stream) {
  const auto smem_bytes = [](int batch) {
    return 2 * sizeof(int32_t) * (static_cast<size_t>(batch) + 1);
  };
  // Set once, to what the largest batch takes: calls of other threads rely on it.
  static std::atomic<uint64_t> done[4];
  const cudaError_t err = once_per_device(done, [&] {
    return cudaFuncSetAttribute(plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem_bytes(LS_MAX_PLAN_BATCH)));
  });
  if (err != cudaSuccess) return err;
  const int64_t want = (args.total_new + kPlanThreads - 1) / kPlanThreads;
  const unsigned grid = static_cast<unsigned>(want < 1 ? 1 : want > 148 * 4 ? 148 * 4 : want);
  return launch_early(plan_pages_kernel, dim3(grid), dim3(kPlanThreads), smem_bytes(args.batch),
                      stream, args);
}

cudaError_t launch_append_kv(const AppendArgs& args, cudaStream_t stream) {
  // A request of n tokens writes at most n blocks and at most n / 64 + 2.
  const int64_t ragged = args.total_new / kPage + 2 * static_cast<int64_t>(args.batch);
  const int64_t blocks = args.total_new < ragged ? args.total_new : ragged;
  if (blocks == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(args.num_groups));
  // Up to two tokens a request on average: single warps (512 tokens of 512
  // requests 2.8 us against 7.4; a prompt of 131072 tokens 57 us against 35).
  // Idle requests count: a prompt of 16384 tokens beside 8191 of them takes the
  // single warps, 35 us, where alone it takes 6.
  return args.total_new <= 2 * static_cast<int64_t>(args.batch)
             ? launch_early(append_kv_kernel<32>, grid, dim3(64), 0, stream, args)
             : launch_early(append_kv_kernel<128>, grid, dim3(256), 0, stream, args);
}

}  // namespace ls
