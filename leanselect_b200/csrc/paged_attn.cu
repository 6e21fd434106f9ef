// Attention over the 8-bit paged cache (decode steps, short drafts, page-listed chunks).
//
// For query row t of request b at position p and head h of group g:
//   out = sum_k w_k v_k / sum_k w_k,  w_k = exp(scale q.k_k)
// over the keys of the row's pages at positions <= p, with k = ks * code and
// v = vs * code (e4m3 codes, one ks and vs per (page, group)).
//
// A (token, group) row reads 16 KB of codes per page for 16 heads: the path
// is bound by moving pages, from HBM when caches are long and from L2 when
// rows share pages.  So the codes go straight from the TMA ring into f16
// fragments (e4m3 converts exactly), and all scales are folded in elsewhere:
//   * ks multiplies the scores' factor, per page;
//   * vs is folded into the exponent: P' = 2^(x + log2 vs - M), so that
//     sum P' code needs no page factor, and the row sum takes P' / vs;
//   * q is scaled per row by a power of two into f16's range.
// M is a lazily raised reference (it moves only when x + log2 vs exceeds it
// by 14 binades; it is set 6 below the maximum), so P' <= 2^14 holds f16's 11
// bits down to 2^-20 of the largest.  Sums and accumulators are fp32.
//
// Work split.  All rows' page lists are laid end to end and cut into equal
// ranges, one per CTA, two CTAs per SM: ragged batches stay balanced and one
// long row fills the GPU.  A row inside one range is written at once; the
// parts of a row cut by range borders go to a workspace and
// paged_merge_kernel joins them.  The cut depends on the shapes and lengths
// alone, and no sum uses atomics, so equal calls give equal bits.
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.h"
#include "page_list.cuh"

namespace ls {
namespace {

constexpr int kPage = LS_PAGE_TOKENS;
constexpr int kStages = 4;
constexpr int kTileBytes = kPage * 128;      // one page of one group, K or V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kConsumers = 4;                // warps; each owns 16 keys of every page
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr float kSlack = 14.f, kHeadroom = 6.f;  // binades, see above
constexpr float kMinScale = 0x1p-40f, kMaxScale = 0x1p48f;

enum StageFlag { kFirst = 1, kLast = 2, kData = 4, kStop = 8 };

// What a consumer needs to know of one ring stage.
struct StageMeta {
  int flags;
  int key0;        // position of the page's first key
  float k_scale, v_log2, v_inv;
  int limit;       // last visible position (-1: none)
  int token, group;
  int part;        // workspace part, -1: the row is whole in this CTA
};

struct PagedSmem {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t join;   // the consumer warps' meeting point, bounded like every wait
  StageMeta meta[kStages];
  int abort_flag;
  int64_t scan[kConsumers + 1];
  int32_t start_b;
  int64_t start_off;
  int32_t pages[LS_MAX_TOPK];
  float m_part[kConsumers][16];
  float l_part[kConsumers][16];
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two e4m3 codes (the low or the high half of a word) as f16x2.
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` in a 128B-swizzled box.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) {
  return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}

// Pages a request of `len` cached tokens is scheduled with: at least one, so
// that every row is visited and written.
__device__ __forceinline__ int64_t scheduled_pages(int64_t len) {
  return len > 0 ? (len + kPage - 1) / kPage : 1;
}

// A request as the kernels see it: lengths that would leave the packed rows
// or the block table are cut and reported.
struct Request {
  int64_t q0;
  int nq, len;
  bool bad;
};

__device__ __forceinline__ Request load_request(const PagedAttnArgs& a, int b) {
  Request r;
  r.q0 = __ldg(a.cu_q + b);
  int64_t nq = __ldg(a.cu_q + b + 1) - r.q0;
  int64_t len = __ldg(a.seq_lens + b);
  const int64_t most = static_cast<int64_t>(a.max_blocks) * kPage;
  r.bad = r.q0 < 0 || nq < 0 || r.q0 + nq > a.total_q || len < 0 || len > most;
  if (r.q0 < 0 || nq < 0 || r.q0 + nq > a.total_q) nq = 0;
  r.nq = static_cast<int>(nq);
  r.len = static_cast<int>(min(max(len, int64_t{0}), most));
  return r;
}

// First work unit of CTA i when `work` units are cut into n ranges, and the
// CTA that unit w belongs to.
__device__ __forceinline__ int64_t range_start(int64_t i, int64_t work, int64_t n) {
  return i * work / n;
}
__device__ __forceinline__ int range_of(int64_t w, int64_t work, int64_t n) {
  return static_cast<int>(((w + 1) * n + work - 1) / work - 1);
}

__global__ void __launch_bounds__(kThreads, 2) paged_attn_kernel(const __grid_constant__ PagedAttnArgs args) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* stages = smem;
  float* acc = reinterpret_cast<float*>(stages + kStages * kStageBytes);  // [warps][16][128]
  PagedSmem* sm = reinterpret_cast<PagedSmem*>(acc + kConsumers * 16 * 128);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = args.num_groups;
  const bool listed = args.topk > 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm->full[s], 1);
      mbar_init(&sm->empty[s], kConsumers);
    }
    mbar_init(&sm->join, kConsumers);
    sm->abort_flag = 0;
    fence_barrier_init();
  }

  // ---- the work of all rows, and where this CTA's range starts
  // listed: row r = (group, token) has `topk` units, ordered group-major.
  // dense: request by request, (group, token) rows of scheduled_pages units.
  int64_t work;
  int64_t rows_listed = 0;
  if (listed) {
    const int64_t rows = min(max(static_cast<int64_t>(__ldg(args.cu_q + args.batch)), int64_t{0}),
                             args.total_q);
    rows_listed = rows;
    work = rows * G * args.topk;
    __syncthreads();
  } else {
    const int per = (args.batch + kThreads - 1) / kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, args.batch);
    const int b1 = min(b0 + per, args.batch);
    int64_t own = 0;
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
      const Request r = load_request(args, b);
      own += static_cast<int64_t>(r.nq) * G * scheduled_pages(r.len);
      bad = bad || r.bad;
    }
    if (bad && blockIdx.x == 0) report(args.status, LS_DEVERR_SEQLENS);
    int64_t x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sm->scan[warp] = x;
    __syncthreads();
    int64_t before = x - own;
    work = 0;
    for (int w = 0; w < kConsumers + 1; ++w) {
      if (w < warp) before += sm->scan[w];
      work += sm->scan[w];
    }
    const int64_t n_all = min(static_cast<int64_t>(gridDim.x), work);
    const int64_t w0 = blockIdx.x < n_all ? range_start(blockIdx.x, work, n_all) : -1;
    if (w0 >= before && w0 < before + own) {
      int64_t at = before;
      for (int b = b0; b < b1; ++b) {
        const Request r = load_request(args, b);
        const int64_t units = static_cast<int64_t>(r.nq) * G * scheduled_pages(r.len);
        if (w0 < at + units) {
          sm->start_b = b;
          sm->start_off = w0 - at;
          break;
        }
        at += units;
      }
    }
    __syncthreads();
  }
  const int64_t n_ctas = min(static_cast<int64_t>(gridDim.x), work);
  int2* header = args.headers + blockIdx.x;
  if (blockIdx.x >= n_ctas) {
    if (threadIdx.x == 0) *header = make_int2(-1, 0);
    return;
  }
  const int64_t w_begin = range_start(blockIdx.x, work, n_ctas);
  const int64_t w_end = range_start(blockIdx.x + 1, work, n_ctas);
  volatile int* abort_flag = &sm->abort_flag;

  if (warp == kConsumers) {
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      tma_prefetch_desc(&args.tm_k);
      tma_prefetch_desc(&args.tm_v);
    }
    int fill = 0;   // stages filled so far
    bool ok = true;
    int2 head = make_int2(-1, 0);
    int64_t w = w_begin;
    int b = listed ? 0 : sm->start_b;
    int64_t off = listed ? 0 : sm->start_off;  // dense: unit inside request b
    while (w < w_end && ok) {
      // ---- the row that unit w belongs to
      int64_t units, a, token;
      int g;
      Request req;
      if (listed) {
        units = args.topk;
        const int64_t row = w / units;
        a = w % units;
        g = static_cast<int>(row / rows_listed);
        token = row % rows_listed;
        b = find_sequence(args.cu_q, args.batch, token);
        req = load_request(args, b);
        if (req.bad && lane == 0) report(args.status, LS_DEVERR_SEQLENS);
      } else {
        if (b >= args.batch) break;  // lengths changed under the kernel
        req = load_request(args, b);
        units = scheduled_pages(req.len);
        if (off >= units * req.nq * G) {
          off = 0;
          ++b;
          continue;
        }
        const int64_t row = off / units;
        a = off % units;
        g = static_cast<int>(row / req.nq);
        token = req.q0 + row % req.nq;
      }
      const int64_t e = min(units, a + (w_end - w));
      const int t_rel = static_cast<int>(token - req.q0);
      int limit = req.len - 1;
      if (args.causal) limit = min(limit, req.len - req.nq + t_rel);
      if (t_rel < 0 || t_rel >= req.nq) limit = -1;
      const int whole = a == 0 && e == units;
      const int part = whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (a == 0 ? 1 : 0);
      if (a == 0 && e < units)
        head = make_int2(static_cast<int>(token * G + g),
                         range_of(w - a + units - 1, work, n_ctas));

      // ---- its pages, and this CTA's share of them
      int n_row;
      if (listed) {
        const int32_t* list = args.topk_idx + (static_cast<int64_t>(g) * args.total_q + token) *
                                                  args.topk;
        const int n_pages = (req.len + kPage - 1) / kPage;
        int32_t v[4];
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = 32 * r + lane;
          const int32_t p = pos < args.topk ? __ldg(list + pos) : -1;
          bad = bad || p >= n_pages;
          v[r] = (p >= 0 && p < n_pages && static_cast<int64_t>(p) * kPage <= limit) ? p
                                                                                  : kPageSentinel;
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0) report(args.status, LS_DEVERR_PAGE_INDEX);
        __syncwarp();
        n_row = warp_compact_pages(v, sm->pages, lane);
        __syncwarp();
      } else {
        n_row = limit >= 0 ? limit / kPage + 1 : 0;
      }
      const int lo = static_cast<int>(a * n_row / units), hi = static_cast<int>(e * n_row / units);

      const int32_t* table = args.block_table + static_cast<int64_t>(b) * args.max_blocks;
      bool first = true;
      for (int base = lo; base < hi && ok; base += 32) {
        // 32 pages' table entries and scales at once, one per lane.
        const int i = base + lane;
        int32_t logical = -1, page = -1;
        float ks = 0.f, vs = 1.f;
        if (i < hi) {
          logical = listed ? sm->pages[i] : i;
          page = __ldg(table + logical);
          if (page < 0 || page >= args.num_pages) {
            page = -1;
            report(args.status, LS_DEVERR_PAGE_INDEX);
          } else {
            const int64_t at = static_cast<int64_t>(page) * G + g;
            ks = __ldg(args.k_scale + at);
            vs = __ldg(args.v_scale + at);
          }
        }
        ks = fminf(fmaxf(ks, kMinScale), kMaxScale);
        vs = fminf(fmaxf(vs, kMinScale), kMaxScale);
        const float v_log2 = __log2f(vs), v_inv = 1.f / vs;
        const int n = min(32, hi - base);
        for (int j = 0; j < n; ++j) {
          const int32_t lp = __shfl_sync(0xffffffffu, logical, j);
          const int32_t pp = __shfl_sync(0xffffffffu, page, j);
          const float kj = __shfl_sync(0xffffffffu, ks, j);
          const float lj = __shfl_sync(0xffffffffu, v_log2, j);
          const float ij = __shfl_sync(0xffffffffu, v_inv, j);
          const bool last = base + j + 1 == hi;
          if (pp < 0 && !last && !first) continue;
          const int s = fill % kStages;
          if (lane == 0) {
            ok = mbar_wait(&sm->empty[s], ((fill / kStages) & 1) ^ 1, args.status, abort_flag);
            if (ok) {
              StageMeta m;
              m.flags = (first ? kFirst : 0) | (last ? kLast : 0) | (pp >= 0 ? kData : 0);
              m.key0 = lp * kPage;
              m.k_scale = kj;
              m.v_log2 = lj;
              m.v_inv = ij;
              m.limit = limit;
              m.token = static_cast<int>(token);
              m.group = g;
              m.part = part;
              sm->meta[s] = m;
              if (pp >= 0) {
                uint8_t* st = stages + s * kStageBytes;
                const int32_t y = (pp * G + g) * kPage;
                mbar_arrive_expect_tx(&sm->full[s], kStageBytes);
                tma_load_2d(st, &args.tm_k, &sm->full[s], 0, y);
                tma_load_2d(st + kTileBytes, &args.tm_v, &sm->full[s], 0, y);
              } else {
                mbar_arrive(&sm->full[s]);
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
          ++fill;
          first = false;
        }
      }
      if (ok && lo >= hi) {
        // A share without pages still writes its row (or its empty part).
        const int s = fill % kStages;
        if (lane == 0) {
          ok = mbar_wait(&sm->empty[s], ((fill / kStages) & 1) ^ 1, args.status, abort_flag);
          if (ok) {
            StageMeta m{};
            m.flags = kFirst | kLast;
            m.limit = limit;
            m.token = static_cast<int>(token);
            m.group = g;
            m.part = part;
            sm->meta[s] = m;
            mbar_arrive(&sm->full[s]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (ok) ++fill;
      }
      off += e - a;
      w += e - a;
    }
    if (lane == 0) {
      const int s = fill % kStages;
      if (ok) ok = mbar_wait(&sm->empty[s], ((fill / kStages) & 1) ^ 1, args.status, abort_flag);
      if (ok) {
        sm->meta[s].flags = kStop;
        mbar_arrive(&sm->full[s]);
      }
      *header = ok ? head : make_int2(-1, 0);
      if (!ok) {
        // Copies in flight must land before the CTA gives up its memory.
        for (int k = max(0, fill - kStages); k < fill; ++k)
          mbar_wait(&sm->full[k % kStages], (k / kStages) & 1, nullptr, nullptr);
      }
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int gq = lane >> 2, c = lane & 3;  // fragment row / key, and quad lane
  const int Hg = args.heads_per_group;
  uint32_t qa[8][4];
  float o[16][4];
  float f0 = 0.f, f1 = 0.f;                 // score factors of rows gq and gq + 8
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const int key_base = warp * 16;
  uint32_t joins = 0;
  // All consumer warps meet; false once a wait has given up anywhere (the
  // row then stays unwritten).
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm->join);
    return mbar_wait(&sm->join, joins++ & 1, args.status, abort_flag);
  };

  for (int i = 0;; ++i) {
    const int s = i % kStages;
    if (!mbar_wait(&sm->full[s], (i / kStages) & 1, args.status, abort_flag)) return;
    const StageMeta meta = sm->meta[s];
    if (meta.flags & kStop) return;

    if (meta.flags & kFirst) {
      // Q fragments.  The 32 dims a quad lane holds of a key row (32c ..) are
      // the contraction's order: k-step kk takes dims 32c + 4kk .. + 3.
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int h = gq + 8 * half;
        uint4 raw[4];
        float amax = 0.f;
        const uint4* src = reinterpret_cast<const uint4*>(
            args.q + (static_cast<int64_t>(meta.token) * args.num_heads + meta.group * Hg + h) * 128 +
            32 * c);
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[k] = h < Hg ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^-e with e the exponent of the row's largest value, kept to where
        // the factor stays normal under every page scale: f16 then holds
        // every value to 2^-25 of the largest.
        const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -60), 78);
        const float down = __int_as_float((127 - e) << 23);
        const float factor = args.scale_log2 * __int_as_float((127 + e) << 23);
        if (half == 0) f0 = factor; else f1 = factor;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            qa[2 * k + (j >> 1)][half + 2 * (j & 1)] =
                pack_f16x2(bf16_lo(w[j]) * down, bf16_hi(w[j]) * down);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
    }

    const int page_key0 = meta.key0 + key_base;
    if ((meta.flags & kData) && page_key0 <= meta.limit) {
      const uint32_t st = smem_u32(stages + s * kStageBytes);
      // ---- S = Q K^T for this warp's 16 keys, two accumulator sets a tile
      float sc[2][4], sh[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
        sh[n][0] = sh[n][1] = sh[n][2] = sh[n][3] = 0.f;
        const int key = key_base + n * 8 + gq;
        const uint4 ka = lds128(st + sw128(key, 2 * c));
        const uint4 kb = lds128(st + sw128(key, 2 * c + 1));
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          mma_f16_16816(sc[n], qa[kk], f16x2_lo(wa[kk]), f16x2_hi(wa[kk]));
          mma_f16_16816(sh[n], qa[kk + 4], f16x2_lo(wb[kk]), f16x2_hi(wb[kk]));
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] += sh[n][e];
      // ---- keys past the limit
      const bool ragged = page_key0 + 15 > meta.limit;
      if (ragged) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (page_key0 + n * 8 + 2 * c + (e & 1) > meta.limit) sc[n][e] = -INFINITY;
      }
      // ---- online softmax in the log2 domain
      const float k0 = f0 * meta.k_scale, k1 = f1 * meta.k_scale;
      float x0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])) * k0 + meta.v_log2;
      float x1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3])) * k1 + meta.v_log2;
      if (__any_sync(0xffffffffu, x0 > m0 + kSlack || x1 > m1 + kSlack)) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        float a0 = 1.f, a1 = 1.f;
        if (x0 > m0 + kSlack) {
          a0 = ex2(m0 - (x0 - kHeadroom));
          m0 = x0 - kHeadroom;
        }
        if (x1 > m1 + kSlack) {
          a1 = ex2(m1 - (x1 - kHeadroom));
          m1 = x1 - kHeadroom;
        }
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= a0;
          o[j][1] *= a0;
          o[j][2] *= a1;
          o[j][3] *= a1;
        }
      }
      const float d0 = meta.v_log2 - (m0 == -INFINITY ? 0.f : m0);
      const float d1 = meta.v_log2 - (m1 == -INFINITY ? 0.f : m1);
      float p[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        p[n][0] = ex2(fmaf(sc[n][0], k0, d0));
        p[n][1] = ex2(fmaf(sc[n][1], k0, d0));
        p[n][2] = ex2(fmaf(sc[n][2], k1, d1));
        p[n][3] = ex2(fmaf(sc[n][3], k1, d1));
      }
      l0 = fmaf((p[0][0] + p[0][1]) + (p[1][0] + p[1][1]), meta.v_inv, l0);
      l1 = fmaf((p[0][2] + p[0][3]) + (p[1][2] + p[1][3]), meta.v_inv, l1);
      uint32_t pa[4];
      pa[0] = pack_f16x2(p[0][0], p[0][1]);
      pa[1] = pack_f16x2(p[0][2], p[0][3]);
      pa[2] = pack_f16x2(p[1][0], p[1][1]);
      pa[3] = pack_f16x2(p[1][2], p[1][3]);
      // ---- O += P V.  A quad lane's four keys (2c, 2c+1, 2c+8, 2c+9), 16
      // dims each (16 gq ..): accumulator tile j holds dim 16 n + j.
      const uint32_t vt = st + kTileBytes;
      uint32_t vw[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int in_warp = 2 * c + (r & 1) + 8 * (r >> 1);
        const uint4 v = lds128(vt + sw128(key_base + in_warp, gq));
        vw[r][0] = v.x;
        vw[r][1] = v.y;
        vw[r][2] = v.z;
        vw[r][3] = v.w;
        // Rows past the limit may hold anything, NaN codes among it.
        if (ragged && page_key0 + in_warp > meta.limit)
          vw[r][0] = vw[r][1] = vw[r][2] = vw[r][3] = 0;
      }
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const uint32_t lo0 = __byte_perm(vw[0][q4], vw[1][q4], 0x5140);
        const uint32_t hi0 = __byte_perm(vw[0][q4], vw[1][q4], 0x7362);
        const uint32_t lo1 = __byte_perm(vw[2][q4], vw[3][q4], 0x5140);
        const uint32_t hi1 = __byte_perm(vw[2][q4], vw[3][q4], 0x7362);
        mma_f16_16816(o[4 * q4], pa, f16x2_lo(lo0), f16x2_lo(lo1));
        mma_f16_16816(o[4 * q4 + 1], pa, f16x2_hi(lo0), f16x2_hi(lo1));
        mma_f16_16816(o[4 * q4 + 2], pa, f16x2_lo(hi0), f16x2_lo(hi1));
        mma_f16_16816(o[4 * q4 + 3], pa, f16x2_hi(hi0), f16x2_hi(hi1));
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm->empty[s]);
    if (!(meta.flags & kLast)) continue;

    // ---- end of this CTA's share of the row: join the four warps
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (c == 0) {
      sm->m_part[warp][gq] = m0;
      sm->m_part[warp][gq + 8] = m1;
      sm->l_part[warp][gq] = l0;
      sm->l_part[warp][gq + 8] = l1;
    }
    if (!meet()) return;
    float mt0 = -INFINITY, mt1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) {
      mt0 = fmaxf(mt0, sm->m_part[w][gq]);
      mt1 = fmaxf(mt1, sm->m_part[w][gq + 8]);
    }
    const float s0 = m0 == -INFINITY ? 0.f : ex2(m0 - mt0);
    const float s1 = m1 == -INFINITY ? 0.f : ex2(m1 - mt1);
    // float4 i of a thread's 32 dims sits at 8c + (i ^ (c, row parity)): the
    // eight lanes of a store or load phase touch eight bank groups.
    float4* mine = reinterpret_cast<float4*>(acc) + warp * 16 * 32;
    const int swz = c | ((gq & 1) << 2);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = k >> 2, j = 4 * (k & 3);
      mine[gq * 32 + 8 * c + (k ^ swz)] = make_float4(o[j][e] * s0, o[j + 1][e] * s0,
                                                      o[j + 2][e] * s0, o[j + 3][e] * s0);
      mine[(gq + 8) * 32 + 8 * c + (k ^ swz)] =
          make_float4(o[j][2 + e] * s1, o[j + 1][2 + e] * s1, o[j + 2][2 + e] * s1,
                      o[j + 3][2 + e] * s1);
    }
    if (!meet()) return;
    {
      const int row = threadIdx.x >> 3, seg = threadIdx.x & 7;
      float mt = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) mt = fmaxf(mt, sm->m_part[w][row]);
#pragma unroll
      for (int w = 0; w < kConsumers; ++w)
        lt += sm->m_part[w][row] == -INFINITY
                  ? 0.f
                  : sm->l_part[w][row] * ex2(sm->m_part[w][row] - mt);
      float4 sum[4];
      const int rswz = (seg >> 1) | ((row & 1) << 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sum[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int at = row * 32 + 8 * (seg >> 1) + ((4 * (seg & 1) + k) ^ rswz);
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) {
          const float4 x = reinterpret_cast<const float4*>(acc)[w * 16 * 32 + at];
          sum[k].x += x.x;
          sum[k].y += x.y;
          sum[k].z += x.z;
          sum[k].w += x.w;
        }
      }
      if (row < Hg) {
        if (meta.part >= 0) {
          const int64_t prow = static_cast<int64_t>(meta.part) * 16 + row;
          float4* dst = reinterpret_cast<float4*>(args.part_o + prow * 128) + 4 * seg;
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = sum[k];
          if (seg == 0)
            *reinterpret_cast<float2*>(args.part_ml + prow * 2) = make_float2(mt, lt);
        } else {
          const int h = meta.group * Hg + row;
          const float f = mt == -INFINITY ? 0.f : 1.f / lt;
          uint4 packed[2];
          uint32_t* pw = reinterpret_cast<uint32_t*>(packed);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            pw[2 * k] = pack_bf16x2(sum[k].x * f, sum[k].y * f);
            pw[2 * k + 1] = pack_bf16x2(sum[k].z * f, sum[k].w * f);
          }
          uint4* dst = reinterpret_cast<uint4*>(
              args.out + (static_cast<int64_t>(meta.token) * args.num_heads + h) * 128 + 16 * seg);
          dst[0] = packed[0];
          dst[1] = packed[1];
          if (args.lse != nullptr && seg == 0)
            args.lse[static_cast<int64_t>(h) * args.total_q + meta.token] =
                mt == -INFINITY ? INFINITY : (mt + log2f(lt)) * 0.69314718055994531f;
        }
      }
    }
    // The next row's partials must not overwrite what is still being read.
    if (!meet()) return;
  }
}

size_t paged_smem_bytes() {
  return 1024 + kStages * kStageBytes + kConsumers * 16 * 128 * sizeof(float) + sizeof(PagedSmem);
}

// Joins the parts of the row that CTA j of the attention kernel began and did
// not finish: its second part and the first parts of CTAs j + 1 .. hi.  One
// block per (j, head); warp w takes parts w, w + 8, ...
constexpr int kMergeWarps = 8;

__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_kernel(const __grid_constant__ PagedAttnArgs args) {
  const int j = blockIdx.x, h = blockIdx.y;
  const int2 head = args.headers[j];
  if (head.x < 0) return;
  __shared__ float4 sum[kMergeWarps][32];
  __shared__ float m_w[kMergeWarps], l_w[kMergeWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = head.y - j + 1;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < n; i += kMergeWarps) {
    const int64_t part = i == 0 ? 2 * j + 1 : 2 * (j + i);
    const int64_t prow = part * 16 + h;
    const float2 ml = *reinterpret_cast<const float2*>(args.part_ml + prow * 2);
    const float4 x = reinterpret_cast<const float4*>(args.part_o + prow * 128)[lane];
    if (ml.x == -INFINITY) continue;
    const float mx = fmaxf(m, ml.x);
    const float a = m == -INFINITY ? 0.f : ex2(m - mx), b = ex2(ml.x - mx);
    acc.x = acc.x * a + x.x * b;
    acc.y = acc.y * a + x.y * b;
    acc.z = acc.z * a + x.z * b;
    acc.w = acc.w * a + x.w * b;
    l = l * a + ml.y * b;
    m = mx;
  }
  sum[warp][lane] = acc;
  if (lane == 0) {
    m_w[warp] = m;
    l_w[warp] = l;
  }
  __syncthreads();
  if (warp != 0) return;
  float mt = -INFINITY, lt = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) mt = fmaxf(mt, m_w[w]);
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) {
    if (m_w[w] == -INFINITY) continue;
    const float a = ex2(m_w[w] - mt);
    const float4 x = sum[w][lane];
    t.x = fmaf(x.x, a, t.x);
    t.y = fmaf(x.y, a, t.y);
    t.z = fmaf(x.z, a, t.z);
    t.w = fmaf(x.w, a, t.w);
    lt = fmaf(l_w[w], a, lt);
  }
  const float f = mt == -INFINITY ? 0.f : 1.f / lt;
  const int64_t token = head.x / args.num_groups;
  const int hh = (head.x % args.num_groups) * args.heads_per_group + h;
  uint2 packed;
  packed.x = pack_bf16x2(t.x * f, t.y * f);
  packed.y = pack_bf16x2(t.z * f, t.w * f);
  reinterpret_cast<uint2*>(args.out + (token * args.num_heads + hh) * 128)[lane] = packed;
  if (args.lse != nullptr && lane == 0)
    args.lse[static_cast<int64_t>(hh) * args.total_q + token] =
        mt == -INFINITY ? INFINITY : (mt + log2f(lt)) * 0.69314718055994531f;
}

}  // namespace

cudaError_t launch_paged_attn(const PagedAttnArgs& args, int ctas, cudaStream_t stream) {
  const size_t smem = paged_smem_bytes();
  const cudaError_t err = cudaFuncSetAttribute(
      paged_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (err != cudaSuccess) return err;
  paged_attn_kernel<<<ctas, kThreads, smem, stream>>>(args);
  paged_merge_kernel<<<dim3(ctas, args.heads_per_group), 32 * kMergeWarps, 0, stream>>>(args);
  return cudaGetLastError();
}

}  // namespace ls
