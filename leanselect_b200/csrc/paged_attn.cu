// Attention over the 8-bit paged cache (decode steps, short drafts, page-listed chunks).
//
// For query row t of request b at position p and head h of group g:
//   out = sum_k w_k v_k / sum_k w_k,  w_k = exp(scale q.k_k)
// over the keys of the row's pages at positions <= p, with k = ks * code and
// v = vs * code (e4m3 codes, one ks and vs per (page, group)).
//
// A tile of 16 query rows (the heads of one group; with fewer than 16 heads
// those of several tokens of a request) reads 16 KB of codes per page and
// does 0.5 MFLOP with them: on long caches HBM bounds it, on lists of pages
// that rows share the tensor pipe.  So the codes go straight from the TMA
// ring into f16 fragments (e4m3 converts exactly; the 8-bit form of mma.sync
// took 1.35 times as long here), and all scales are folded in elsewhere:
//   * ks multiplies the scores' factor, per page;
//   * vs is folded into the exponent: P' = 2^(x + log2 vs - M), so that
//     sum P' code needs no page factor, and the row sum takes P' / vs;
//   * q is scaled per row by a power of two into f16's range.
// M is a lazily raised reference (it moves only when x + log2 vs exceeds it
// by 14 binades; it is set 6 below the maximum), so P' <= 2^14 holds f16's 11
// bits down to 2^-20 of the largest: rounding the weights to f16 costs half a
// step of 2^-11, less than the bf16 output.  Sums and accumulators are fp32.
//
// Work split.  All tiles' pages are laid end to end and cut into equal ranges,
// two per SM: ragged batches stay balanced and one long row fills the GPU.  A
// tile inside one range is written at once; the parts of a tile cut by range
// borders go to a workspace and a second kernel joins them.  The cut depends
// on the shapes and lengths alone, and no sum uses atomics, so equal calls
// give equal bits.
//
// One CTA per SM holds two teams of four consumer warps with 216 registers a
// thread (each has a range of its own) and four producer warps with 72: the
// accumulators of a 16 x 128 tile, the queries and a page's fragments stay in
// registers, where two CTAs per SM would leave 168 a thread.  Two warps of a team share a page, 32 keys each,
// and the pairs take alternate pages from rings of their own: 64 KB in flight
// per team, and half the waits and votes per key of 16-key shares.
//
// Measured (CUDA-graph replays): 64 ragged requests up to 32768 tokens, 2 x 8
// heads, 596 MB of codes: 101 us, 5.9 TB/s, 0.90 of the measured copy rate
// (95 us with all arithmetic taken out; called from Python on inputs that
// change 115 us, 0.79).  One request of 131072 tokens, 2 x 16
// heads, 67 MB: 23.5 us, of which the stream takes 9, launch and first page
// 4.5, the rows' end 1.2 and the merge 5; the other 3.7 are not placed.  A chunk of 512 tokens with 67 listed
// pages each, 2 x 16 heads, 16 MB cached: 174 us, 207 TFLOP/s, against 71 us
// for the page copies alone and 64 us for the products at mma.sync's rate (8
// cycles per m16n8k16 and SM quarter): two warps per quarter, each a chain of
// ~2300 cycles a page (wait 280, scores 620, softmax 540, values 500, the rest
// bookkeeping), keep the tensor pipe 40 % busy.  Tried and dropped there: three teams
// at 152 registers (noted at 152 us in one form, 224 in another that was measured
// again; one long request 4 to 9 us slower), the next page's scores formed beside
// this page's product with V (168-186 us).
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.h"
#include "page_list.cuh"

namespace ls {
namespace {

constexpr int kPage = LS_PAGE_TOKENS;
constexpr int kTileBytes = kPage * 128;      // one page of one group, K or V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kStages = 2;                   // ring of a warp pair
constexpr int kTeams = 2;                    // teams per CTA, each with a range of its own
constexpr int kWarps = 4;                    // consumer warps of a team: two pairs
constexpr int kPairs = 2;                    // pairs take alternate pages, 32 keys a warp
constexpr int kThreads = 128 * (kTeams + 1);
constexpr int kProducerRegs = 72, kConsumerRegs = 216, kLaunchRegs = 168;
static_assert(kProducerRegs + kTeams * kConsumerRegs <= (kTeams + 1) * kLaunchRegs,
              "the split must fit the registers the block is launched with");
static_assert(kTeams * kPairs == 4, "warpgroup 0 has one producer warp per pair");
constexpr int kMinUnits = 1;                 // pages a range has at least (one request of 4096
                                             // tokens: 9.9 us, 10.7 with 2, 11.2 with 4)
constexpr int kRingBytes = kStages * kStageBytes;
constexpr int kSumBytes = kWarps * 16 * 128 * 4;  // a team's row sums, one set per warp
constexpr float kSlack = 14.f, kHeadroom = 6.f;  // binades, see above
constexpr float kMinScale = 0x1p-40f, kMaxScale = 0x1p48f;

enum StageFlag { kLast = 1, kData = 2, kStop = 4 };  // a row's last stage; a page in it; no more rows

// What a pair's consumers need to know of one stage.
struct __align__(16) PageDesc {
  int key0;        // position of the page's first key
  float k_scale, v_log2, v_inv;
  int limit;       // last position the tile's last token sees
  int token;       // the tile's first token
  int row;         // StageFlag | group << 4 | (workspace part + 1) << 20, part -1: none
  uint32_t tile;   // tokens of the tile << 16 | those of them that list the page
};
constexpr int kDescs = 64;  // a batch of 32 never reaches the stages still in the ring

// The work unit a range begins at: unit `unit` of row (token, group) of
// request `b`, token being the tile's first, counted in the request; with page
// lists of single tokens b is -1 and the token counted in the batch.
struct Start {
  int b, group, token, unit;
};

struct PairSmem {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  PageDesc desc[kDescs];
  int y[kDescs];  // the pages' first rows in the tensor maps (-1: no data)
  // listed: the row's sorted pages; for tiles of several tokens page << 16 |
  // the tokens that list it
  uint32_t pages[kPagedMaxUnion];
};

struct TeamSmem {
  PairSmem pair[kPairs];
  uint64_t join;   // the consumer warps' meeting point, bounded like every wait
  int abort_flag;
  Start start;     // where the team's range begins
  float m_part[2][kWarps][16];  // alternate rows use alternate halves
  float l_part[2][kWarps][16];
};

struct PagedSmem {
  TeamSmem team[kTeams];
  int scan[kThreads / 32];
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm(
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

// mbar_wait for warps that wait often and long: the thread is suspended for up
// to 20 us a try, so that it takes no issue slots from the warps it waits for.
__device__ __forceinline__ bool mbar_sleep(uint64_t* bar, uint32_t parity, int32_t* status,
                                           volatile int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  uint64_t start = 0;
  while (true) {
    uint32_t ok = 0;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, P;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(20000)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    const uint64_t now = globaltimer();
    if (start == 0) start = now;
    if (now - start > LS_WAIT_TIMEOUT_NS) {
      report(status, LS_DEVERR_TIMEOUT);
      *abort_flag = 1;
      return false;
    }
  }
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

// Joining the parts of a row.  A part's reference m is -inf when it has no key
// (its sums are 0), but also when all its scores are NaN, since the maximum
// passes over NaN: its row sum is NaN then, and times the weight 0 it makes the
// whole row's NaN, as it has to.  So l says whether a row has keys: with one it
// is NaN or at least the 2^-42 that the largest score leaves (2^6, over the
// largest value scale), and 0 without.
__device__ __forceinline__ float part_weight(float m, float m_row) {
  return m == -INFINITY ? 0.f : ex2(m - m_row);
}
__device__ __forceinline__ float row_factor(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.f ? INFINITY : (m + log2f(l)) * 0.69314718055994531f;
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

// One page of one group, K then V, into a ring stage.
__device__ __forceinline__ void load_page(const PagedAttnArgs& args, uint8_t* stage, uint64_t* bar,
                                          int y) {
  tma_load_2d(stage, &args.tm_k, bar, 0, y);
  tma_load_2d(stage + kTileBytes, &args.tm_v, bar, 0, y);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Query fragments of one row of heads in f16, scaled by a power of two so that
// the row's largest value is near 1: f16 then holds every value to 2^-25 of
// the largest.  The 32 dims a quad lane holds of a key row (32c ..) are the
// contraction's order: k-step kk takes dims 32c + 4kk .. + 3.  kHalf: at most
// 8 rows of heads, rows 8 .. 15 of the tile stay zero.
template <bool kHalf>
__device__ __forceinline__ void load_query(const PagedAttnArgs& args, int token, int group,
                                           int tokens, int gq, int c, uint32_t (&qa)[8][4],
                                           float* f0, float* f1) {
  const int heads = args.heads_per_group;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int h = gq + 8 * half;
    if (kHalf && half == 1) {
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) qa[kk][1] = qa[kk][3] = 0;
      break;
    }
    // Tile row h is head h % heads of token h / heads.
    const int64_t row =
        static_cast<int64_t>(token + h / heads) * args.num_heads + group * heads + h % heads;
    const uint4* src = reinterpret_cast<const uint4*>(args.q + row * 128 + 32 * c);
    uint4 raw[4];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      raw[k] = h < heads * tokens ? load_input(src + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // The exponent is kept to where the factor stays normal under every page
    // scale, as far as the row's largest value then fits f16 (below 2^15).
    const int top = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    const int e = min(max(top, -60), max(78, top - 14));
    const float down = __int_as_float((127 - e) << 23);
    // Nor does a tiny softmax scale take it to 0, which times the -inf of a masked
    // key would be NaN: products of 2^17 make at most 2^-21 of it.
    const float factor =
        fmaxf(args.scale_log2 * __int_as_float((127 + e) << 23), 0x1p-86f);
    if (half == 0) *f0 = factor; else *f1 = factor;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        qa[2 * k + (j >> 1)][half + 2 * (j & 1)] =
            pack_f16x2(bf16_lo(w[j]) * down, bf16_hi(w[j]) * down);
    }
  }
}

// Whether the first `rows` of a warp's 32 value rows hold a NaN code.
__device__ __forceinline__ bool has_nan(uint32_t v, int rows, int lane) {
  bool found = false;
  for (int r = lane; r < rows; r += 32)
    for (int i = 0; i < 8; ++i) {
      const uint4 x = lds128(v + r * 128 + ((i ^ r) & 7) * 16);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) found = found || __vcmpeq4(w[j] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
    }
  return __any_sync(0xffffffffu, found);
}

// The pages that any of a tile's tokens lists, ascending, as page << 16 | the
// tokens that do; returns how many.  One bit per (page, token) is collected in
// `pages` by page number, then the list is compacted in place.
__device__ __forceinline__ int union_pages(const PagedAttnArgs& args, uint32_t* pages, int token,
                                           int tokens, int g, int n_pages, int limit, int lane) {
  const int most = min(n_pages, kPagedMaxUnion);
  for (int i = lane; i < most; i += 32) pages[i] = 0;
  __syncwarp();
  bool bad = n_pages > kPagedMaxUnion;
  const int32_t* list = args.topk_idx + (static_cast<int64_t>(g) * args.total_q + token) * args.topk;
  for (int t = 0; t < tokens; ++t) {
    const int limit_t = args.causal ? limit - (tokens - 1 - t) : limit;
#pragma unroll
    for (int r = 0; r < LS_MAX_TOPK / 32; ++r) {
      const int pos = 32 * r + lane;
      const int32_t p = pos < args.topk ? load_input(list + t * args.topk + pos) : -1;
      bad = bad || p >= n_pages;
      if (p >= 0 && p < most && p * kPage <= limit_t) atomicOr(pages + p, 1u << t);
    }
  }
  if (bad) report(args.status, LS_DEVERR_PAGE_INDEX);
  __syncwarp();
  int n = 0;
  for (int base = 0; base < most; base += 32) {
    const int i = base + lane;
    const uint32_t m = i < most ? pages[i] : 0;
    const uint32_t some = __ballot_sync(0xffffffffu, m != 0);
    if (m != 0) pages[n + __popc(some & ((1u << lane) - 1))] = static_cast<uint32_t>(i) << 16 | m;
    n += __popc(some);
    __syncwarp();
  }
  return n;
}

// B fragments of 16 keys' values in f16.  A quad lane's four keys (2c, 2c + 1,
// 2c + 8, 2c + 9) are read 16 dims each (16 gq ..); tile j holds dim 16 n + j.
// Keys past the row's limit (`seen` of the warp's 32) may hold anything, NaN
// codes among it, and count as zeros.
__device__ __forceinline__ void load_values(uint32_t stage, uint32_t off0, uint32_t off1, int t,
                                            int c, int seen, uint32_t (&vb)[16][2]) {
  uint32_t w[4][4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint4 v = lds128(stage + ((r & 1) ? off1 : off0) + t * 2048 + (r >> 1) * 1024);
    w[r][0] = v.x;
    w[r][1] = v.y;
    w[r][2] = v.z;
    w[r][3] = v.w;
  }
  if (seen < 32) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * t + 2 * c + (r & 1) + 8 * (r >> 1) >= seen) w[r][0] = w[r][1] = w[r][2] = w[r][3] = 0;
  }
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t lo = __byte_perm(w[2 * half][q4], w[2 * half + 1][q4], 0x5140);
      const uint32_t hi = __byte_perm(w[2 * half][q4], w[2 * half + 1][q4], 0x7362);
      vb[4 * q4][half] = f16x2_lo(lo);
      vb[4 * q4 + 1][half] = f16x2_hi(lo);
      vb[4 * q4 + 2][half] = f16x2_lo(hi);
      vb[4 * q4 + 3][half] = f16x2_hi(hi);
    }
  }
}

__device__ __forceinline__ void mma_values(float (&o)[16][4], const uint32_t (&p)[4],
                                           const uint32_t (&vb)[16][2]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) mma_f16_16816(o[j], p, vb[j][0], vb[j][1]);
}

// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` in a 128B-swizzled box.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) {
  return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}

// Pages a request of `len` cached tokens is scheduled with: at least one, so
// that every row is visited and written.
__device__ __forceinline__ int scheduled_pages(int len) {
  return len > 0 ? (len + kPage - 1) / kPage : 1;
}

// Units of a row of such a request: its pages, or as many as the tile's tokens
// can list between them.  kPagedRowCost is added to every row: its queries,
// the meeting of its warps and its output take about as long as four pages, so
// that a range of many short rows would last longer than one of a long row
// (requests of 15623, 1 and 7622 tokens, 8 heads: 34 us without it).
__device__ __forceinline__ int row_units(const PagedAttnArgs& a, int len) {
  const int pages = scheduled_pages(len);
  return a.topk > 0 ? min(a.pack * a.topk, pages) : pages;
}

// A request as the kernels see it: lengths that would leave the packed rows
// or the block table are cut and reported.
struct Request {
  int q0, nq, len;
  bool bad;
};

__device__ __forceinline__ Request load_request(const PagedAttnArgs& a, int b) {
  Request r;
  r.q0 = load_input(a.cu_q + b);
  const int end = load_input(a.cu_q + b + 1), len = load_input(a.seq_lens + b);
  const int most = a.max_blocks * kPage;  // at most 2^30
  const bool rows_ok = r.q0 >= 0 && end >= r.q0 && end <= a.total_q;
  r.bad = !rows_ok || len < 0 || len > most;
  r.nq = rows_ok ? end - r.q0 : 0;
  r.len = min(max(len, 0), most);
  return r;
}

// Last request whose first row is at or before `row`.
__device__ __forceinline__ int find_request(const PagedAttnArgs& a, int row) {
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (load_input(a.cu_q + mid) <= row) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A range that begins in no row: offsets that count packed rows many times can
// carry the sums past 32 bits (they are reported as they are read).
constexpr int kNoRow = -2;

// `work` units (pages) cut into ranges of at least kMinUnits, as equal as can
// be; paged_schedule.h keeps work below 2^31.
struct Cut {
  int ranges, size, longer;  // `longer` ranges have one unit more
  __device__ __forceinline__ Cut(int work) {
    ranges = min(static_cast<int>(gridDim.x) * kTeams, max(1, (work + kMinUnits - 1) / kMinUnits));
    size = work / ranges;
    longer = work - size * ranges;
  }
  __device__ __forceinline__ int start(int i) const { return i * size + min(i, longer); }
};

template <bool kHalf, bool kShared>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs args) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  PagedSmem* shared =
      reinterpret_cast<PagedSmem*>(smem + kTeams * (kPairs * kRingBytes + kSumBytes));

  allow_next_launch();  // the merge: it waits for this grid's end

  const int warp_id = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = args.num_groups;
  const bool listed = args.topk > 0, single = listed && !kShared;
  const int pack = kShared ? args.pack : 1;  // tokens of a tile

  if (threadIdx.x < kTeams) {
    TeamSmem* t = &shared->team[threadIdx.x];
    for (int p = 0; p < kPairs; ++p)
      for (int s = 0; s < kStages; ++s) {
        mbar_init(&t->pair[p].full[s], 1);
        mbar_init(&t->pair[p].empty[s], kWarps / kPairs);
      }
    mbar_init(&t->join, kWarps);
    t->abort_flag = 0;
    fence_barrier_init();
  }

  wait_for_inputs();

  // ---- the work of all rows, and where the teams' ranges start
  // Page lists of single tokens: row (group, token) has `units` units, ordered
  // group-major.  Otherwise request by request, (group, tile of tokens) rows of
  // row_units units.
  const int range0 = static_cast<int>(blockIdx.x) * kTeams;
  int work, rows_listed = 0;
  if (single) {
    rows_listed = min(max(load_input(args.cu_q + args.batch), 0), static_cast<int>(args.total_q));
    const int units = args.units + kPagedRowCost;
    work = rows_listed * G * units;
    const Cut cut(work);
    if (threadIdx.x < kTeams && range0 + static_cast<int>(threadIdx.x) < cut.ranges && work > 0) {
      const int w0 = cut.start(range0 + threadIdx.x);
      const int row = w0 / units;
      shared->team[threadIdx.x].start = {-1, row / rows_listed, row % rows_listed,
                                         w0 - row * units};
    }
  } else if (args.batch <= 32) {
    // One request per lane, in every warp: no meeting of the block.
    Request r{0, 0, 0, false};
    if (lane < args.batch) r = load_request(args, lane);
    if (r.bad && blockIdx.x == 0 && warp_id == 0) report(args.status, LS_DEVERR_SEQLENS);
    const int tiles = (r.nq + pack - 1) / pack;
    const int units = row_units(args, r.len) + kPagedRowCost, own = tiles * G * units;
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    work = __shfl_sync(0xffffffffu, upto, 31);
    const Cut cut(work);
    if (warp_id < kTeams) {
      const int off = range0 + warp_id < cut.ranges ? cut.start(range0 + warp_id) - (upto - own) : -1;
      const bool here = off >= 0 && off < own;
      if (here) {
        const int row = off / units;
        shared->team[warp_id].start = {lane, row / tiles, row % tiles * pack, off - row * units};
      }
      if (!__any_sync(0xffffffffu, here) && lane == 0) shared->team[warp_id].start.b = kNoRow;
    }
  } else {
    const int per = (args.batch + kThreads - 1) / kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, args.batch);
    const int b1 = min(b0 + per, args.batch);
    int own = 0;
    bool bad = false;
    Request r{0, 0, 0, false};
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      r = load_request(args, b);
      own += (r.nq + pack - 1) / pack * G * (row_units(args, r.len) + kPagedRowCost);
      bad = bad || r.bad;
    }
    if (bad && blockIdx.x == 0) report(args.status, LS_DEVERR_SEQLENS);
    int before = own;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) shared->scan[warp_id] = before;
    if (threadIdx.x < kTeams) shared->team[threadIdx.x].start.b = kNoRow;
    before -= own;
    __syncthreads();
    work = 0;
#pragma unroll 1
    for (int w = 0; w < kThreads / 32; ++w) {
      const int x = shared->scan[w];
      if (w < warp_id) before += x;
      work += x;
    }
    const Cut cut(work);
#pragma unroll 1
    for (int t = 0; t < kTeams; ++t) {
      int off = range0 + t < cut.ranges ? cut.start(range0 + t) - before : -1;
      if (off < 0 || off >= own) continue;
      for (int b = b0; b < b1; ++b) {
        if (b1 - b0 > 1) r = load_request(args, b);
        const int tiles = (r.nq + pack - 1) / pack;
        const int units = row_units(args, r.len) + kPagedRowCost, all = tiles * G * units;
        if (off < all) {
          const int row = off / units;
          shared->team[t].start = {b, row / tiles, row % tiles * pack, off - row * units};
          break;
        }
        off -= all;
      }
    }
  }
  __syncthreads();

  // From here on the warpgroups part for good: the producers give registers
  // up, the consumers take them (each before anything else in its branch).
  const bool producer = warp_id < 4;
  const int team = producer ? warp_id / kPairs : (warp_id >> 2) - 1;
  const int pair = producer ? warp_id % kPairs : (warp_id & 3) / (kWarps / kPairs);
  TeamSmem* sm = &shared->team[team];
  PairSmem* ps = &sm->pair[pair];
  uint8_t* ring = smem + (team * kPairs + pair) * kRingBytes;
  float* sums = reinterpret_cast<float*>(smem + kTeams * kPairs * kRingBytes + team * kSumBytes);
  const Cut cut(work);
  const int range = range0 + team;
  const bool idle = range >= cut.ranges || work == 0 || sm->start.b == kNoRow;
  volatile int* abort_flag = &sm->abort_flag;

  if (producer) {
    // ------------------------------------------------------------- producer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    int2* header = args.headers + range;
    if (idle) {
      if (pair == 0 && lane == 0) *header = make_int2(-1, 1);
      return;
    }
    int left = cut.start(range + 1) - cut.start(range);
    if (lane == 0) {
      tma_prefetch_desc(&args.tm_k);
      tma_prefetch_desc(&args.tm_v);
    }
    int fill = 0, slot = 0;  // stages filled so far, and the ring slot of the next
    uint32_t phase = 1;      // parity that says the slot is free
    bool ok = true;          // lane 0's view; the warp learns of it per batch
    int2 head = make_int2(-1, 1);
    Start at = sm->start;
    Request req{0, 0, 0, false};
    if (!single) req = load_request(args, at.b);
    // A border inside a row's leading units, which stand for its own cost, moves
    // to the row's begin, here and below; `at.unit` counts pages from here on.
    if (at.unit <= kPagedRowCost) {
      left += at.unit;
      at.unit = 0;
    } else {
      at.unit -= kPagedRowCost;
    }
    while (left > 0 && ok) {
      // ---- the row that the next unit belongs to
      int token, tokens = 1;
      if (single) {
        token = at.token;
        if (at.b < 0 || token < req.q0 || token >= req.q0 + req.nq) {
          at.b = find_request(args, token);
          req = load_request(args, at.b);
          if (req.bad && lane == 0) report(args.status, LS_DEVERR_SEQLENS);
        }
      } else {
        token = req.q0 + at.token;
        tokens = min(pack, req.nq - at.token);
      }
      const int units = single ? args.units : row_units(args, req.len);
      const int done = at.unit > 0 ? at.unit + kPagedRowCost : 0;
      if (done + left <= kPagedRowCost) break;  // the row is the next range's
      const int unit_end = min(units, done + left - kPagedRowCost);
      const int t_rel = token - req.q0;
      int limit = req.len - 1;
      if (args.causal) limit = min(limit, req.len - req.nq + t_rel + tokens - 1);
      if (t_rel < 0 || t_rel >= req.nq) limit = -1;
      const int g = at.group;
      // A row cut by the range's borders goes to the workspace: its begin to
      // the range's second part, what continues an earlier range to the first.
      int part = -1;
      if (at.unit > 0) {
        part = 2 * range;
        if (unit_end < units) head.y &= ~1;  // and goes on behind this range too
      } else if (unit_end < units) {
        part = 2 * range + 1;
        head.x = token * G + g;
        head.y |= tokens << 1;
      }

      // ---- its pages, and this pair's share of them: every other one, or
      // one stage without data
      int n_row;
      const int n_pages = (req.len + kPage - 1) / kPage;
      if (single) {
        const int32_t* list =
            args.topk_idx + (static_cast<int64_t>(g) * args.total_q + token) * args.topk;
        int32_t v[4];
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = 32 * r + lane;
          const int32_t p = pos < args.topk ? load_input(list + pos) : -1;
          bad = bad || p >= n_pages;
          v[r] = (p >= 0 && p < n_pages && p * kPage <= limit) ? p : kPageSentinel;
        }
        if (bad) report(args.status, LS_DEVERR_PAGE_INDEX);
        __syncwarp();
        n_row = warp_compact_pages(v, reinterpret_cast<int32_t*>(ps->pages), lane);
        __syncwarp();
      } else if (listed) {
        n_row = union_pages(args, ps->pages, token, tokens, g, n_pages, limit, lane);
      } else {
        n_row = limit >= 0 ? limit / kPage + 1 : 0;
      }
      // (more pages than units: max_seqlen_k was no bound; the last unit takes them)
      const int lo = min(at.unit, n_row) + pair, hi = unit_end < units ? min(unit_end, n_row) : n_row;
      const int count = max(0, (hi - lo + 1) >> 1);
      const int n_stages = max(1, count);

      const int32_t* table = args.block_table + static_cast<int64_t>(at.b) * args.max_blocks;
      for (int base = 0; base < n_stages && ok; base += 32) {
        // 32 pages at once, one per lane: table entry, then both scales.
        PageDesc d;
        int y = -1;
        d.key0 = 0;
        uint32_t mask = (1u << tokens) - 1;
        float ks = 1.f, vs = 1.f;
        if (base + lane < count) {
          const int i = lo + 2 * (base + lane);
          const uint32_t entry = listed ? ps->pages[i] : i;
          const int logical = listed && !single ? entry >> 16 : entry;
          if (listed && !single) mask = entry & 0xFFFF;
          const int page = load_input(table + logical);
          d.key0 = logical * kPage;
          if (page >= 0 && page < args.num_pages) {
            y = (page * G + g) * kPage;
            ks = load_input(args.k_scale + static_cast<int64_t>(page) * G + g);
            vs = load_input(args.v_scale + static_cast<int64_t>(page) * G + g);
          } else {
            report(args.status, LS_DEVERR_PAGE_INDEX);
          }
        }
        const int n = min(32, n_stages - base);
        // The first copies start before the scales are here.
        const int early = min(n, kStages);
        int y0[kStages];
#pragma unroll
        for (int j = 0; j < kStages; ++j) y0[j] = __shfl_sync(0xffffffffu, y, j);
        int s0 = slot;
        uint32_t p0 = phase;
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kStages; ++j) {
            if (j < early && ok) {
              ok = mbar_sleep(&ps->empty[s0], p0, args.status, abort_flag);
              if (ok && y0[j] >= 0) {
                mbar_expect_tx(&ps->full[s0], kStageBytes);
                load_page(args, ring + s0 * kStageBytes, &ps->full[s0], y0[j]);
              }
              if (++s0 == kStages) {
                s0 = 0;
                p0 ^= 1;
              }
            }
          }
        }
        ks = fminf(fmaxf(ks, kMinScale), kMaxScale);
        vs = fminf(fmaxf(vs, kMinScale), kMaxScale);
        d.k_scale = ks;
        d.v_log2 = __log2f(vs);
        d.v_inv = 1.f / vs;
        d.limit = limit;
        d.token = token;
        const int nth = base + lane;
        d.row = (nth + 1 == n_stages ? kLast : 0) | (y >= 0 ? kData : 0) | g << 4 | (part + 1) << 20;
        d.tile = static_cast<uint32_t>(tokens) << 16 | mask;
        if (lane < n) {
          ps->desc[(fill + lane) % kDescs] = d;
          ps->y[(fill + lane) % kDescs] = y;
        }
        __syncwarp();
        if (lane == 0) {
          for (int j = 0; j < n; ++j) {
            if (j < early) {
              // also after a wait that gave up: what is in flight may land
              mbar_arrive(&ps->full[slot]);
            } else {
              ok = ok && mbar_sleep(&ps->empty[slot], phase, args.status, abort_flag);
              if (!ok) break;
              const int y = ps->y[(fill + j) % kDescs];
              if (y >= 0) {
                mbar_arrive_expect_tx(&ps->full[slot], kStageBytes);
                load_page(args, ring + slot * kStageBytes, &ps->full[slot], y);
              } else {
                mbar_arrive(&ps->full[slot]);
              }
            }
            if (++slot == kStages) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        fill += n;
      }
      // ---- on to the next row
      left -= unit_end + kPagedRowCost - done;
      at.unit = 0;
      if (single) {
        if (++at.token == rows_listed) {
          at.token = 0;
          ++at.group;
        }
      } else if ((at.token += pack) >= req.nq) {
        at.token = 0;
        if (++at.group == G) {
          at.group = 0;
          do {
            ++at.b;
            if (at.b >= args.batch) left = 0;  // lengths changed under the kernel
            else req = load_request(args, at.b);
          } while (left > 0 && req.nq == 0);
        }
      }
    }
    if (lane == 0) {
      if (ok) ok = mbar_sleep(&ps->empty[slot], phase, args.status, abort_flag);
      if (ok) {
        ps->desc[fill % kDescs].row = kStop;
        mbar_arrive(&ps->full[slot]);
      } else {
        // Copies in flight must land before the CTA gives up its memory: the
        // last kStages slots filled, newest first.
        for (int k = 0; k < kStages; ++k) {
          if (slot == 0) {
            slot = kStages;
            phase ^= 1;
          }
          --slot;
          mbar_wait(&ps->full[slot], phase ^ 1, nullptr, nullptr);
        }
      }
      if (pair == 0) *header = ok ? head : make_int2(-1, 1);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  if (idle) return;
  const int gq = lane >> 2, c = lane & 3;  // fragment row / key, and quad lane
  const int Hg = args.heads_per_group;
  const int warp = warp_id & 3;
  const int key_base = (warp & 1) * 32;
  // Lane offsets inside a stage.  K: chunk 2c of key gq of a tile (the next
  // chunk is 16 bytes off, before or behind); V: chunk gq of keys 2c, 2c + 1.
  const uint32_t k_off = sw128(gq, 2 * c) + key_base * 128;
  const uint32_t v_off0 = sw128(2 * c, gq) + key_base * 128 + kTileBytes;
  const uint32_t v_off1 = sw128(2 * c + 1, gq) + key_base * 128 + kTileBytes;
  uint32_t qa[8][4];
  float o[16][4];
  float f0 = 0.f, f1 = 0.f;                 // score factors of rows gq and gq + 8
  uint32_t joins = 0;
  // All consumer warps meet; false once a wait has given up anywhere (the
  // row then stays unwritten).
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm->join);
    return mbar_sleep(&sm->join, joins++ & 1, args.status, abort_flag);
  };

  int slot = 0, stage = 0, row_parity = 0;
  uint32_t phase = 0;
  // The first row is known from the start: its queries load while its pages do.
  int token = sm->start.token, group = sm->start.group, tokens = 1;
  if (!single) {
    const Request r = load_request(args, sm->start.b);
    tokens = min(pack, r.nq - token);
    token += r.q0;
  }
  const int tok0 = gq / Hg, tok1 = (gq + 8) / Hg;  // tokens of this lane's tile rows
  while (true) {
    load_query<kHalf>(args, token, group, kShared ? tokens : 1, gq, c, qa, &f0, &f1);
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int flags;
    do {
      if (!mbar_sleep(&ps->full[slot], phase, args.status, abort_flag)) return;
      const PageDesc& desc = ps->desc[stage++ % kDescs];
      flags = desc.row;
      if (flags & kStop) return;  // a range that holds no row

      // Keys of this warp that the last token may see: all 32, some or none.
      const int seen = desc.limit - (desc.key0 + key_base) + 1;
      if ((flags & kData) && seen > 0) {
        const uint32_t st = smem_u32(ring + slot * kStageBytes);
        // ---- S = Q K^T for this warp's 32 keys, four tiles of eight
        float sc[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint4 ka = lds128(st + k_off + n * 1024);
          const uint4 kb = lds128(st + (k_off ^ 16) + n * 1024);
          const uint32_t w[8] = {ka.x, ka.y, ka.z, ka.w, kb.x, kb.y, kb.z, kb.w};
          sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_f16_16816(sc[n], qa[kk], f16x2_lo(w[kk]), f16x2_hi(w[kk]));
        }
        // The values of the first 16 keys are converted while the products run.
        uint32_t vb[16][2];
        load_values(st, v_off0, v_off1, 0, c, seen, vb);
        // ---- keys past a token's limit, and tokens that do not list the page
        // (kShared; the first token sees `back` keys less than the last)
        const int back = kShared && args.causal ? tokens - 1 : 0;
        const uint32_t mask = kShared ? desc.tile & 0xFFFF : 1;
        const bool partial = seen - back < 32 || (kShared && mask != (1u << tokens) - 1);
        if (partial) {
          int seen0 = seen, seen1 = seen;
          if (kShared) {
            seen0 = (mask >> tok0 & 1) ? seen - max(back - tok0, 0) : 0;
            seen1 = (mask >> tok1 & 1) ? seen - max(back - tok1, 0) : 0;
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n * 8 + 2 * c + (e & 1) >= (e < 2 ? seen0 : seen1)) sc[n][e] = -INFINITY;
        }
        // ---- online softmax in the log2 domain
        const float k0 = f0 * desc.k_scale, k1 = f1 * desc.k_scale, v_log2 = desc.v_log2;
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          x0 = fmaxf(x0, fmaxf(sc[n][0], sc[n][1]));
          if (!kHalf) x1 = fmaxf(x1, fmaxf(sc[n][2], sc[n][3]));
        }
        x0 = fmaf(x0, k0, v_log2);
        if (!kHalf) x1 = fmaf(x1, k1, v_log2);
        if (__any_sync(0xffffffffu, x0 - m0 > kSlack || (!kHalf && x1 - m1 > kSlack))) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
          float a0 = 1.f, a1 = 1.f;
          if (x0 - m0 > kSlack) {
            a0 = ex2(m0 - (x0 - kHeadroom));
            m0 = x0 - kHeadroom;
          }
          l0 *= a0;
          if (!kHalf) {
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
            if (x1 - m1 > kSlack) {
              a1 = ex2(m1 - (x1 - kHeadroom));
              m1 = x1 - kHeadroom;
            }
            l1 *= a1;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j][0] *= a0;
            o[j][1] *= a0;
            if (!kHalf) {
              o[j][2] *= a1;
              o[j][3] *= a1;
            }
          }
        }
        // Subtracted after the rounding that the maximum has seen too: scores whose
        // last bit is worth binades (beyond 2^24) still give weights in f16's range.
        const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
        float sum0 = 0.f, sum1 = 0.f;
        uint32_t pa[2][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float p0 = ex2(fmaf(sc[n][0], k0, v_log2) - r0);
          const float p1 = ex2(fmaf(sc[n][1], k0, v_log2) - r0);
          sum0 += p0 + p1;
          pa[n >> 1][2 * (n & 1)] = pack_f16x2(p0, p1);
          if (kHalf) {
            pa[n >> 1][2 * (n & 1) + 1] = 0;
          } else {
            const float p2 = ex2(fmaf(sc[n][2], k1, v_log2) - r1);
            const float p3 = ex2(fmaf(sc[n][3], k1, v_log2) - r1);
            sum1 += p2 + p3;
            pa[n >> 1][2 * (n & 1) + 1] = pack_f16x2(p2, p3);
          }
        }
        l0 = fmaf(sum0, desc.v_inv, l0);
        if (!kHalf) l1 = fmaf(sum1, desc.v_inv, l1);
        // ---- O += P V, the other 16 keys converted behind the first product
        if (kShared && partial && tokens > 1 &&
            has_nan(st + kTileBytes + key_base * 128, min(seen, 32), lane)) {
          // A value that some token does not see is NaN, and 0 * NaN would
          // reach its rows: one token at a time, without the others' keys.
          for (int t = 0; t < tokens; ++t) {
            if (!(mask >> t & 1)) continue;
            const int seen_t = seen - max(back - t, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t p[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) p[i] = ((i & 1) ? tok1 : tok0) == t ? pa[u][i] : 0;
              load_values(st, v_off0, v_off1, u, c, seen_t, vb);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16_16816(d, p, vb[j][0], vb[j][1]);
                if (tok0 == t) {
                  o[j][0] += d[0];
                  o[j][1] += d[1];
                }
                if (tok1 == t) {
                  o[j][2] += d[2];
                  o[j][3] += d[3];
                }
              }
            }
          }
        } else {
          mma_values(o, pa[0], vb);
          load_values(st, v_off0, v_off1, 1, c, seen, vb);
          mma_values(o, pa[1], vb);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ps->empty[slot]);
      if (++slot == kStages) {
        slot = 0;
        phase ^= 1;
      }
    } while (!(flags & kLast));

    // ---- end of this range's share of the row: join the four warps
    const int part = (flags >> 20) - 1;
    float (*m_part)[16] = sm->m_part[row_parity];
    float (*l_part)[16] = sm->l_part[row_parity];
    row_parity ^= 1;
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (c == 0) {
      m_part[warp][gq] = m0;
      m_part[warp][gq + 8] = m1;
      l_part[warp][gq] = l0;
      l_part[warp][gq + 8] = l1;
    }
    if (!meet()) return;
    float mt0 = -INFINITY, mt1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mt0 = fmaxf(mt0, m_part[w][gq]);
      mt1 = fmaxf(mt1, m_part[w][gq + 8]);
    }
    const float s0 = part_weight(m0, mt0), s1 = part_weight(m1, mt1);
    // float4 k of a thread's 32 dims sits at 8c + (k ^ (c, row parity)): the
    // eight lanes of a store or load phase touch eight bank groups.
    const int swz = c | ((gq & 1) << 2);
#pragma unroll
    for (int half = 0; half < (kHalf ? 1 : 2); ++half) {
      float4* dst = reinterpret_cast<float4*>(sums) + (warp * 16 + gq + 8 * half) * 32 + 8 * c;
      const float f = half ? s1 : s0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = 2 * half + (k >> 2), j = 4 * (k & 3);
        dst[k ^ swz] = make_float4(o[j][e] * f, o[j + 1][e] * f, o[j + 2][e] * f, o[j + 3][e] * f);
      }
    }
    if (!meet()) return;
    {
      const int row = (threadIdx.x & 127) >> 3, seg = threadIdx.x & 7;
      float mt = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, m_part[w][row]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        lt = fmaf(l_part[w][row], part_weight(m_part[w][row], mt), lt);
      if (row < (kShared ? Hg * tokens : Hg)) {
        float4 sum[4];
        const int rswz = (seg >> 1) | ((row & 1) << 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4* src = reinterpret_cast<const float4*>(sums) + row * 32 + 8 * (seg >> 1) +
                              ((4 * (seg & 1) + k) ^ rswz);
          sum[k] = src[0];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) {
            const float4 x = src[w * 16 * 32];
            sum[k] = make_float4(sum[k].x + x.x, sum[k].y + x.y, sum[k].z + x.z, sum[k].w + x.w);
          }
        }
        if (part >= 0) {
          const int64_t prow = static_cast<int64_t>(part) * 16 + row;
          float4* dst = reinterpret_cast<float4*>(args.part_o + prow * 128) + 4 * seg;
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = sum[k];
          if (seg == 0)
            *reinterpret_cast<float2*>(args.part_ml + prow * 2) = make_float2(mt, lt);
        } else {
          const int h = group * Hg + (kShared ? row % Hg : row);
          const int t = token + (kShared ? row / Hg : 0);
          const float f = row_factor(lt);
          uint4 packed[2];
          uint32_t* pw = reinterpret_cast<uint32_t*>(packed);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            pw[2 * k] = pack_bf16x2(sum[k].x * f, sum[k].y * f);
            pw[2 * k + 1] = pack_bf16x2(sum[k].z * f, sum[k].w * f);
          }
          uint4* dst = reinterpret_cast<uint4*>(
              args.out + (static_cast<int64_t>(t) * args.num_heads + h) * 128 + 16 * seg);
          dst[0] = packed[0];
          dst[1] = packed[1];
          if (args.lse != nullptr && seg == 0)
            args.lse[static_cast<int64_t>(h) * args.total_q + t] = row_lse(mt, lt);
        }
      }
    }
    // The next row writes the other half of m_part and l_part, and `sums` only
    // after the warps have met again.  Its first stage says which it is.
    if (!mbar_sleep(&ps->full[slot], phase, args.status, abort_flag)) return;
    const PageDesc& next = ps->desc[stage % kDescs];
    if (next.row & kStop) return;
    token = next.token;
    if (kShared) tokens = next.tile >> 16;
    group = (next.row >> 4) & 0xFFFF;
  }
}

size_t paged_smem_bytes() {
  return 1024 + kTeams * (kPairs * kRingBytes + kSumBytes) + sizeof(PagedSmem);
}

// A load that stays where it is written, ahead of the sums that use it.
__device__ __forceinline__ float4 load_part(const float* p) {
  float4 x;
  asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "l"(p));
  return x;
}

// Writes one joined tile row (head `head` % heads of the tile's token `head` /
// heads): lane l holds its dims 4l .. 4l + 3.
__device__ __forceinline__ void write_row(const PagedAttnArgs& args, int row, int head, int lane,
                                          float4 o, float m, float l) {
  const float f = row_factor(l);
  const int heads = args.heads_per_group;
  const int64_t token = row / args.num_groups + head / heads;
  const int h = (row % args.num_groups) * heads + head % heads;
  uint2 packed;
  packed.x = pack_bf16x2(o.x * f, o.y * f);
  packed.y = pack_bf16x2(o.z * f, o.w * f);
  reinterpret_cast<uint2*>(args.out + (token * args.num_heads + h) * 128)[lane] = packed;
  if (args.lse != nullptr && lane == 0)
    args.lse[static_cast<int64_t>(h) * args.total_q + token] = row_lse(m, l);
}

// The rows cut by range borders.  A row that range j begins and does not
// finish has its first part in the range's second workspace part; the ranges
// behind it hold one part each (their first), up to the one whose header says
// that the row ends there.
__device__ __forceinline__ int64_t part_row(int j, int i, int head) {
  return static_cast<int64_t>(i == 0 ? 2 * j + 1 : 2 * (j + i)) * 16 + head;
}

// Far fewer rows than ranges (a decode step of a few long requests): a row has
// many parts.  One block per (row, head); thread k looks after range k, warp w
// sums parts w, w + 24, ...  What a range's parts weigh is loaded with its
// header, before it is known which of them belong to the row: the kernel is a
// chain of round trips, and this one saves a link.
constexpr int kMergeWarps = 24, kMergeAhead = 7;

__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_many_kernel(
    const __grid_constant__ PagedAttnArgs args, int ranges) {
  __shared__ float4 sum[kMergeWarps][32];
  __shared__ float weight[kPagedMaxRanges];
  __shared__ float warp_m[kMergeWarps], warp_l[kMergeWarps];
  __shared__ int first, behind, tokens;
  static_assert(kPagedMaxRanges <= 32 * kMergeWarps, "one thread per range");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x, h = blockIdx.y;
  if (tid == 0) first = behind = ranges;
  __syncthreads();
  allow_next_launch();
  wait_for_inputs();
  const float2* mls = reinterpret_cast<const float2*>(args.part_ml);
  int2 head = make_int2(-1, 1);
  float2 ml = make_float2(-INFINITY, 0.f), begin = ml;
  if (tid < ranges) {
    head = args.headers[tid];
    ml = mls[static_cast<int64_t>(2 * tid) * 16 + h];
    begin = mls[static_cast<int64_t>(2 * tid + 1) * 16 + h];
  }
  if (head.x == row) {
    first = tid;
    tokens = head.y >> 1;
  }
  __syncthreads();
  const int j = first;
  if (j >= ranges || h >= args.heads_per_group * tokens) return;  // the row is whole in one range
  if (tid > j && tid < ranges && (head.y & 1)) atomicMin(&behind, tid);
  __syncthreads();
  const int n = min(behind, ranges - 1) - j + 1;
  if (tid == j) ml = begin;
  if (tid < j || tid >= j + n) ml = make_float2(-INFINITY, 0.f);
  float m = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) warp_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, warp_m[w]);
  const float mine = part_weight(ml.x, m);
  if (tid >= j && tid < j + n) weight[tid - j] = mine;
  float l = ml.y * mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane == 0) warp_l[warp] = l;
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = warp; base < n; base += kMergeAhead * kMergeWarps) {
    float4 x[kMergeAhead];
#pragma unroll
    for (int k = 0; k < kMergeAhead; ++k) {
      const int i = min(base + k * kMergeWarps, n - 1);  // no branch: all loads in flight
      x[k] = load_part(args.part_o + part_row(j, i, h) * 128 + 4 * lane);
    }
#pragma unroll
    for (int k = 0; k < kMergeAhead; ++k) {
      const int i = base + k * kMergeWarps;
      const float w = i < n ? weight[i] : 0.f;
      acc = make_float4(fmaf(x[k].x, w, acc.x), fmaf(x[k].y, w, acc.y), fmaf(x[k].z, w, acc.z),
                        fmaf(x[k].w, w, acc.w));
    }
  }
  sum[warp][lane] = acc;
  __syncthreads();
  if (warp != 0) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) l += warp_l[w];
  float4 t = sum[0][lane];
#pragma unroll
  for (int w = 1; w < kMergeWarps; ++w) {
    const float4 x = sum[w][lane];
    t = make_float4(t.x + x.x, t.y + x.y, t.z + x.z, t.w + x.w);
  }
  write_row(args, row, h, lane, t, m, l);
}

// Otherwise most cut rows have a few parts.  One warp per (range, head); lane
// i looks after part i of 32 at a time.
__global__ void __launch_bounds__(256) paged_merge_few_kernel(
    const __grid_constant__ PagedAttnArgs args, int ranges) {
  const int j = blockIdx.x, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 8 + (threadIdx.x >> 5);
  allow_next_launch();
  wait_for_inputs();
  const int2 head = args.headers[j];
  const int row = head.x;
  if (row < 0 || h >= args.heads_per_group * (head.y >> 1)) return;  // most ranges here
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  bool more = true;
  for (int base = 0; more; base += 32) {
    const int k = j + base + lane;
    int ends_row = 1;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (k < ranges) {
      ends_row = args.headers[k].y & 1;
      ml = reinterpret_cast<const float2*>(args.part_ml)[part_row(j, base + lane, h)];
    }
    const uint32_t ends = __ballot_sync(0xffffffffu, base + lane > 0 && ends_row != 0);
    more = ends == 0;
    const int n = min(more ? 32 : __ffs(ends), ranges - j - base);
    if (lane >= n) ml = make_float2(-INFINITY, 0.f);
    float mx = fmaxf(m, ml.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float keep = part_weight(m, mx), w = part_weight(ml.x, mx);
    m = mx;
    l = fmaf(l, keep, ml.y * w);  // a lane's share; summed at the end
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
    for (int i = 0; i < n; i += 4) {
      float4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        x[u] = load_part(args.part_o + part_row(j, base + min(i + u, n - 1), h) * 128 + 4 * lane);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float wi = __shfl_sync(0xffffffffu, w, (i + u) & 31);
        const float f = i + u < n ? wi : 0.f;
        acc = make_float4(fmaf(x[u].x, f, acc.x), fmaf(x[u].y, f, acc.y), fmaf(x[u].z, f, acc.z),
                          fmaf(x[u].w, f, acc.w));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  write_row(args, row, h, lane, acc, m, l);
}

}  // namespace

// Once per device: the register split of the kernel draws on what the block is
// launched with, so a build that gives it fewer registers must not run; and the
// shared memory limit.
template <bool kHalf, bool kShared>
cudaError_t prepare_attn_kernel() {
  static std::atomic<uint64_t> done[4];
  return once_per_device(done, [] {
    cudaFuncAttributes attr;
    const cudaError_t err = cudaFuncGetAttributes(&attr, paged_attn_kernel<kHalf, kShared>);
    if (err != cudaSuccess) return err;
    if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(paged_attn_kernel<kHalf, kShared>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(paged_smem_bytes()));
  });
}

template <bool kHalf, bool kShared>
cudaError_t launch_attn_kernel(const PagedAttnArgs& args, int ranges, cudaStream_t stream) {
  cudaError_t err = prepare_attn_kernel<kHalf, kShared>();
  if (err != cudaSuccess) return err;
  const int ctas = (ranges + kTeams - 1) / kTeams;
  err = launch_early(paged_attn_kernel<kHalf, kShared>, dim3(ctas), dim3(kThreads), paged_smem_bytes(),
                     stream, args);
  if (err != cudaSuccess) return err;
  const int64_t rows = args.total_q * args.num_groups;
  const int heads = args.heads_per_group * args.pack;  // rows of a tile
  ranges = ctas * kTeams;
  // More than 16 parts a row: by row.  2 rows of 131072 keys 23.4 us (by range
  // 49.8), 8 rows of 65536 34.3 (38.2), 16 rows of 32768 34.1 (34.1), 64 listed
  // rows 34.4 (24.8).  All four are tiles of one token: the rule counts tokens,
  // so tiles of several go by range with up to `pack` times as many parts a row
  // (32 tokens of 2 x 1 heads over 131072 keys take 47 us that way; the other
  // side was not measured).
  if (rows * 16 < ranges)
    return launch_early(paged_merge_many_kernel, dim3(static_cast<unsigned>(rows), heads),
                        dim3(32 * kMergeWarps), 0, stream, args, ranges);
  return launch_early(paged_merge_few_kernel, dim3(ranges, (heads + 7) / 8), dim3(256), 0, stream,
                      args, ranges);
}

cudaError_t launch_paged_attn(const PagedAttnArgs& args, int ranges, cudaStream_t stream) {
  const bool half = args.heads_per_group * args.pack <= 8;
  if (args.pack > 1)
    return half ? launch_attn_kernel<true, true>(args, ranges, stream)
                : launch_attn_kernel<false, true>(args, ranges, stream);
  return half ? launch_attn_kernel<true, false>(args, ranges, stream)
              : launch_attn_kernel<false, false>(args, ranges, stream);
}

}  // namespace ls
