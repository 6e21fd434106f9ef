"""The 8-bit paged cache on the GPU against its 64-bit oracle (needs a B200).

Tolerances:
* planning: whole numbers, equal;
* cache write: codes and scales equal bit for bit (both round the exact
  quotient once, scales are powers of two);
* attention, per output value, with A = sum w|v| and R = max sum |q||k| scale
  of the row from the oracle and N its keys:
    2^-8 (|ref| + e)  rounding of the bf16 output: half a step of the value
  that is rounded, which is ref with an error of up to e, plus
    e = A (2^-11 + 2 d + N 2^-24) + 2^-31 B  with d = 128 2^-23 R + 2^-20 and
  B = max (w vs) sum |code|:
  the weights are rounded to f16 (half a step 2^-11), a score of 128 products
  is off by at most d (each fp32 addition 2^-23 relative when it truncates;
  2^-20 for the exponential and the logarithms of the scales) which moves a
  weight and the row sum by d each, and N fp32 additions of products.
  Weights times value scale are held in f16 relative to a reference that puts
  the largest at 2^6 or more, so a weight in f16's subnormals is off by up to
  2^-25, which is 2^-31 of the largest.
  Queries are held to 2^-25 of their row's largest value: 128 2^-25 is inside d.
* log-sum-exp: d + N 2^-24 for the sum, and 2^-22 (|ref| + 64) for the
  roundings of the reference exponent.
"""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import paged_cache as ora

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU too
    pytest.skip("needs CUDA", allow_module_level=True)

from leanselect_b200 import _native, ops  # noqa: E402

DEV = torch.device("cuda", 0)
PAGE = 64
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def clean_status():
    torch.cuda.synchronize()
    ops.status_word(DEV).zero_()
    yield
    torch.cuda.synchronize()
    assert ops.check_status(DEV) == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prefix(v):
    return [sum(v[:i]) for i in range(len(v) + 1)]


def up(n):
    return -(-n // PAGE)


def tolerance(ref, bounds, n_keys):
    mass, reach, grain = bounds
    d = 128 * 2.0 ** -23 * reach[..., None] + 2.0 ** -20
    e = mass * (2.0 ** -11 + 2 * d + n_keys * 2.0 ** -24) + 2.0 ** -31 * grain
    return 2.0 ** -8 * (ref.abs() + e) + e


# ---------------------------------------------------------------------------
# plan_pages
# ---------------------------------------------------------------------------

def first_table(context, width, pool, gen):
    """A block table for the cached tokens and the free list that is left."""
    perm = torch.randperm(pool, generator=gen).tolist()
    table = []
    for c in context:
        table.append([perm.pop() for _ in range(up(c))] + [-1] * (width - up(c)))
    return table, perm


@pytest.mark.parametrize("context, new, pad", [
    ([0], [1], 0),
    ([63], [1], 0),
    ([64], [1], 0),
    ([0, 5, 64, 127, 128], [0, 0, 0, 0, 0], 3),
    ([0, 1, 63, 64, 65, 200], [1, 64, 1, 0, 63, 129], 0),
    ([130, 0, 7], [3, 0, 300], 11),
    ([0, 0, 640], [1000, 0, 1], 0),
])
def test_plan_small(context, new, pad):
    gen = torch.Generator().manual_seed(1)
    width = max(up(c + n) for c, n in zip(context, new)) + 2
    table, free = first_table(context, width, 100, gen)
    total = sum(new) + pad
    dev_table = i32(table)
    p = ops.plan_pages(i32(context), i32(new), dev_table, i32(free), i32([2]), total)
    ref = ora.plan(context, new, table, free, 2, total)
    check_plan(p, ref, dev_table, table)


def check_plan(p, ref, dev_table, table):
    assert dev_table.tolist() == table
    assert p.seq_lens.tolist() == ref["seq"]
    assert p.cu_seqlens_q.tolist() == ref["cu_q"]
    assert p.cu_blocks.tolist() == ref["cu_blocks"]
    assert p.slots.tolist() == ref["slots"]
    assert p.positions.tolist() == ref["positions"]
    assert p.free_head.tolist() == [ref["head"]]


@pytest.mark.parametrize("batch, longest", [(1, 40000), (37, 3000), (700, 70), (3001, 3)])
def test_plan_large_and_ragged(batch, longest):
    gen = torch.Generator().manual_seed(batch)
    context = torch.randint(0, 300, (batch,), generator=gen).tolist()
    new = torch.randint(0, longest + 1, (batch,), generator=gen).tolist()
    need = sum(up(c) + up(n) + 1 for c, n in zip(context, new))
    width = max(up(c + n) for c, n in zip(context, new))
    table, free = first_table(context, width, need, gen)
    dev_table = i32(table)
    p = ops.plan_pages(i32(context), i32(new), dev_table, i32(free), i32([0]), sum(new))
    check_plan(p, ora.plan(context, new, table, free, 0, sum(new)), dev_table, table)


def test_plan_at_its_largest_batch():
    batch = _native.LS_MAX_PLAN_BATCH
    context, new = [63] * batch, [2] * batch
    table = [[i, -1] for i in range(batch)]
    free = list(range(batch, 2 * batch))
    dev_table = i32(table)
    p = ops.plan_pages(i32(context), i32(new), dev_table, i32(free), i32([0]), 2 * batch)
    check_plan(p, ora.plan(context, new, table, free, 0, 2 * batch), dev_table, table)


def test_plan_out_of_pages_marks_tokens_and_status():
    table = [[-1] * 4, [-1] * 4]
    dev_table = i32(table)
    p = ops.plan_pages(i32([0, 0]), i32([100, 70]), dev_table, i32([5, 6, 7]), i32([0]), 170)
    check_plan(p, ora.plan([0, 0], [100, 70], table, [5, 6, 7], 0, 170), dev_table, table)
    with pytest.raises(_native.LeanSelectError, match="PAGES"):
        ops.check_status(DEV)


@pytest.mark.parametrize("context, new, total", [
    ([-1, 4], [2, 2], 4),      # a negative length counts as 0
    ([0, 4], [-3, 2], 2),
    ([0, 250], [1, 20], 21),   # past max_blocks = 4
    ([0, 0], [5, 5], 7),       # more tokens than the packed rows
])
def test_plan_bad_lengths_are_reported(context, new, total):
    dev_table = i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    p = ops.plan_pages(i32(context), i32(new), dev_table, i32([8, 9]), i32([0]), total)
    slots = p.slots.tolist()
    assert len(slots) == total and all(-1 <= s < 10 * 64 for s in slots)
    if context[1] == 250:
        assert slots[1 + 6:] == [-1] * 14 and slots[1] == 7 * 64 + 58
    with pytest.raises(_native.LeanSelectError, match="SEQLENS"):
        ops.check_status(DEV)


PLAN_THREADS = r"""
#include <atomic>
#include <thread>
#include <vector>
#include "leanselect_b200.h"

// Plans of `calls` steps each from `count` threads that start together; the
// first failing code, or 0.
extern "C" int run(int count, int calls, const int32_t* batch, int32_t* const* ctx,
                   int32_t* const* add, int32_t* const* table, int32_t* const* out,
                   int32_t* const* head, int32_t* status, void* const* stream) {
  std::atomic<int> waiting(count), failed(0);
  std::vector<std::thread> threads;
  for (int i = 0; i < count; ++i)
    threads.emplace_back([&, i] {
      const int b = batch[i];
      for (--waiting; waiting.load() > 0;) {}
      for (int k = 0; k < calls; ++k) {
        const int rc = ls_plan_pages(ctx[i], add[i], b, table[i], 2, nullptr, 0, head[i], 0, out[i],
                                     out[i] + b, out[i] + 2 * b + 1, nullptr, nullptr,
                                     head[i] + 1, status, stream[i]);
        int none = 0;
        if (rc != LS_OK) failed.compare_exchange_strong(none, rc);
      }
    });
  for (auto& t : threads) t.join();
  return failed.load();
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_plans_from_several_threads(tmp_path):
    """Batches whose plans need different amounts of shared memory, planned at once."""
    lib = Path(_native.load()._name)
    src, so = tmp_path / "threads.cpp", tmp_path / "threads.so"
    src.write_text(PLAN_THREADS)
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-pthread", "-I", str(include),
                    str(src), "-o", str(so), str(lib), f"-Wl,-rpath,{lib.parent}"], check=True)
    batches = [5200, 6100, 7000, 8192, 40]
    tensors = [[i32([63] * b), i32([0] * b), i32([[-1, -1]] * b),
                torch.empty(3 * b + 2, dtype=torch.int32, device=DEV), i32([0, -1])]
               for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()

    def pointers(values):
        return (ctypes.c_void_p * len(values))(*values)

    rows = [pointers([t[i].data_ptr() for t in tensors]) for i in range(5)]
    rc = ctypes.CDLL(str(so)).run(
        len(batches), 400, (ctypes.c_int32 * len(batches))(*batches), *rows,
        ctypes.c_void_p(ops.status_word(DEV).data_ptr()),
        pointers([s.cuda_stream for s in streams]))
    torch.cuda.synchronize()
    assert rc == 0, _native.load().ls_status_string(rc)
    for b, t in zip(batches, tensors):
        assert t[4].tolist() == [0, 0] and t[3][:b].tolist() == [63] * b


def test_plan_refusals():
    good = dict(context_lens=i32([0]), new_lens=i32([1]), block_table=i32([[-1]]),
                free_pages=i32([0]), free_head=i32([0]), total_new=1)
    for change in (dict(new_lens=i32([1, 1])), dict(block_table=i32([[-1], [-1]])),
                   dict(block_table=i32([[-1]]).long()), dict(total_new=-1),
                   dict(total_new=1 << 31),
                   dict(free_head=i32([0, 0])),
                   dict(block_table=i32([[-1] * 4])[:, ::2])):
        with pytest.raises(ValueError):
            ops.plan_pages(**{**good, **change})


# ---------------------------------------------------------------------------
# append_kv
# ---------------------------------------------------------------------------

def empty_cache(pages, G, seed):
    """Pages full of leftovers: any code but NaN, any scale."""
    gen = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 127, (pages, G, PAGE, 128), generator=gen, dtype=torch.uint8)
             for _ in range(2)]
    scales = [torch.exp2(torch.randint(-8, 3, (pages, G), generator=gen).float())
              for _ in range(2)]
    return [c.view(FP8).to(DEV) for c in codes] + [s.to(DEV) for s in scales]


def as_values(codes):
    return codes.float().double().cpu()


def run_append(context, new, G, k, v, cache, table):
    width = len(table[0])
    plan = ops.PagePlan(
        i32(context), i32([c + n for c, n in zip(context, new)]), i32(prefix(new)),
        i32(prefix([up(c + n) - c // PAGE if n else 0 for c, n in zip(context, new)])),
        torch.tensor([table[b][p // PAGE] * PAGE + p % PAGE if table[b][p // PAGE] >= 0 else -1
                      for b in range(len(new)) for p in range(context[b], context[b] + new[b])],
                     dtype=torch.int64, device=DEV), None)
    assert width
    want = [as_values(cache[0]), as_values(cache[1]), cache[2].double().cpu(),
            cache[3].double().cpu()]
    ops.append_kv(k, v, plan, cache[0], cache[1], cache[2], cache[3])
    ora.append(k.cpu(), context, new, table, want[0], want[2])
    ora.append(v.cpu(), context, new, table, want[1], want[3])
    for got, ref in zip((as_values(cache[0]), as_values(cache[1]), cache[2].double().cpu(),
                         cache[3].double().cpu()), want):
        assert torch.equal(got.nan_to_num(1234.0), ref.nan_to_num(1234.0))


@pytest.mark.parametrize("context, new, G", [
    ([0], [1], 1),
    ([63], [1], 2),
    ([64], [1], 2),
    ([1], [63], 3),
    ([0, 17, 64, 100], [64, 47, 0, 1], 2),
    ([30, 0, 127, 5], [200, 65, 2, 700], 4),
    ([3], [1], 16),
])
def test_append(context, new, G):
    gen = torch.Generator().manual_seed(7)
    width = max(up(c + n) for c, n in zip(context, new))
    table, _ = first_table([c + n for c, n in zip(context, new)], width, 64, gen)
    cache = empty_cache(64, G, 3)
    n = sum(new)
    # Magnitudes over many binades, so that scales grow, stay and hit old pages.
    size = torch.exp2(torch.randint(-20, 12, (n, G, 1), generator=gen).float())
    k = (torch.randn(n, G, 128, generator=gen) * size).bfloat16().to(DEV)
    v = (torch.randn(n, G, 128, generator=gen)).bfloat16().to(DEV)
    run_append(context, new, G, k, v, cache, table)


@pytest.mark.parametrize("batch, kind", [(33, "one"), (300, "one"), (300, "sparse"),
                                         (1200, "sparse"), (90, "ragged"), (1100, "late")])
def test_append_finds_the_request_of_every_page(batch, kind):
    """Batches beyond one probe of 32 requests: a token each, few requests with
    tokens, requests of many pages, and all tokens in the last requests."""
    gen = torch.Generator().manual_seed(batch)
    context = torch.randint(0, 100, (batch,), generator=gen).tolist()
    if kind == "one":
        new = [1] * batch
    elif kind == "sparse":
        new = [(b % 61 == 7) * (1 + b % 3) for b in range(batch)]
    elif kind == "late":
        new = [0] * (batch - 5) + [70, 0, 3, 200, 1]
    else:
        new = [(b * 37) % 150 for b in range(batch)]
    need = [up(c + n) for c, n in zip(context, new)]
    table, _ = first_table([c + n for c, n in zip(context, new)], max(need), sum(need) + 4, gen)
    k = torch.randn(sum(new), 1, 128, generator=gen).bfloat16().to(DEV)
    run_append(context, new, 1, k, -k, empty_cache(sum(need) + 4, 1, 3), table)


def test_append_offsets_that_are_no_prefix_sums_are_reported():
    """Bad block offsets end the search and write nothing out of range."""
    cache = empty_cache(3, 1, 1)
    k = torch.zeros(100, 1, 128, dtype=torch.bfloat16, device=DEV)
    for cu_blocks in ([5] * 100 + [7], [0] * 50 + [90] * 50 + [8], list(range(100, -1, -1))):
        plan = ops.PagePlan(i32([0] * 100), i32([1] * 100), i32(list(range(101))),
                            i32(cu_blocks), torch.zeros(100, dtype=torch.int64, device=DEV), None)
        ops.append_kv(k, k, plan, *cache)
        torch.cuda.synchronize()
        ops.status_word(DEV).zero_()


@pytest.mark.parametrize("cu_blocks, reported", [
    ([5] * 100 + [7], True),               # blocks before the first request's
    ([0] * 50 + [90] * 50 + [8], True),    # more than the total
    (list(range(100, -1, -1)), False),     # a total of none: nothing to write
])
def test_append_bad_offsets_write_to_no_page_without_a_slot(cu_blocks, reported):
    """All slots are in page 0: whatever the offsets say, pages 1 and 2 are left alone."""
    gen = torch.Generator().manual_seed(3)
    cache = empty_cache(3, 1, 1)
    before = [c.clone() for c in cache]
    k = torch.randn(100, 1, 128, generator=gen).bfloat16().to(DEV)
    plan = ops.PagePlan(i32([0] * 100), i32([1] * 100), i32(list(range(101))), i32(cu_blocks),
                        torch.zeros(100, dtype=torch.int64, device=DEV), None)
    ops.append_kv(k, k, plan, *cache)
    if reported:
        with pytest.raises(_native.LeanSelectError, match="SEQLENS"):
            ops.check_status(DEV)
    for a, b in zip(before, cache):
        first = 0 if cu_blocks[-1] == 0 else 1
        assert torch.equal(a.view(torch.uint8)[first:], b.view(torch.uint8)[first:])


def test_append_extremes():
    """Zeros, subnormals, values at and next to 448 s, infinities and NaN."""
    gen = torch.Generator().manual_seed(5)
    rows = []
    for special in (0.0, 1e-40, 448.0, 450.0, 2.0 ** -60, 3e38, math.inf, math.nan, 896.0):
        r = torch.randn(64, 1, 128, generator=gen) * (1e-3 if special else 0.0)
        if special in (1e-40, 2.0 ** -60):
            r.zero_()
        r[5, 0, 3] = special
        r[9, 0, 4] = -special
        rows.append(r)
    k = torch.cat(rows).bfloat16().to(DEV)
    cache = empty_cache(20, 1, 3)
    table = [list(range(3, 3 + len(rows)))]
    run_append([0], [k.shape[0]], 1, k, k.flip(0), cache, table)


def test_append_grows_a_page_token_by_token():
    """A page written one token at a time rescales what it holds, as the oracle does."""
    gen = torch.Generator().manual_seed(11)
    cache = empty_cache(4, 2, 9)
    size = torch.exp2(torch.arange(70).float() / 6)[:, None, None]
    k = (torch.randn(70, 2, 128, generator=gen) * size).bfloat16().to(DEV)
    v = (torch.randn(70, 2, 128, generator=gen) / size).bfloat16().to(DEV)
    for t in range(70):
        run_append([t], [1], 2, k[t:t + 1], v[t:t + 1], cache, [[2, 0]])


def test_append_views_of_a_fused_projection_and_other_types():
    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(90, 8 * 128, generator=gen).bfloat16().to(DEV)
    k, v = qkv[:, 4 * 128:6 * 128].view(90, 2, 128), qkv[:, 6 * 128:].view(90, 2, 128)
    assert not k.is_contiguous()
    table = [[1, 3]]
    run_append([20], [90], 2, k, v, empty_cache(5, 2, 1), table)
    # Heads that are not contiguous, and fp32 values: rounded to bf16 on the way in.
    odd = torch.randn(90, 128, 2, generator=gen).to(DEV).transpose(1, 2)
    cache, twin = empty_cache(5, 2, 1), empty_cache(5, 2, 1)
    for c, x in ((cache, odd), (twin, odd.bfloat16().contiguous())):
        plan = ops.plan_pages(i32([0]), i32([90]), i32([[-1, -1]]), i32([4, 2]), i32([0]), 90)
        ops.append_kv(x, x, plan, *c)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, twin))


def test_append_one_token_with_heads_first_and_unaligned_rows():
    gen = torch.Generator().manual_seed(4)
    k = torch.randn(3, 1, 128, generator=gen).bfloat16().to(DEV).transpose(0, 1)
    run_append([70], [1], 3, k, k, empty_cache(4, 3, 1), [[2, 0]])
    flat = torch.randn(20 * 3 * 128 + 1, generator=gen).bfloat16().to(DEV)
    k = flat[1:].view(20, 3, 128)
    run_append([60], [20], 3, k, -k, empty_cache(4, 3, 1), [[2, 0]])


def test_append_skips_tokens_without_pages_and_bad_pages():
    gen = torch.Generator().manual_seed(2)
    k = torch.randn(130, 1, 128, generator=gen).bfloat16().to(DEV)
    run_append([0], [130], 1, k, k, empty_cache(6, 1, 1), [[4, -1, 2]])
    cache = empty_cache(6, 1, 1)
    before = [c.clone() for c in cache]
    slots = torch.arange(6 * 64, 6 * 64 + 64, dtype=torch.int64, device=DEV)  # page 6 of 6
    plan = ops.PagePlan(i32([0]), i32([64]), i32([0, 64]), i32([0, 1]), slots, None)
    ops.append_kv(k[:64], k[:64], plan, *cache)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
               for a, b in zip(cache, before))
    with pytest.raises(_native.LeanSelectError, match="PAGE_INDEX"):
        ops.check_status(DEV)


def test_append_refusals():
    cache = empty_cache(3, 2, 1)
    plan = ops.plan_pages(i32([0]), i32([5]), i32([[-1]]), i32([0]), i32([0]), 5)
    k = torch.zeros(5, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.append_kv(k, k, plan, *cache)
    for args in ((k[:, :1], k[:, :1], plan, *cache), (k, k[:4], plan, *cache),
                 (k[:4], k[:4], plan, *cache),
                 (k, k, plan, cache[0].view(torch.uint8), *cache[1:]),
                 (k, k, plan, cache[0], cache[1][:2], *cache[2:]),
                 (k, k, plan, *cache[:2], cache[2].double(), cache[3])):
        with pytest.raises(ValueError):
            ops.append_kv(*args)


# ---------------------------------------------------------------------------
# paged_attn
# ---------------------------------------------------------------------------

def make_cache(seq, G, seed, sizes=(1.0, 1.0), nan_tail=True):
    """Quantised random K/V of the requests in scattered pages; rows behind a
    request's last token hold NaN codes."""
    gen = torch.Generator().manual_seed(seed)
    need = [up(max(n, 0)) for n in seq]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=gen).tolist()
    width = max(max(need), 1)
    table = []
    pools = []
    for size in sizes:
        x = torch.randn(pool, G, PAGE, 128, generator=gen, dtype=torch.float64) * size
        x = x * torch.exp2(torch.randint(-3, 4, (pool, G, 1, 1), generator=gen).double())
        amax = x.abs().amax((2, 3))
        s = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
        pools.append((ora.e4m3(x / s[:, :, None, None]), s.float()))
    for n in need:
        table.append([perm.pop() for _ in range(n)] + [-1] * (width - n))
    codes = [c.float().to(FP8) for c, _ in pools]
    if nan_tail:
        for c in codes:
            raw = c.view(torch.uint8)
            for b, n in enumerate(seq):
                if n > 0 and n % PAGE:
                    raw[table[b][n // PAGE], :, n % PAGE:] = 0x7F
            raw[perm] = 0x7F
    return codes, [s for _, s in pools], table


def run_attend(H, G, seq, nq, *, idx=None, causal=True, scale=None, seed=0, pad=0, sizes=(1.0, 1.0),
               qsize=1.5, q_dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed + 100)
    codes, scales, table = make_cache(seq, G, seed, sizes)
    N = sum(nq) + pad
    q = (torch.randn(N, H, 128, generator=gen) * qsize).to(q_dtype)
    cu = prefix(nq)
    out = torch.full((N, H, 128), 3.0, dtype=q_dtype, device=DEV)
    got, lse = ops.paged_attn(
        q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV),
        i32(table), i32(seq), i32(cu), max(nq), max(max(seq), 0), causal=causal,
        topk_idx=None if idx is None else idx.to(DEV), softmax_scale=scale, return_lse=True,
        out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, ref_lse, bounds = ora.attend(
        q.bfloat16(), codes[0].float(), codes[1].float(), scales[0], scales[1], table,
        [max(n, 0) for n in seq], cu, idx, scale, causal, torch.full((N, H, 128), 3.0))
    n_keys = max(max(seq), 1)
    d = 128 * 2.0 ** -23 * bounds[1] + 2.0 ** -20
    tol = tolerance(ref, bounds, n_keys)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())
    live = cu[-1]
    a, r = lse.double().cpu()[:, :live], ref_lse[:, :live]
    assert torch.equal(torch.isinf(a), torch.isinf(r))
    fin = torch.isfinite(r)
    ltol = d.T[:, :live] + n_keys * 2.0 ** -24 + 2.0 ** -22 * (r.abs() + 64)
    assert bool(((a - r).abs()[fin] <= ltol[fin]).all()), float(((a - r).abs() - ltol)[fin].max())
    return got


@pytest.mark.parametrize("H, G", [(32, 2), (16, 2), (16, 1), (4, 4), (5, 1), (12, 6), (16, 16)])
@pytest.mark.parametrize("length", [1, 16, 63, 64, 65, 1000])
def test_decode_lengths_and_heads(H, G, length):
    run_attend(H, G, [length], [1], seed=length)


@pytest.mark.parametrize("causal", [True, False])
def test_dense_ragged_batch(causal):
    run_attend(32, 2, [1, 500, 64, 129, 2048, 77, 300], [1, 4, 0, 3, 1, 2, 70], causal=causal)


def test_rows_without_keys_are_zero():
    """Empty requests, and rows that stand before position 0."""
    run_attend(16, 2, [0, 5, 0, 3], [1, 1, 2, 6])


@pytest.mark.parametrize("H, G", [(8, 8), (32, 2)])
def test_short_rows_between_long_ones(H, G):
    """Ranges that begin in a row's leading units, hold many short rows or none."""
    run_attend(H, G, [9000, 1, 1, 5000, 0, 2, 64, 1, 1], [1, 1, 2, 1, 1, 1, 0, 1, 1], seed=3)
    run_attend(H, G, [1] * 700, [1] * 700, seed=4)


@pytest.mark.parametrize("batch", [33, 500])
@pytest.mark.parametrize("listed", [False, True])
def test_drafts_of_many_requests(batch, listed):
    """Batches that the whole block adds up, several tokens each, some none."""
    gen = torch.Generator().manual_seed(batch)
    seq = torch.randint(0, 200, (batch,), generator=gen).tolist()
    nq = torch.randint(0, 4, (batch,), generator=gen).tolist()
    idx = page_lists(seq, nq, 2, 3, 3, "future") if listed else None
    run_attend(8, 2, seq, nq, idx=idx, seed=batch)


def test_no_rows_and_no_tokens():
    codes, scales, table = make_cache([64], 2, 3)
    cache = [codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV)]
    q = torch.empty(0, 32, 128, dtype=torch.bfloat16, device=DEV)
    out, lse = ops.paged_attn(q, *cache, i32(table), i32([64]), i32([0, 0]), 0, 64, return_lse=True)
    assert out.shape == (0, 32, 128) and lse.shape == (32, 0)
    plan = ops.plan_pages(i32([64]), i32([0]), i32([[0, -1]]), i32([1]), i32([0]), 0)
    ops.append_kv(q[:, :2], q[:, :2], plan, *cache)
    assert plan.slots.numel() == 0 and plan.seq_lens.tolist() == [64]


def test_rows_behind_the_last_request_are_left():
    run_attend(16, 2, [200, 90], [2, 1], pad=5)


@pytest.mark.parametrize("batch, length", [(1, 20000), (3, 7001), (150, 130), (400, 40)])
def test_many_splits_and_many_rows(batch, length):
    """One row cut into a part per CTA; several rows per CTA."""
    gen = torch.Generator().manual_seed(batch)
    seq = torch.randint(1, length + 1, (batch,), generator=gen).tolist()
    seq[0] = length
    run_attend(16, 1, seq, [1] * batch, seed=batch)


@pytest.mark.parametrize("sizes, qsize", [((8.0, 1e-3), 1.5), ((0.01, 100.0), 4.0),
                                          ((1.0, 2.0 ** -28), 1.5), ((1.0, 2.0 ** 44), 1.5),
                                          ((2.0 ** -28, 1.0), 2.0 ** 28)])
def test_scales_and_peaked_rows(sizes, qsize):
    run_attend(32, 2, [700, 100], [2, 1], sizes=sizes, qsize=qsize, seed=4)


@pytest.mark.parametrize("power", [40, 47, 50, 60, 78])
@pytest.mark.parametrize("n", [1, 4])
def test_scores_of_any_size(power, n):
    """Scores far beyond 2^24, whose last bit is worth binades: queries along one key each,
    so that the row is that key's value (every other key scores a quarter less)."""
    H, length = 4, 300
    codes, scales, table = make_cache([length], 1, 9)
    gen = torch.Generator().manual_seed(power)
    signs = torch.randint(0, 2, (up(length), PAGE, 128), generator=gen).double() * 2 - 1
    for j, page in enumerate(table[0]):
        codes[0][page, 0] = signs[j].float().to(FP8)
        scales[0][page] = 2.0 ** -20
    at = [17, 64, 130, 255][:n]
    flat = signs.reshape(-1, 128)
    # products with the other keys are at most 128 - 2 * 16
    assert all(int((flat[:length] @ flat[a]).topk(2).values[1]) <= 96 for a in at)
    q = torch.stack([flat[a] for a in at])[:, None].expand(n, H, 128) * 2.0 ** power
    got, lse = ops.paged_attn(
        q.bfloat16().contiguous().to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV),
        scales[1].to(DEV), i32(table), i32([length]), i32([0, n]), n, length, return_lse=True)
    for i, a in enumerate(at):
        page, row = table[0][a // PAGE], a % PAGE
        want = codes[1][page, 0, row].double() * float(scales[1][page, 0])
        assert torch.equal(got[i].double().cpu(), want.expand(H, 128))
        score = 128 * 2.0 ** (power - 20) / math.sqrt(128)
        assert bool(((lse[:, i].double().cpu() - score).abs() <= 2.0 ** -20 * score).all())


@pytest.mark.parametrize("power", [93, 94, 110, 127])
def test_queries_up_to_the_largest(power):
    """bf16 queries beyond f16's range under their scaling: along one key each, as above."""
    test_scores_of_any_size(power, 4)


@pytest.mark.parametrize("scale, qsize", [(1e-30, 0.0), (1e-20, 0.0), (1e-38, 1.5), (1e-42, 1.5),
                                          (0.1, 0.0), (0.1, 1e-30)])
def test_scores_next_to_zero(scale, qsize):
    """Softmax scales and queries so small that their product with a key's scale
    underflows: the weights are equal, masked keys stay out."""
    run_attend(16, 2, [200, 70, 1], [1, 3, 1], scale=scale, qsize=qsize)
    run_attend(16, 1, [9000], [1], scale=scale, qsize=qsize)


def test_pages_of_very_different_value_scales():
    """A row whose weight sits in a page of tiny values next to pages of large ones."""
    gen = torch.Generator().manual_seed(6)
    codes, scales, table = make_cache([256], 1, 6)
    scales[1][table[0][0]] = 2.0 ** -30
    scales[1][table[0][1]] = 2.0 ** 10
    q = torch.randn(1, 16, 128, generator=gen).bfloat16()
    # the first page's first key points along the query
    codes[0][table[0][0], 0, 0] = (q[0, 0].float() * 100).clamp(-448, 448).to(FP8)
    scales[0][table[0][0]] = 0.25
    ref, _, bounds = ora.attend(q, codes[0].float(), codes[1].float(), scales[0], scales[1],
                                     table, [256], [0, 1])
    got = ops.paged_attn(q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV),
                         scales[1].to(DEV), i32(table), i32([256]), i32([0, 1]), 1, 256)
    tol = tolerance(ref, bounds, 256)
    assert bool(((got.double().cpu() - ref).abs() <= tol).all())


def page_lists(seq, nq, G, T, seed, kind):
    gen = torch.Generator().manual_seed(seed)
    rows = []
    for b, n in enumerate(nq):
        for i in range(n):
            last = max(0, (seq[b] - n + i) // PAGE)
            per = []
            for _ in range(G):
                if kind == "empty" and (i + b) % 2 == 0:
                    per.append([-1] * T)
                    continue
                pick = torch.randperm(last + 1, generator=gen)[:T].tolist()
                if kind == "ascending":
                    pick = sorted(pick)
                elif kind == "repeats":
                    pick = (pick + pick[:3] + [-1, 0, 0])[:T]
                elif kind == "future":     # pages past the row's position, within the request
                    pick = torch.randperm(up(max(seq[b], 1)), generator=gen)[:T].tolist()
                per.append(pick + [-1] * (T - len(pick)))
            rows.append(per)
    return torch.tensor(rows, dtype=torch.int32).transpose(0, 1).contiguous()


@pytest.mark.parametrize("kind", ["ascending", "shuffled", "repeats", "future", "empty"])
@pytest.mark.parametrize("H, G, T", [(32, 2, 67), (16, 2, 128), (6, 2, 5), (16, 1, 1)])
def test_listed_pages(kind, H, G, T):
    seq, nq = [3000, 64, 1, 900], [1, 2, 1, 17]
    run_attend(H, G, seq, nq, idx=page_lists(seq, nq, G, T, 5, kind), seed=T)


def test_listed_chunk_many_rows():
    seq, nq = [2000], [333]
    run_attend(16, 2, seq, nq, idx=page_lists(seq, nq, 2, 12, 5, "ascending"), seed=2)


def test_listed_rows_with_padding_and_no_causal_limit():
    seq, nq = [700, 300], [3, 2]
    idx = page_lists(seq, nq, 2, 7, 5, "future")
    idx = torch.nn.functional.pad(idx, (0, 0, 0, 4), value=0)
    run_attend(32, 2, seq, nq, idx=idx, pad=4, causal=False)


@pytest.mark.parametrize("H, G", [(4, 1), (16, 2), (6, 2), (3, 1), (16, 16), (32, 2), (9, 1)])
@pytest.mark.parametrize("listed", [False, True])
def test_tokens_of_a_request_share_tiles(H, G, listed):
    """Drafts and chunks: tiles of several tokens, the last of them partly filled,
    rows before position 0, requests of no and of few tokens."""
    seq, nq = [300, 0, 64, 7, 1500], [5, 0, 17, 9, 33]
    idx = None
    if listed:
        idx = page_lists(seq, nq, G, 9, 3, "repeats")
        idx[:, 3] = -1
    for causal in (True, False):
        run_attend(H, G, seq, nq, idx=idx, causal=causal, seed=H)


@pytest.mark.parametrize("kind", ["ascending", "shuffled", "repeats", "future", "empty"])
@pytest.mark.parametrize("H, G", [(4, 1), (10, 2), (6, 2), (3, 1)])
def test_lists_that_overlap_are_joined(kind, H, G):
    """Lists three times as long as the requests' pages, for many rows: one tile holds
    several tokens and walks the union of their pages."""
    seq, nq = [1500, 64, 0, 700, 7], [40, 17, 0, 33, 9]
    idx = page_lists(seq, nq, G, 128, 4, kind)
    idx = torch.nn.functional.pad(idx, (0, 0, 0, 300), value=0)   # rows behind the last request
    for causal in (True, False):
        run_attend(H, G, seq, nq, idx=idx, causal=causal, seed=G, pad=300)


@pytest.mark.parametrize("kind", ["ascending", "shuffled", "future"])
def test_joined_lists_of_512_pages(kind):
    """The longest request that lists are joined for, whose union fills the shared table;
    ranges of more pages than one batch of a producer warp."""
    seq, nq = [512 * PAGE], [400]
    run_attend(2, 2, seq, nq, idx=page_lists(seq, nq, 2, 128, 6, kind), seed=6)


@pytest.mark.parametrize("H, G, T, longest, most", [
    (1, 1, 128, 21800, 8),    # tiles of 8 rows, 341 pages
    (6, 2, 60, 6400, 9),      # tiles of 15 rows
    (8, 2, 128, 10800, 7),    # four tokens of 4 heads
])
@pytest.mark.parametrize("batch", [20, 45])
def test_joined_lists_of_many_requests(H, G, T, longest, most, batch):
    """Requests of no, one and several tokens, found by warp and by the whole block."""
    gen = torch.Generator().manual_seed(batch)
    seq = [1 + int(longest * x ** 4) for x in torch.rand(batch, generator=gen).tolist()]
    nq = torch.randint(0, most + 1, (batch,), generator=gen).tolist()
    seq[3], nq[3], nq[4], nq[5], nq[6] = longest, most, 0, 1, most
    idx = page_lists(seq, nq, G, T, 2, "repeats")
    # rows behind the last request, for the work that joining is worth
    pad = 9000 // (G * T)
    idx = torch.nn.functional.pad(idx, (0, 0, 0, pad), value=0)
    run_attend(H, G, seq, nq, idx=idx, seed=batch, pad=pad)


def test_joined_lists_past_their_512_pages_are_passed_over_and_reported():
    """max_seqlen_k that is no bound: pages from the 512th on are not attended to."""
    H, length, n = 2, 515 * PAGE, 80
    codes, scales, table = make_cache([length], H, 2)
    gen = torch.Generator().manual_seed(2)
    q = torch.randn(n, H, 128, generator=gen).bfloat16()
    idx = page_lists([length], [n], H, 128, 2, "shuffled")
    idx[:, :, 5] = 512 + torch.arange(n, dtype=torch.int32) % 3
    got = ops.paged_attn(q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV),
                         scales[1].to(DEV), i32(table), i32([length]), i32([0, n]), n, 512 * PAGE,
                         topk_idx=idx.to(DEV))
    want, _, bounds = ora.attend(q, codes[0].float(), codes[1].float(), scales[0], scales[1], table,
                                 [length], [0, n], torch.where(idx < 512, idx, -1))
    assert bool(((got.double().cpu() - want).abs() <= tolerance(want, bounds, length)).all())
    with pytest.raises(_native.LeanSelectError, match="PAGE_INDEX"):
        ops.check_status(DEV)


def test_long_requests_keep_single_lists():
    """Lists of requests beyond the shared table (512 pages), several tokens each."""
    seq, nq = [33000, 200], [3, 4]
    run_attend(8, 2, seq, nq, idx=page_lists(seq, nq, 2, 40, 3, "ascending"), seed=1)


@pytest.mark.parametrize("listed", [False, True])
def test_nan_stays_with_the_rows_that_see_it(listed):
    """A NaN value reaches the tokens that attend to it and no others of their tile."""
    H, G, length, n = 4, 1, 200, 4
    codes, scales, table = make_cache([length], G, 5, nan_tail=False)
    raw = [c.view(torch.uint8) for c in codes]
    last = table[0][length // PAGE]
    raw[1][last, 0, (length - 2) % PAGE, 7] = 0x7F   # seen by the last two tokens
    raw[0][last, 0, (length - 1) % PAGE, 9] = 0xFF   # a key that the last token sees
    idx = None
    if listed:
        raw[1][table[0][1], 0, 5, 3] = 0xFF          # in a page that tokens 1 and 3 list
        idx = torch.tensor([[[0, 3, -1], [0, 1, 3], [0, 2, 3], [1, 3, -1]]], dtype=torch.int32)
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(n, H, 128, generator=gen).bfloat16()
    got = ops.paged_attn(q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV),
                         scales[1].to(DEV), i32(table), i32([length]), i32([0, n]), n, length,
                         topk_idx=None if idx is None else idx.to(DEV)).double().cpu()
    want, _, bounds = ora.attend(q, codes[0].float(), codes[1].float(), scales[0], scales[1], table,
                                 [length], [0, n], idx)
    # NaN in the sum of a dim at any weight, as 0 * NaN; whole rows for the NaN key
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(want.isnan()[n - 1].all()) and not bool(want.isnan()[0].any())
    ok = ~want.isnan()
    err = (got - want).abs()
    assert bool((err[ok] <= tolerance(want, bounds, length)[ok]).all())


def test_nan_and_bad_pages_in_joined_lists():
    """As above for lists that are joined: four tokens with one key set each, and a bad page."""
    H, G, length, n = 4, 1, 200, 4
    codes, scales, table = make_cache([length], G, 5, nan_tail=False)
    raw = [c.view(torch.uint8) for c in codes]
    raw[1][table[0][3], 0, 198 % PAGE, 7] = 0x7F      # seen by the last two tokens
    raw[0][table[0][3], 0, 199 % PAGE, 9] = 0xFF      # a key that the last token sees
    raw[1][table[0][1], 0, 5, 3] = 0xFF               # in a page that tokens 1 and 3 list
    idx = torch.full((1, 1200, 128), -1, dtype=torch.int32)
    for i, pages in enumerate([[0, 3], [0, 1, 3], [0, 2, 3], [3, 1]]):
        idx[0, i, 5:5 + len(pages)] = torch.tensor(pages, dtype=torch.int32)
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(1200, H, 128, generator=gen).bfloat16()

    def both():
        out = torch.full_like(q, 2.0, device=DEV)
        ops.paged_attn(q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV),
                       scales[1].to(DEV), i32(table), i32([length]), i32([0, n]), n, length,
                       topk_idx=idx.to(DEV), out=out)
        assert bool((out[n:] == 2.0).all())
        want, _, bounds = ora.attend(q[:n], codes[0].float(), codes[1].float(), scales[0],
                                     scales[1], table, [length], [0, n], idx[:, :n])
        got = out[:n].double().cpu()
        assert torch.equal(got.isnan(), want.isnan())
        ok = ~want.isnan()
        assert bool(((got - want).abs()[ok] <= tolerance(want, bounds, length)[ok]).all())
        return want

    want = both()
    assert bool(want.isnan()[3].all()) and bool(want.isnan()[1, :, 3].all())
    assert not bool(want.isnan()[0].any())
    table[0][2] = 10 ** 6
    idx[0, 2, 0] = 9                                  # past the request's pages
    both()
    with pytest.raises(_native.LeanSelectError, match="PAGE_INDEX"):
        ops.check_status(DEV)


def nan_case(H, G, seq, nq, *, idx=None, nan_keys=(), nan_rows=(), seed=5):
    """Output, lse and the oracle's for a cache with NaN keys ``(request, first, last + 1)``
    and NaN query rows; where they are NaN and where a row has no key must agree."""
    codes, scales, table = make_cache(seq, G, seed)
    raw = codes[0].view(torch.uint8)
    for b, first, end in nan_keys:
        for p in range(first, end):
            raw[table[b][p // PAGE], :, p % PAGE] = 0x7F
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(nq), H, 128, generator=gen).bfloat16()
    for t in nan_rows:
        q[t, 0] = math.nan
    got, lse = ops.paged_attn(
        q.to(DEV), codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV),
        i32(table), i32(seq), i32(prefix(nq)), max(nq), max(seq),
        topk_idx=None if idx is None else idx.to(DEV), return_lse=True)
    want, want_lse, bounds = ora.attend(q, codes[0].float(), codes[1].float(), scales[0], scales[1],
                                        table, seq, prefix(nq), idx)
    got, lse = got.double().cpu(), lse.double().cpu()
    assert bool(want_lse.isnan().any())
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(lse.isnan(), want_lse.isnan())
    assert torch.equal(lse.isinf(), want_lse.isinf())
    ok, fine = ~want.isnan(), torch.isfinite(want_lse)
    assert bool(((got - want).abs()[ok] <= tolerance(want, bounds, max(seq))[ok]).all())
    d = 128 * 2.0 ** -23 * bounds[1].T + 2.0 ** -20
    ltol = d + max(seq) * 2.0 ** -24 + 2.0 ** -22 * (want_lse.abs() + 64)
    assert bool(((lse - want_lse).abs()[fine] <= ltol[fine]).all())


@pytest.mark.parametrize("H, G, seq, nq", [
    (16, 1, [1, 70, 0], [1, 1, 1]),          # rows inside one range
    (8, 2, [5000], [1]),                     # one row in many parts: joined by row
    (8, 1, [3000] * 24, [1] * 24),           # rows of a few parts: joined by range
    (4, 1, [300, 5], [5, 2]),                # several tokens a tile
    (4, 1, [2600] * 8, [4] * 8),             # and tiles cut by range borders
])
def test_lse_of_nan_scores_is_nan(H, G, seq, nq):
    """Every key of a warp's share, of a page, of a row, or the query itself is NaN: the
    row's lse is NaN, never finite and never the +inf of a row without keys."""
    last = seq[0]
    for first, end in ((0, 1), (0, min(last, 32)), (0, min(last, 64)), (last - 1, last), (0, last)):
        nan_case(H, G, seq, nq, nan_keys=[(0, first, end)])
    nan_case(H, G, seq, nq, nan_rows=[0])


@pytest.mark.parametrize("H, n", [(16, 3), (4, 3), (4, 1200)])
def test_lse_of_nan_scores_in_listed_pages(H, n):
    """As above where rows list their pages: alone, and (1200 rows of 4 heads) joined."""
    T = 128 if n > 3 else 3
    idx = torch.full((1, n, T), -1, dtype=torch.int32)
    for i in range(n):
        pages = ([0], [1, 2], [0, 2], [])[i % 4]
        idx[0, i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    seq = [max(190, n)]
    nan_case(H, 1, seq, [n], idx=idx, nan_keys=[(0, 0, 64)])
    nan_case(H, 1, seq, [n], idx=idx, nan_rows=[1, n - 2])


def test_bad_pages_are_passed_over_and_reported():
    codes, scales, table = make_cache([300, 64], 2, 3)
    table[0][1] = 10 ** 6
    table[0][3] = -1
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(2, 32, 128, generator=gen).bfloat16()
    args = (codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV), i32(table),
            i32([300, 64]), i32([0, 1, 2]), 1, 300)
    for idx in (None, torch.tensor([[[3, 1, 0, 4], [0, 9, -1, -1]]] * 2, dtype=torch.int32)):
        got = ops.paged_attn(q.to(DEV), *args, topk_idx=None if idx is None else idx.to(DEV))
        ref, _, bounds = ora.attend(q, codes[0].float(), codes[1].float(), scales[0], scales[1],
                                     table, [300, 64], [0, 1, 2], idx)
        assert bool(((got.double().cpu() - ref).abs() <= tolerance(ref, bounds, 300)).all())
        with pytest.raises(_native.LeanSelectError, match="PAGE_INDEX"):
            ops.check_status(DEV)


def test_bad_lengths_are_reported_and_stay_in_bounds():
    codes, scales, table = make_cache([100, 64], 1, 3)
    cache = (codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV), i32(table))
    q = torch.randn(3, 16, 128, device=DEV).bfloat16()
    for seq, cu in (([100, 100000], [0, 1, 2]), ([-5, 64], [0, 1, 2]), ([100, 64], [0, 2, 9]),
                    ([100, 64], [0, 3, 1])):
        ops.paged_attn(q, *cache, i32(seq), i32(cu), 1, 128)
        with pytest.raises(_native.LeanSelectError):
            ops.check_status(DEV)


def test_offsets_that_count_rows_many_times_are_reported():
    """Offsets that go back and forth over the packed rows, so that the scheduled pages
    pass 32 bits; every single request is within the limits."""
    N, G, blocks = 8193, 8, 16380
    codes, scales, _ = make_cache([64], G, 1)
    cu = []
    for _ in range(4 * 289 // 2):
        cu += [0, N - 1]
    batch = len(cu)
    cu.append(0)
    q = torch.zeros(N, G, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.full((batch, blocks), -1, dtype=torch.int32, device=DEV)
    ops.paged_attn(q, codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV),
                   table, i32([blocks * PAGE] * batch), i32(cu), 1, blocks * PAGE)
    with pytest.raises(_native.LeanSelectError, match="SEQLENS"):
        ops.check_status(DEV)
    run_attend(8, 2, [70], [1])


def test_lists_of_very_many_requests():
    """One token each of 140000 requests of 512 pages, 32 heads, lists long enough to be
    joined: rows alone are within 32 bits of work, tiles of joined lists would not be."""
    N, H, T = 140000, 32, 96
    codes, scales, _ = make_cache([64], H, 1, nan_tail=False)
    cache = [codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV)]
    gen = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(N, H, 128, generator=gen, device=DEV, dtype=torch.bfloat16)
    idx = torch.full((H, N, T), -1, dtype=torch.int32, device=DEV)
    idx[..., 0] = 500
    out = torch.full_like(q, math.nan)
    # all blocks are page 0, of 512 x 64 tokens the row lists one page
    _, lse = ops.paged_attn(q, *cache, torch.zeros(N, 512, dtype=torch.int32, device=DEV),
                            torch.full((N,), 512 * 64, dtype=torch.int32, device=DEV),
                            torch.arange(N + 1, dtype=torch.int32, device=DEV), 16, 512 * 64,
                            topk_idx=idx, return_lse=True, out=out)
    del idx
    k, v = (c[0].double() * s[0].double()[:, None, None] for c, s in ((cache[0], cache[2]),
                                                                     (cache[1], cache[3])))
    for t in range(0, N, 10000):
        qr = q[t:t + 10000].double()
        x = torch.einsum("thd,hkd->thk", qr, k) / math.sqrt(128)
        w = torch.softmax(x, -1)
        sv = cache[3][0].double()
        bounds = (torch.einsum("thk,hkd->thd", w, v.abs()),
                  torch.einsum("thd,hkd->thk", qr.abs(), k.abs()).amax(-1) / math.sqrt(128),
                  (w.amax(-1) * sv)[..., None] * (v.abs() / sv[:, None, None]).sum(1))
        want = torch.einsum("thk,hkd->thd", w, v)
        err = (out[t:t + 10000].double() - want).abs()
        assert bool((err <= tolerance(want, bounds, 64)).all())
        want = torch.logsumexp(x, -1)
        ltol = 128 * 2.0 ** -23 * bounds[1] + 2.0 ** -20 + 64 * 2.0 ** -24 + 2.0 ** -22 * (
            want.abs() + 64)
        assert bool(((lse.T[t:t + 10000].double() - want).abs() <= ltol).all())


def test_equal_calls_give_equal_bits_and_other_types_are_cast():
    a = run_attend(32, 2, [5000, 3], [1, 1], seed=9)
    b = run_attend(32, 2, [5000, 3], [1, 1], seed=9)
    assert torch.equal(a, b)
    run_attend(32, 2, [130], [2], seed=9, pad=2, q_dtype=torch.float32)


def test_attention_refusals():
    codes, scales, table = make_cache([100], 2, 3)
    q = torch.zeros(1, 32, 128, dtype=torch.bfloat16, device=DEV)
    good = [q, codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV),
            i32(table), i32([100]), i32([0, 1]), 1, 100]
    ops.paged_attn(*good)
    for at, value in ((0, q[:, :31]), (0, q[..., :64]), (1, good[1].view(torch.uint8)),
                      (2, good[2][:1]), (3, good[3].double()), (5, i32(table + table)),
                      (6, i32([100, 100])), (7, i32([0]))):
        with pytest.raises(ValueError):
            ops.paged_attn(*[value if i == at else x for i, x in enumerate(good)])
    with pytest.raises(ValueError):
        ops.paged_attn(*good, topk_idx=i32([[[0]]]))
    with pytest.raises(ValueError):
        ops.paged_attn(*good, out=q.float())
    with pytest.raises(_native.LeanSelectError, match="heads per group"):
        ops.paged_attn(torch.zeros(1, 34, 128, dtype=torch.bfloat16, device=DEV), *good[1:])


# ---------------------------------------------------------------------------
# a run of the three, as a decode loop uses them
# ---------------------------------------------------------------------------

def test_prompt_then_decode_steps():
    """Two requests: ragged prompts, then steps of one token, against the oracle
    over what the cache holds."""
    gen = torch.Generator().manual_seed(21)
    G, H, width, pool = 2, 32, 8, 24
    cache = empty_cache(pool, G, 5)
    table, free = [[-1] * width for _ in range(3)], torch.randperm(pool, generator=gen).tolist()
    dev_table, dev_free, head = i32(table), i32(free), i32([0])
    context, at = [0, 0, 0], 0
    ctx = i32(context)
    mirror = [as_values(cache[0]), as_values(cache[1]), cache[2].double().cpu(),
              cache[3].double().cpu()]
    for new in ([130, 0, 63], [1, 1, 1], [1, 1, 1], [0, 70, 1], [2, 1, 1]):
        n = sum(new)
        plan = ops.plan_pages(ctx, i32(new), dev_table, dev_free, head, n)
        ref = ora.plan(context, new, table, free, at, n)
        check_plan(plan, ref, dev_table, table)
        k, v = (torch.randn(n, G, 128, generator=gen).bfloat16() for _ in range(2))
        q = torch.randn(n, H, 128, generator=gen).bfloat16()
        ops.append_kv(k.to(DEV), v.to(DEV), plan, *cache)
        ora.append(k, context, new, table, mirror[0], mirror[2])
        ora.append(v, context, new, table, mirror[1], mirror[3])
        got = ops.paged_attn(q.to(DEV), *cache, dev_table, plan.seq_lens, plan.cu_seqlens_q,
                             max(new), max(ref["seq"]))
        want, _, bounds = ora.attend(q, *mirror, table, ref["seq"], ref["cu_q"])
        tol = tolerance(want, bounds, 256)
        assert bool(((got.double().cpu() - want).abs() <= tol).all())
        context, at = ref["seq"], ref["head"]
        ctx, head = plan.seq_lens, plan.free_head


# ---------------------------------------------------------------------------
# streams, graphs, custom ops
# ---------------------------------------------------------------------------

def step_inputs(batch, G, H, seed, length):
    """Device tensors of a decode step over a filled cache."""
    gen = torch.Generator().manual_seed(seed)
    seq = torch.randint(1, length + 1, (batch,), generator=gen).tolist()
    codes, scales, table = make_cache([n + 8 for n in seq], G, seed, nan_tail=False)
    cache = [codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV)]
    q = torch.randn(batch, H, 128, generator=gen).bfloat16().to(DEV)
    return seq, cache, i32(table), q


def test_calls_on_several_streams_at_once():
    """Interleaved steps of four batches on four streams give what each gives alone."""
    steps = [step_inputs(b, 2, 32, b, 3000) for b in (1, 7, 64, 3)]
    args = [(q, *cache, table, i32(seq), i32(list(range(len(seq) + 1))), 1, max(seq))
            for seq, cache, table, q in steps]
    alone = [ops.paged_attn(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[] for _ in args]
    for _ in range(6):
        for i, (s, a) in enumerate(zip(streams, args)):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attn(*a))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(o, alone[i]) for o in outs)


def test_two_captured_steps_replayed_together():
    """Graphs of a whole decode step (plan, write, attention) advance on the device;
    two of them replayed on two streams equal the eager steps."""
    G, H, steps = 2, 16, 5

    def state(batch, seed):
        seq, cache, table, _ = step_inputs(batch, G, H, seed, 200)
        width = table.shape[1]
        more = torch.full((batch, 3), -1, dtype=torch.int32, device=DEV)
        pool = cache[0].shape[0]
        grown = [torch.cat([c, c[:batch]]).clone() if c.dtype != FP8 else
                 torch.cat([c.view(torch.uint8), c.view(torch.uint8)[:batch]]).view(FP8).clone()
                 for c in cache]
        # the make_cache tables already hold room for eight more tokens
        gen = torch.Generator().manual_seed(seed)
        feed = [(torch.randn(batch, G, 128, generator=gen).bfloat16().to(DEV),
                 torch.randn(batch, G, 128, generator=gen).bfloat16().to(DEV),
                 torch.randn(batch, H, 128, generator=gen).bfloat16().to(DEV))
                for _ in range(steps)]
        table = torch.cat([table, more], dim=1)
        for b, n in enumerate(seq):  # blocks past the cached tokens are handed out again
            table[b, up(n):] = -1
        return dict(ctx=i32(seq), cache=grown, table=table.contiguous(), width=width,
                    free=torch.arange(pool, pool + batch, dtype=torch.int32, device=DEV),
                    head=i32([0]), feed=feed, batch=batch, ones=i32([1] * batch))

    def step(s, k, v, q):
        plan = ops.plan_pages(s["ctx"], s["ones"], s["table"], s["free"], s["head"], s["batch"])
        ops.append_kv(k, v, plan, *s["cache"])
        out = ops.paged_attn(q, *s["cache"], s["table"], plan.seq_lens, plan.cu_seqlens_q, 1, 256)
        s["ctx"].copy_(plan.seq_lens)
        s["head"].copy_(plan.free_head)
        return out

    eager = []
    for batch, seed in ((5, 1), (9, 2)):
        s = state(batch, seed)
        eager.append([step(s, *f).clone() for f in s["feed"]])
        eager[-1].append([c.clone() for c in s["cache"]])
    captured = []
    for batch, seed in ((5, 1), (9, 2)):
        s = state(batch, seed)
        warm = state(batch, seed)
        step(warm, *warm["feed"][0])
        feed = [t.clone() for t in s["feed"][0]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s, *feed)
        captured.append((s, feed, graph, out, torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for t in range(steps):
        for s, feed, graph, out, stream, outs in captured:
            with torch.cuda.stream(stream):
                for dst, src in zip(feed, s["feed"][t]):
                    dst.copy_(src)
                graph.replay()
                outs.append(out.clone())
    torch.cuda.synchronize()
    for want, (s, _, _, _, _, outs) in zip(eager, captured):
        assert all(torch.equal(a, b) for a, b in zip(want[:-1], outs))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(want[-1], s["cache"]))


def test_custom_ops_run_the_same_kernels():
    import leanselect_b200.torch_ops  # noqa: F401

    registered = torch.ops.leanselect_b200
    seq, cache, table, q = step_inputs(4, 2, 16, 3, 500)
    cu = i32([0, 1, 2, 3, 4])
    want, want_lse = ops.paged_attn(q, *cache, table, i32(seq), cu, 1, max(seq), return_lse=True)
    out, lse = registered.paged_attn(q, *cache, table, i32(seq), cu, 1, max(seq), None, 0.0, True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    tables = [table.clone(), table.clone()]
    free = i32(list(range(10)))
    plan = ops.plan_pages(i32(seq), i32([1, 0, 2, 1]), tables[0], free, i32([1]), 4)
    got = registered.plan_pages(i32(seq), i32([1, 0, 2, 1]), tables[1], free, i32([1]), 4)
    for a, b in zip(got, (plan.seq_lens, plan.cu_seqlens_q, plan.cu_blocks, plan.slots,
                          plan.positions, plan.free_head)):
        assert torch.equal(a, b)
    assert torch.equal(*tables)
    k = torch.randn(4, 2, 128, device=DEV).bfloat16()
    twins = [[c.clone() for c in cache] for _ in range(2)]
    ops.append_kv(k, k, plan, *twins[0])
    registered.append_kv(k, k, plan.context_lens, *got[:4], *twins[1])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*twins))


# ---------------------------------------------------------------------------
# the host model
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def model():
    from leanselect_b200.model import MiniCPMShape, PrefillModel

    shape = MiniCPMShape(vocab_size=500, hidden_size=256, intermediate_size=512, num_layers=2,
                         num_heads=16, num_kv_heads=2, max_position=4096,
                         original_max_position=4096, router_heads=4, router_dim=32)
    return PrefillModel(shape, DEV, seed=3)


def test_model_decodes_over_its_cache(model, monkeypatch):
    """Prefill with a cache, a draft of several tokens and single steps: each layer's
    write and attention equal the oracle's on the tensors the model gave them."""
    from leanselect_b200 import PagedKVCache

    s = model.shape
    lengths = [150, 64, 5]
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, s.vocab_size, (sum(lengths),), generator=gen).to(DEV)
    cu = i32(prefix(lengths))
    cache = PagedKVCache(s.num_layers, 3, 200, 12, s.num_kv_heads, device=DEV)
    plain = model.prefill(ids, cu, lengths)
    assert torch.equal(model.prefill(ids, cu, lengths, cache=cache), plain)
    assert cache.lengths == lengths and cache.seq_lens.tolist() == lengths

    calls = []
    append, attend = ops.append_kv, ops.paged_attn

    def spy_append(k, v, plan, *layer):
        before = [as_values(layer[0]), as_values(layer[1]), layer[2].double().cpu(),
                  layer[3].double().cpu()]
        append(k, v, plan, *layer)
        context, new = plan.context_lens.tolist(), torch.diff(plan.cu_seqlens_q).tolist()
        table = cache.block_table.tolist()
        ora.append(k.cpu(), context, new, table, before[0], before[2])
        ora.append(v.cpu(), context, new, table, before[1], before[3])
        for got, want in zip((as_values(layer[0]), as_values(layer[1]), layer[2].double().cpu(),
                              layer[3].double().cpu()), before):
            assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
        calls.append("write")

    def spy_attend(q, *args, **kwargs):
        out = attend(q, *args, **kwargs)
        kp, vp, ks, vs, table, seq, cuq = args[:7]
        idx = kwargs.get("topk_idx")
        want, _, bounds = ora.attend(q.cpu(), as_values(kp), as_values(vp), ks.cpu(), vs.cpu(),
                                     table.tolist(), seq.tolist(), cuq.tolist(),
                                     None if idx is None else idx.cpu())
        assert bool(((out.double().cpu() - want).abs() <= tolerance(want, bounds, 256)).all())
        calls.append("attend")
        return out

    monkeypatch.setattr(ops, "append_kv", spy_append)
    monkeypatch.setattr(ops, "paged_attn", spy_attend)
    new = [3, 1, 0]
    draft = torch.randint(0, s.vocab_size, (4,), generator=gen).to(DEV)
    logits = model.decode(draft, cache, new)
    assert logits.shape == (4, s.vocab_size) and bool(torch.isfinite(logits).all())
    # one token each, over listed pages: the sink and the last pages
    lists = torch.tensor([[[0, 1, 2], [0, 1, -1], [0, -1, -1]]] * 2, dtype=torch.int32, device=DEV)
    logits = model.decode(draft[:3], cache, page_lists=lambda i, q: lists)
    assert logits.shape == (3, s.vocab_size)
    assert cache.lengths == [154, 66, 6] and cache.seq_lens.tolist() == [154, 66, 6]
    assert calls == ["write", "attend"] * (2 * s.num_layers)
    # A finished request's pages serve the next one.
    cache.release(1)
    assert cache.taken == 3 + 1 and cache.seq_lens.tolist() == [154, 0, 6]
    model.decode(torch.zeros(40, dtype=torch.long, device=DEV), cache, [0, 40, 0])
    assert cache.block_table[1, 0].item() >= 0 and cache.taken == 5


def test_generate_is_the_loop_of_its_steps(model):
    from leanselect_b200 import PagedKVCache
    from leanselect_b200.runner import PrefillRunner

    runner = PrefillRunner(model.shape, DEV, model=model)
    lengths, steps = [70, 3], 4
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(0, model.shape.vocab_size, (sum(lengths),), generator=gen)
    out = runner.generate(ids, lengths, steps)
    assert out.shape == (2, steps) and out.device.type == "cpu"
    cache = PagedKVCache(model.shape.num_layers, 2, 80, 4, 2, device=DEV)
    tok = model.prefill(ids.to(DEV), i32(prefix(lengths)), lengths, cache=cache).argmax(-1)
    for t in range(steps):
        assert torch.equal(tok.cpu(), out[:, t])
        if t + 1 < steps:
            tok = model.decode(tok, cache).argmax(-1)
    for bad in (([], 3), ([0, 5], 3), (lengths, 0)):
        with pytest.raises(ValueError):
            runner.generate(ids, *bad)


def test_model_decode_refusals(model):
    from leanselect_b200 import PagedKVCache

    s = model.shape
    cache = PagedKVCache(s.num_layers, 1, 65, 1, s.num_kv_heads, device=DEV)
    with pytest.raises(ValueError, match="prefill"):
        model.decode(torch.zeros(1, dtype=torch.long, device=DEV), cache)
    ids = torch.zeros(64, dtype=torch.long, device=DEV)
    model.prefill(ids, i32([0, 64]), [64], cache=cache)
    with pytest.raises(ValueError, match="empty"):
        model.prefill(ids, i32([0, 64]), [64], cache=cache)
    with pytest.raises(ValueError, match="sum"):
        model.decode(ids[:2], cache)
    with pytest.raises(ValueError, match="new tokens"):
        model.decode(ids[:0], cache, [0])
    with pytest.raises(ValueError, match="tokens"):
        model.decode(ids[:2], cache, [2])
    with pytest.raises(RuntimeError, match="out of pages"):
        model.decode(ids[:1], cache)
    assert cache.lengths == [64] and cache.taken == 1


@pytest.mark.parametrize("size", [0.5, 1000.0, 1e6, math.inf])
def test_a_failed_step_keeps_only_the_scale_it_raised(size):
    """A step fails after its rows were written into a half-filled page: lengths and pages
    are the old ones, older values moved by no more than the rounding to a scale that grew,
    and the next step, with other rows, is the oracle's over what the page holds now."""
    from leanselect_b200 import PagedKVCache

    gen = torch.Generator().manual_seed(8)

    def rows(n, scale=1.0):
        return (torch.randn(n, 2, 128, generator=gen) * scale).bfloat16().to(DEV)

    cache = PagedKVCache(1, 1, 192, 3, 2, device=DEV)
    with cache.step([104]) as plan:
        ops.append_kv(rows(104), rows(104), plan, *cache.layer(0))
    layer, page = cache.layer(0), int(cache.block_table[0, 1])
    before = [(as_values(layer[i])[page, :, :40], layer[2 + i][page].double().cpu())
              for i in range(2)]
    first = [t[cache.block_table[0, 0]].clone() for t in layer]
    with pytest.raises(RuntimeError, match="a later layer"):
        with cache.step([30]) as plan:
            ops.append_kv(rows(30, size), rows(30, size), plan, *layer)
            raise RuntimeError("a later layer")
    assert cache.lengths == [104] and cache.seq_lens.tolist() == [104] and cache.taken == 2
    assert cache.free_head.tolist() == [2]
    for a, t in zip(first, layer):  # full pages as they were
        assert torch.equal(a.view(torch.uint8), t[cache.block_table[0, 0]].view(torch.uint8))
    for i, (codes, old) in enumerate(before):
        now = layer[2 + i][page].double().cpu()
        assert bool((now >= old).all()) and (size > 1 or torch.equal(now, old))
        x = codes * old[:, None, None]
        y = as_values(layer[i])[page, :, :40] * now[:, None, None]
        assert bool(((x - y).abs() <= 2.0 ** -10 * now[:, None, None]).all())
        normal = x.abs() >= 2.0 ** -6 * now[:, None, None]
        assert torch.equal(x[normal], y[normal])
    mirror = [as_values(layer[0]), as_values(layer[1]), layer[2].double().cpu(),
              layer[3].double().cpu()]
    k, v = rows(1), rows(1)
    with cache.step([1]) as plan:
        ops.append_kv(k, v, plan, *layer)
        table = cache.block_table.tolist()
    ora.append(k.cpu(), [104], [1], table, mirror[0], mirror[2])
    ora.append(v.cpu(), [104], [1], table, mirror[1], mirror[3])
    for got, want in zip((as_values(layer[0]), as_values(layer[1]), layer[2].double().cpu(),
                          layer[3].double().cpu()), mirror):
        assert torch.equal(got.nan_to_num(1234.0), want.nan_to_num(1234.0))


def test_failed_steps_leave_the_cache_as_it_was(model):
    """A prefill and a decode step that raise between layers, then the same steps again."""
    from leanselect_b200 import PagedKVCache

    s = model.shape
    gen = torch.Generator().manual_seed(12)
    lengths = [70, 128]
    ids = torch.randint(0, s.vocab_size, (sum(lengths),), generator=gen).to(DEV)
    cu = i32(prefix(lengths))
    caches = [PagedKVCache(s.num_layers, 2, 192, 6, s.num_kv_heads, device=DEV) for _ in range(2)]
    with pytest.raises(ValueError, match="sum"):
        model.prefill(ids, cu, [70, 127], cache=caches[0])
    shallow = PagedKVCache(1, 2, 192, 6, s.num_kv_heads, device=DEV)
    with pytest.raises(IndexError):
        model.prefill(ids, cu, lengths, cache=shallow)
    for c in (caches[0], shallow):
        assert c.lengths == [0, 0] and c.taken == 0 and c.rope_len == 0
    toks = [model.prefill(ids, cu, lengths, cache=c).argmax(-1) for c in caches]
    assert torch.equal(toks[0], toks[1])

    def fails_in_the_second_layer(i, q):
        if i:
            raise RuntimeError("no lists")
        return torch.zeros(s.num_kv_heads, 2, 1, dtype=torch.int32, device=DEV)

    with pytest.raises(RuntimeError, match="no lists"):
        model.decode(toks[0], caches[0], page_lists=fails_in_the_second_layer)
    assert caches[0].lengths == lengths and caches[0].taken == 4
    for _ in range(2):
        logits = [model.decode(toks[0], c) for c in caches]
        assert torch.equal(*logits)
    assert torch.equal(caches[0].block_table, caches[1].block_table)
