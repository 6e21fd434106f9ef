"""The paged cache's argument checks and its 64-bit oracle, without a GPU."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from leanselect_b200 import _native, ops
from oracle import paged_cache as ora

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p((1 << 20) + 4)
INVALID, UNSUPPORTED, ALIGNMENT = (_native.LS_ERR_INVALID_ARGUMENT, _native.LS_ERR_UNSUPPORTED,
                                   _native.LS_ERR_ALIGNMENT)


def refused(name, base, changes, code, text):
    args = list(base)
    for at, value in changes.items():
        args[at] = value
    lib = _native.load()
    assert getattr(lib, name)(*args) == code
    assert text in lib.ls_last_error()


PLAN = [FAKE, FAKE, 4, FAKE, 8, FAKE, 16, FAKE, 100, FAKE, FAKE, FAKE, FAKE, FAKE, ODD, None, None]


@pytest.mark.parametrize("changes, code, text", [
    ({0: None}, INVALID, b"null"),
    ({9: None}, INVALID, b"null output"),
    ({14: FAKE}, INVALID, b"free_head"),
    ({2: 0}, INVALID, b"sizes"),
    ({4: 0}, INVALID, b"sizes"),
    ({5: None}, INVALID, b"free_pages"),
    ({8: -1}, INVALID, b"total_new"),
    ({8: 1 << 31}, INVALID, b"total_new"),
    ({12: None}, INVALID, b"slots"),
    ({2: _native.LS_MAX_PLAN_BATCH + 1}, UNSUPPORTED, b"LS_MAX_PLAN_BATCH"),
    ({}, INVALID, b"seq_lens must not be an input"),
])
def test_plan_refusals(changes, code, text):
    refused("ls_plan_pages", PLAN, changes, code, text)


APPEND = [FAKE, FAKE, 256, 256, 10, 2, 2, 128, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
          FAKE, 5, None, None]


@pytest.mark.parametrize("changes, code, text", [
    ({0: None}, INVALID, b"null"),
    ({13: None}, INVALID, b"null cache"),
    ({17: 0}, INVALID, b"cache sizes"),
    ({17: 1 << 24}, INVALID, b"out of range"),
    ({7: 64}, UNSUPPORTED, b"head_dim"),
    ({2: 128}, INVALID, b"strides"),
    ({3: 260}, ALIGNMENT, b"strides"),
    ({1: ODD}, ALIGNMENT, b"v is not"),
    ({14: ODD}, ALIGNMENT, b"v_pages"),
    ({5: 0}, INVALID, b"sizes"),
])
def test_append_refusals(changes, code, text):
    refused("ls_append_kv", APPEND, changes, code, text)


def test_append_of_nothing_is_ok():
    args = list(APPEND)
    args[0] = args[1] = args[12] = None
    args[4] = 0
    assert _native.load().ls_append_kv(*args) == _native.LS_OK


ATTEND = [FAKE, FAKE, FAKE, FAKE, FAKE, 5, FAKE, 4, FAKE, FAKE, 2, 1, 200, 2, 32, 2, 128, FAKE, 7,
          0.0, 1, FAKE, 1 << 30, FAKE, None, None, None]


@pytest.mark.parametrize("changes, code, text", [
    ({0: None}, INVALID, b"null"),
    ({1: None}, INVALID, b"null cache"),
    ({6: None}, INVALID, b"null"),
    ({16: 64}, UNSUPPORTED, b"head_dim"),
    ({14: 34}, UNSUPPORTED, b"heads per group"),
    ({14: 31}, INVALID, b"multiple"),
    ({18: 129}, UNSUPPORTED, b"LS_MAX_TOPK"),
    ({17: None}, INVALID, b"topk_idx"),
    ({7: 0}, INVALID, b"sizes"),
    ({12: -1}, INVALID, b"max_seqlen"),
    ({0: ODD}, ALIGNMENT, b"q is not"),
    ({22: 100}, INVALID, b"workspace"),
    ({21: None}, INVALID, b"workspace"),
    ({21: ODD}, ALIGNMENT, b"workspace"),
    ({13: 1 << 31}, INVALID, b"out of range"),
])
def test_attention_refusals(changes, code, text):
    refused("ls_paged_attn", ATTEND, changes, code, text)


SCHEDULE = r"""
#include <cstdio>
#include "paged_schedule.h"

int main() {
  ls::PagedSizes s;
  long long total_q;
  while (scanf("%lld %d %d %d %d %d %d %d", &total_q, &s.batch, &s.num_kv_heads,
               &s.heads_per_group, &s.topk, &s.max_blocks, &s.max_seqlen_q, &s.max_seqlen_k) == 8) {
    s.total_q = total_q;
    const ls::PagedSchedule r = ls::paged_schedule(s, 148);
    printf("%d %d %d %d\n", ls::paged_rows_fit(s) ? 1 : 0, r.units, r.pack, r.ranges);
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_scheduled_work_stays_within_32_bits(tmp_path):
    """Every call the range check lets through gives the kernels less than 2^31 units,
    whatever way the tokens are dealt to the requests."""
    root = Path(__file__).resolve().parents[1]
    src, exe = tmp_path / "schedule.cpp", tmp_path / "schedule"
    src.write_text(SCHEDULE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I",
                    str(root / "leanselect_b200" / "csrc"), str(src), "-o", str(exe)], check=True)
    cases = [(n, b, G, hg, topk, blocks, mq, 64 * min(blocks, 512))
             for hg in (1, 3, 8, 16) for topk in (0, 1, 96, 128) for blocks in (1, 40, 512, 2048)
             for mq in (1, 2, 16, 1000) for G in (1, 32)
             for n, b in ((1, 1), (2000, 1), (140000, 140000), (140000, 1000), (4200000, 4199985),
                          (16000000, 16000000), (1 << 26, 3))]
    text = "\n".join(" ".join(map(str, c)) for c in cases)
    out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout
    joined = alone = 0
    for (n, b, G, hg, topk, blocks, mq, mk), line in zip(cases, out.splitlines(), strict=True):
        fits, units, pack, ranges = map(int, line.split())
        assert bool(fits) == (n * G * ((topk or blocks) + 4) < 1 << 31)
        if not fits:
            continue
        assert 1 <= ranges <= 296 and 1 <= pack <= max(1, min(16 // hg, mq))
        # requests of a token each and one of the rest; and tokens dealt evenly
        for lens in ([(b - 1, 1), (1, n - b + 1)], [(b - n % b, n // b), (n % b, n // b + 1)]):
            tiles = sum(count * -(-m // pack) for count, m in lens)
            if topk and pack == 1:
                work = n * G * (units + 4)
            else:
                work = tiles * G * (min(pack * topk, blocks) + 4 if topk else blocks + 4)
            assert work < 1 << 31, (n, b, G, hg, topk, blocks, mq)
        joined += bool(topk) and pack > 1
        alone += (n, b, G, hg, topk, blocks, mq) == (140000, 140000, 32, 1, 96, 512, 16) and pack == 1
    assert joined > 20 and alone == 1


def test_attention_of_no_rows_is_ok():
    args = list(ATTEND)
    args[13] = 0
    assert _native.load().ls_paged_attn(*args) == _native.LS_OK


def test_cpu_tensors_raise():
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.plan_pages(i32, i32, torch.zeros(2, 4, dtype=torch.int32), i32, i32[:1], 0)
    pages = torch.zeros(1, 2, 64, 128).to(torch.float8_e4m3fn)
    scale = torch.ones(1, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attn(torch.zeros(2, 32, 128), pages, pages, scale, scale,
                       torch.zeros(2, 1, dtype=torch.int32), i32, torch.zeros(3, dtype=torch.int32),
                       1, 1)


def test_token_rows_are_laid_out_for_the_kernel():
    """Rows the kernel cannot take as they stand are copied, also where torch calls them
    contiguous: one token with its heads first, rows that begin off a 16-byte boundary."""
    heads_first = torch.randn(4, 1, 128).bfloat16().transpose(0, 1)
    odd = torch.randn(3 * 4 * 128 + 1).bfloat16()[1:].view(3, 4, 128)
    spread = torch.randn(3, 4, 256).bfloat16()[..., ::2]
    same = torch.zeros(1, 4, 128).bfloat16().expand(3, 4, 128)
    for t in (heads_first, odd, spread, same, heads_first.float()):
        rows = ops._token_rows(t)
        assert rows.dtype == torch.bfloat16 and torch.equal(rows, t.bfloat16())
        assert rows.stride() == (4 * 128, 128, 1) and rows.data_ptr() % 16 == 0
    fused = torch.randn(3, 1024).bfloat16()[:, 512:].view(3, 4, 128)
    assert ops._token_rows(fused) is fused


def test_oracle_rounding_is_that_of_torch():
    """Every representable value, every midpoint between two and its neighbours."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), -mid])
    assert torch.equal(ora.e4m3(x), x.float().to(torch.float8_e4m3fn).double())
    assert float(ora.e4m3(torch.tensor(1e30, dtype=torch.float64))) == 448.0
    assert ora.e4m3(torch.tensor(float("nan"), dtype=torch.float64)).isnan()


def test_oracle_plan_by_hand():
    table = [[7, -1, -1], [5, 6, -1]]
    p = ora.plan([63, 128], [3, 1], table, [9, 8], 0, 6)
    assert table == [[7, 9, -1], [5, 6, 8]]
    assert p["slots"] == [7 * 64 + 63, 9 * 64, 9 * 64 + 1, 8 * 64, -1, -1]
    assert p["positions"] == [63, 64, 65, 128, 0, 0]
    assert (p["seq"], p["cu_q"], p["cu_blocks"], p["head"]) == ([66, 129], [0, 3, 4], [0, 2, 3], 2)


def test_oracle_attention_is_softmax_over_the_listed_keys():
    torch.manual_seed(0)
    k, v = (ora.e4m3(torch.randn(4, 1, 64, 128, dtype=torch.float64)) for _ in range(2))
    q = torch.randn(1, 2, 128)
    one = torch.ones(4, 1)
    out, lse, _ = ora.attend(q, k, v, one, one, [[2, 0, 3]], [130], [0, 1],
                                idx=torch.tensor([[[2, 0, 2, -1]]]))
    kk = torch.cat([k[2, 0], k[3, 0, :2]])
    vv = torch.cat([v[2, 0], v[3, 0, :2]])
    ref = torch.nn.functional.scaled_dot_product_attention(q[0].double(), kk, vv)
    assert torch.allclose(out[0], ref, atol=1e-12)
    assert torch.allclose(lse[:, 0], torch.logsumexp(q[0].double() @ kk.T / 128 ** 0.5, -1))


def test_cache_refuses_on_the_host():
    """Bookkeeping errors are raised before anything is launched."""
    from leanselect_b200 import PagedKVCache

    for bad in (dict(batch=0), dict(num_layers=0), dict(num_pages=0), dict(head_dim=64),
                dict(batch=_native.LS_MAX_PLAN_BATCH + 1), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(num_layers=1, batch=2, max_tokens=100, num_pages=3,
                                   num_kv_heads=1, device="cpu"), **bad})
    cache = PagedKVCache(1, 2, 100, 3, 1, device="cpu")
    assert cache.block_table.shape == (2, 2) and cache.max_seqlen == 0
    for new in ([1], [1, -1], [101, 0]):
        with pytest.raises(ValueError):
            cache.plan(new)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.plan([100, 70])
    assert cache.lengths == [0, 0] and cache.taken == 0


def test_custom_op_shapes():
    import leanselect_b200.torch_ops  # noqa: F401

    def t(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    registered = torch.ops.leanselect_b200
    fp8 = torch.float8_e4m3fn
    seq, cu_q, cu_blocks, slots, pos, head = registered.plan_pages(t(5), t(5), t(5, 9), t(30), t(1),
                                                                   70)
    assert (seq.shape, cu_q.shape, cu_blocks.shape, head.shape) == ((5,), (6,), (6,), (1,))
    assert slots.shape == pos.shape == (70,) and slots.dtype == pos.dtype == torch.int64
    cache = (t(8, 2, 64, 128, dtype=fp8), t(8, 2, 64, 128, dtype=fp8),
             t(8, 2, dtype=torch.float32), t(8, 2, dtype=torch.float32))
    kv = t(70, 2, 128, dtype=torch.bfloat16)
    assert registered.append_kv(kv, kv, t(5), seq, cu_q, cu_blocks, slots, *cache) is None
    out, lse = registered.paged_attn(t(70, 16, 128, dtype=torch.bfloat16), *cache, t(5, 9), seq,
                                     cu_q, 30, 500, None, 0.0, True)
    assert out.shape == (70, 16, 128) and lse.shape == (16, 70) and lse.dtype == torch.float32


def test_kernels_launched_early_read_with_ordinary_loads():
    """Such a kernel begins while its predecessor still writes its inputs: loads that need
    data which is constant for the kernel's life (``__ldg``, ``ld.global.nc``, and what the
    compiler makes of const restrict pointers) must not read them."""
    csrc = Path(__file__).resolve().parents[1] / "leanselect_b200" / "csrc"
    early = [f for f in csrc.glob("*.cu") if "launch_early(" in f.read_text()]
    assert {f.name for f in early} >= {"paged_attn.cu", "paged_cache.cu"}
    for f in early:
        text = f.read_text()
        for bad in ("__ldg(", "__ldca(", "global.nc", "__restrict__", "find_sequence("):
            assert bad not in text, (f.name, bad)
