"""Torch-tensor wrappers over the C ABI (device memory and streams come from PyTorch).

Every function takes CUDA tensors, launches on the current stream and returns
new tensors; nothing here computes on the CPU.  bf16 is the compute type of
the kernels: other floating inputs are cast to bf16 at the boundary.

A per-device int32 *status word* collects device-side error bits
(``LS_DEVERR_*``).  It is only read (a stream synchronisation) by
:func:`check_status`, which the tests and ``smoke()`` call.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

import torch

from . import _native
from ._native import LS_MAX_ATTN_SPLITS, LS_MAX_TOPK, LeanSelectError

_STATUS: dict[int, torch.Tensor] = {}


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("leanselect_b200 operates on CUDA tensors only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same CUDA device")
    if dev is None:
        raise ValueError("no tensor given")
    return dev


def _call(dev: torch.device, name: str, *args) -> None:
    """One C-ABI call with ``dev`` as the current device (the kernels launch on
    the calling thread's current device; the reference guards the same way)."""
    with torch.cuda.device(dev):
        _native.call(name, *args)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def status_word(device: torch.device) -> torch.Tensor:
    """The device's status word (int32, accumulates LS_DEVERR_* bits)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    word = _STATUS.get(idx)
    if word is None:
        word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _STATUS[idx] = word
    return word


def check_status(device: torch.device | int | None = None, reset: bool = True) -> int:
    """Synchronise, return the status bits and raise if any is set."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    elif isinstance(device, int):
        device = torch.device("cuda", device)
    word = status_word(device)
    bits = int(word.item())
    if reset and bits:
        word.zero_()
    if bits:
        names = [n for n, b in (("TIMEOUT", _native.LS_DEVERR_TIMEOUT),
                                ("PAGE_INDEX", _native.LS_DEVERR_PAGE_INDEX),
                                ("SEQLENS", _native.LS_DEVERR_SEQLENS),
                                ("PAGES", _native.LS_DEVERR_PAGES)) if bits & b]
        raise LeanSelectError(-bits, f"device status bits set: {'|'.join(names)}")
    return bits


def _bf16(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t.contiguous()


def _i32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t.contiguous()


def host_lengths(cu_seqlens: torch.Tensor | Sequence[int]) -> list[int]:
    """Sequence lengths on the host (one device->host copy, as the reference does)."""
    cu = cu_seqlens.detach().to("cpu").tolist() if torch.is_tensor(cu_seqlens) else list(cu_seqlens)
    return [int(cu[i + 1]) - int(cu[i]) for i in range(len(cu) - 1)]


def atom_count(n: int, kernel_size: int = 32, kernel_stride: int = 16) -> int:
    """Atoms ``CompressK`` keeps for a sequence of ``n`` keys (minicpm.py:710-750)."""
    return 0 if n < kernel_size else (n - kernel_size) // kernel_stride + 1


# ---------------------------------------------------------------------------
# a2: folded weights
# ---------------------------------------------------------------------------

@dataclass
class FoldedWeights:
    """Selector weights in the layouts the kernels consume."""

    wq_t: torch.Tensor   # [G, F, Hg*D] bf16
    wk_t: torch.Tensor   # [G, F, D] bf16
    num_heads: int
    num_kv_heads: int
    head_dim: int
    width: int


def fold_weights(head_mix: torch.Tensor, kv_head_mix: torch.Tensor, q_proj: torch.Tensor,
                 k_proj: torch.Tensor, *, reference_layout: bool = False,
                 dtype: torch.dtype | None = None):
    """``LeanSelectSelector.fused_weights`` (selector.py:144-158) on the GPU.

    With ``reference_layout`` returns ``(q_fused [H, D, F], kv_fused [G, D, F])``
    in fp32 (``dtype=None``) or bf16; otherwise a :class:`FoldedWeights`.
    """
    dev = _require_cuda(head_mix, kv_head_mix, q_proj, k_proj)
    hm, km = head_mix.detach().float().contiguous(), kv_head_mix.detach().float().contiguous()
    qp, kp = q_proj.detach().float().contiguous(), k_proj.detach().float().contiguous()
    H, R = hm.shape
    G = km.shape[0]
    _, D, r = qp.shape
    F = R * r
    if H % G:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    s = _stream(dev)
    if reference_layout:
        if dtype in (None, torch.float32):
            qf = torch.empty(H, D, F, dtype=torch.float32, device=dev)
            kf = torch.empty(G, D, F, dtype=torch.float32, device=dev)
            _call(dev, "ls_fold_weights", hm.data_ptr(), km.data_ptr(), qp.data_ptr(),
                       kp.data_ptr(), H, G, D, R, r, qf.data_ptr(), kf.data_ptr(), None, None,
                       None, None, s)
            if dtype is None or dtype == torch.float32:
                return qf, kf
        if dtype == torch.bfloat16:
            qb = torch.empty(H, D, F, dtype=torch.bfloat16, device=dev)
            kb = torch.empty(G, D, F, dtype=torch.bfloat16, device=dev)
            _call(dev, "ls_fold_weights", hm.data_ptr(), km.data_ptr(), qp.data_ptr(),
                       kp.data_ptr(), H, G, D, R, r, None, None, qb.data_ptr(), kb.data_ptr(),
                       None, None, s)
            return qb, kb
        # Other dtypes: the reference casts the fp32 product (selector.py:155-157).
        qf = torch.empty(H, D, F, dtype=torch.float32, device=dev)
        kf = torch.empty(G, D, F, dtype=torch.float32, device=dev)
        _call(dev, "ls_fold_weights", hm.data_ptr(), km.data_ptr(), qp.data_ptr(),
                   kp.data_ptr(), H, G, D, R, r, qf.data_ptr(), kf.data_ptr(), None, None,
                   None, None, s)
        return qf.to(dtype), kf.to(dtype)
    hg = H // G
    wq_t = torch.empty(G, F, hg * D, dtype=torch.bfloat16, device=dev)
    wk_t = torch.empty(G, F, D, dtype=torch.bfloat16, device=dev)
    _call(dev, "ls_fold_weights", hm.data_ptr(), km.data_ptr(), qp.data_ptr(), kp.data_ptr(),
               H, G, D, R, r, None, None, None, None, wq_t.data_ptr(), wk_t.data_ptr(), s)
    return FoldedWeights(wq_t, wk_t, H, G, D, F)


# ---------------------------------------------------------------------------
# a1: compression
# ---------------------------------------------------------------------------

def compressed_seqlens(cu_seqlens_k: torch.Tensor, kernel_size: int = 32,
                       kernel_stride: int = 16) -> torch.Tensor:
    """``cu_seqlens_compressed`` of ``calc_chunks_with_stride`` (minicpm.py:710-750)."""
    dev = _require_cuda(cu_seqlens_k)
    cu = _i32(cu_seqlens_k)
    out = torch.empty_like(cu)
    _call(dev, "ls_compressed_seqlens", cu.data_ptr(), cu.numel() - 1, kernel_size,
               kernel_stride, out.data_ptr(), status_word(dev).data_ptr(), _stream(dev))
    return out


def compress_keys(k: torch.Tensor, cu_seqlens_k: torch.Tensor, *, kernel_size: int = 32,
                  kernel_stride: int = 16, lengths: Sequence[int] | None = None,
                  total_c: int | None = None):
    """``CompressK.forward`` (minicpm.py:1169-1185): ``k [total_k, G, D] -> (kc, cu_c)``.

    ``lengths`` (host sequence lengths) or ``total_c`` (the number of atoms)
    avoids the device->host copy of ``cu_seqlens_k`` that sizing the output
    otherwise needs.
    """
    dev = _require_cuda(k, cu_seqlens_k)
    if k.ndim != 3:
        raise ValueError("k must be [total_k, num_kv_heads, head_dim]")
    cu = _i32(cu_seqlens_k)
    if total_c is None:
        lens = list(lengths) if lengths is not None else host_lengths(cu)
        total_c = sum(atom_count(n, kernel_size, kernel_stride) for n in lens)
    if k.dtype == torch.float32:
        # fp32 keys stay fp32, as CompressK keeps the input dtype.
        kf = k.contiguous()
        kc = torch.empty(total_c, k.shape[1], k.shape[2], dtype=torch.float32, device=dev)
        cu_c = torch.empty_like(cu)
        _call(dev, "ls_compress_keys_f32", kf.data_ptr(), cu.data_ptr(), cu.numel() - 1,
              kf.shape[0], k.shape[1], k.shape[2], kernel_size, kernel_stride,
              _ptr(kc) if total_c else None, cu_c.data_ptr(), total_c,
              status_word(dev).data_ptr(), _stream(dev))
        return kc, cu_c
    kb = _bf16(k)
    kc = torch.empty(total_c, k.shape[1], k.shape[2], dtype=torch.bfloat16, device=dev)
    cu_c = torch.empty_like(cu)
    _call(dev, "ls_compress_keys", kb.data_ptr(), cu.data_ptr(), cu.numel() - 1, kb.shape[0],
               k.shape[1], k.shape[2], kernel_size, kernel_stride, _ptr(kc) if total_c else None,
               cu_c.data_ptr(), total_c, status_word(dev).data_ptr(), _stream(dev))
    return kc, cu_c


def compress_keys_dual(k: torch.Tensor, cu_seqlens_k: torch.Tensor, *,
                       lengths: Sequence[int] | None = None):
    """``compress_k`` (32/16) and ``compress_k2`` (128/64) of one prefill in one pass over K.

    Returns ``(kc, cu_c, kc2, cu_c2)``, bit for bit what :func:`compress_keys`
    gives for the two geometries (minicpm.py:2785-2792).
    """
    dev = _require_cuda(k, cu_seqlens_k)
    if k.ndim != 3:
        raise ValueError("k must be [total_k, num_kv_heads, head_dim]")
    kb = _bf16(k)
    cu = _i32(cu_seqlens_k)
    lens = list(lengths) if lengths is not None else host_lengths(cu)
    total_c = sum(atom_count(n, 32, 16) for n in lens)
    total_c2 = sum(atom_count(n, 128, 64) for n in lens)
    g, d = k.shape[1], k.shape[2]
    kc = torch.empty(total_c, g, d, dtype=torch.bfloat16, device=dev)
    kc2 = torch.empty(total_c2, g, d, dtype=torch.bfloat16, device=dev)
    cu_c, cu_c2 = torch.empty_like(cu), torch.empty_like(cu)
    _call(dev, "ls_compress_keys_dual", kb.data_ptr(), cu.data_ptr(), cu.numel() - 1,
          max(lens, default=0), kb.shape[0], g, d, _ptr(kc) if total_c else None,
          cu_c.data_ptr(), total_c, _ptr(kc2) if total_c2 else None, cu_c2.data_ptr(), total_c2,
          status_word(dev).data_ptr(), _stream(dev))
    return kc, cu_c, kc2, cu_c2


# ---------------------------------------------------------------------------
# a3/a4: projections
# ---------------------------------------------------------------------------

def project_atom_keys(kc: torch.Tensor, wk_t: torch.Tensor) -> torch.Tensor:
    """``project_atom_keys`` (selector.py:179-190): ``[A, G, D] -> [G, A, F]`` bf16."""
    dev = _require_cuda(kc, wk_t)
    kcb = _bf16(kc)
    A, G, D = kcb.shape
    F = wk_t.shape[1]
    ks = torch.empty(G, A, F, dtype=torch.bfloat16, device=dev)
    if A:
        _call(dev, "ls_project_atom_keys", kcb.data_ptr(), A, G, D, wk_t.data_ptr(), F,
                   ks.data_ptr(), _stream(dev))
    return ks


def project_queries(q: torch.Tensor, wq_t: torch.Tensor, num_kv_heads: int) -> torch.Tensor:
    """``project_queries`` (selector.py:160-177): ``[N, H, D] -> [G, N, F]`` bf16."""
    dev = _require_cuda(q, wq_t)
    qb = _bf16(q)
    N, H, D = qb.shape
    F = wq_t.shape[1]
    qs = torch.empty(num_kv_heads, N, F, dtype=torch.bfloat16, device=dev)
    if N:
        _call(dev, "ls_project_queries", qb.data_ptr(), N, H, num_kv_heads, D, wq_t.data_ptr(),
                   F, qs.data_ptr(), status_word(dev).data_ptr(), _stream(dev))
    return qs


# ---------------------------------------------------------------------------
# a5-a7: scoring and selection
# ---------------------------------------------------------------------------

def score_pages(q: torch.Tensor, weights: FoldedWeights, ks: torch.Tensor,
                cu_seqlens_q: torch.Tensor, cu_seqlens_c: torch.Tensor, max_seqlen_q: int,
                *, block_size: int = 64, kernel_stride: int = 16) -> torch.Tensor:
    """Pooled page scores ``[G, total_q, ceil(max_seqlen_q/64)]`` (no causal mask).

    Stored as fp32; every value is a bf16 number, because the atom scores are
    rounded to bf16 as the reference's bf16 einsum rounds them
    (selector.py:203-207).  These are the scores :func:`select_pages` ranks.
    """
    dev = _require_cuda(q, ks, cu_seqlens_q, cu_seqlens_c)
    qb = _bf16(q)
    total_q = qb.shape[0]
    G = weights.num_kv_heads
    total_c = ks.shape[1]
    pages = (int(max_seqlen_q) + block_size - 1) // block_size
    out = torch.empty(G, total_q, pages, dtype=torch.float32, device=dev)
    cu_q, cu_c = _i32(cu_seqlens_q), _i32(cu_seqlens_c)
    _call(dev, "ls_score_pages", qb.data_ptr(), weights.wq_t.data_ptr(),
               _ptr(ks) if total_c else None, cu_q.data_ptr(), cu_c.data_ptr(),
               cu_q.numel() - 1, int(max_seqlen_q), total_q, total_c, weights.num_heads, G,
               weights.head_dim, weights.width, block_size, kernel_stride, out.data_ptr(),
               status_word(dev).data_ptr(), _stream(dev))
    return out


def score_pages_single(q: torch.Tensor, weights: FoldedWeights, ks: torch.Tensor, seq_len: int,
                       *, block_size: int = 64, kernel_stride: int = 16) -> torch.Tensor:
    """Page scores ``[G, N, ceil(seq_len/64)]`` of query rows against one sequence's atoms.

    The reference's ``score_pages`` with its own ``seq_len`` (selector.py:192-214):
    the page count follows ``seq_len``, not the number of query rows.
    """
    dev = _require_cuda(q, ks)
    qb = _bf16(q)
    total_q = qb.shape[0]
    G = weights.num_kv_heads
    total_c = ks.shape[1]
    pages = (int(seq_len) + block_size - 1) // block_size
    out = torch.empty(G, total_q, pages, dtype=torch.float32, device=dev)
    if total_q == 0 or pages == 0:
        return out
    _call(dev, "ls_score_pages_single", qb.data_ptr(), weights.wq_t.data_ptr(),
          _ptr(ks) if total_c else None, total_q, total_c, int(seq_len), weights.num_heads, G,
          weights.head_dim, weights.width, block_size, kernel_stride, out.data_ptr(),
          status_word(dev).data_ptr(), _stream(dev))
    return out


def atom_scores(q: torch.Tensor, weights: FoldedWeights, ks: torch.Tensor,
                cu_seqlens_q: torch.Tensor, cu_seqlens_c: torch.Tensor, max_seqlen_q: int,
                max_atoms: int) -> torch.Tensor:
    """Raw atom scores ``[G, total_q, max_atoms]`` bf16 (-inf past each sequence's atoms)."""
    dev = _require_cuda(q, ks, cu_seqlens_q, cu_seqlens_c)
    qb = _bf16(q)
    total_q = qb.shape[0]
    G = weights.num_kv_heads
    total_c = ks.shape[1]
    out = torch.empty(G, total_q, int(max_atoms), dtype=torch.bfloat16, device=dev)
    if total_q == 0 or max_atoms == 0:
        return out
    cu_q, cu_c = _i32(cu_seqlens_q), _i32(cu_seqlens_c)
    _call(dev, "ls_atom_scores", qb.data_ptr(), weights.wq_t.data_ptr(),
               _ptr(ks) if total_c else None, cu_q.data_ptr(), cu_c.data_ptr(),
               cu_q.numel() - 1, int(max_seqlen_q), total_q, total_c, weights.num_heads, G,
               weights.head_dim, weights.width, int(max_atoms), out.data_ptr(),
               status_word(dev).data_ptr(), _stream(dev))
    return out


def select_pages(q: torch.Tensor, weights: FoldedWeights, ks: torch.Tensor,
                 cu_seqlens_q: torch.Tensor, cu_seqlens_c: torch.Tensor, max_seqlen_q: int, *,
                 take: int, init_blocks: int = 1, local_blocks: int = 2, block_size: int = 64,
                 kernel_stride: int = 16) -> torch.Tensor:
    """Fused score + pool + forced + top-T: ``topk_idx [G, total_q, take]`` int32."""
    dev = _require_cuda(q, ks, cu_seqlens_q, cu_seqlens_c)
    qb = _bf16(q)
    total_q = qb.shape[0]
    G = weights.num_kv_heads
    total_c = ks.shape[1]
    if take > LS_MAX_TOPK:
        raise ValueError(f"take={take} exceeds LS_MAX_TOPK={LS_MAX_TOPK}")
    idx = torch.empty(G, total_q, take, dtype=torch.int32, device=dev)
    if take == 0 or total_q == 0:
        return idx
    cu_q, cu_c = _i32(cu_seqlens_q), _i32(cu_seqlens_c)
    ws = _workspace(dev, total_q, G, int(max_seqlen_q))
    _call(dev, "ls_select_pages", qb.data_ptr(), weights.wq_t.data_ptr(),
               _ptr(ks) if total_c else None, cu_q.data_ptr(), cu_c.data_ptr(),
               cu_q.numel() - 1, int(max_seqlen_q), total_q, total_c, weights.num_heads, G,
               weights.head_dim, weights.width, int(take), int(init_blocks), int(local_blocks),
               block_size, kernel_stride, idx.data_ptr(), ws.data_ptr(), ws.numel(),
               status_word(dev).data_ptr(), _stream(dev))
    return idx


def select_pages_f32(q: torch.Tensor, q_fused: torch.Tensor, kc: torch.Tensor,
                     kv_fused: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_c: torch.Tensor, max_seqlen_q: int, *, take: int,
                     init_blocks: int = 1, local_blocks: int = 2, block_size: int = 64,
                     kernel_stride: int = 16) -> torch.Tensor:
    """Selection of fp32 inputs in fp32 (the reference's fp32 einsums): ``[G, total_q, take]``.

    ``q_fused [H, D, F]`` / ``kv_fused [G, D, F]`` are the fp32 folded
    weights (``fused_weights()``), ``kc [total_c, G, D]`` the fp32 atoms.
    """
    dev = _require_cuda(q, q_fused, kc, kv_fused, cu_seqlens_q, cu_seqlens_c)
    qf = q.float().contiguous()
    kcf = kc.float().contiguous()
    wq, wk = q_fused.float().contiguous(), kv_fused.float().contiguous()
    total_q, H, D = qf.shape
    total_c, G = kcf.shape[0], kcf.shape[1]
    if take > LS_MAX_TOPK:
        raise ValueError(f"take={take} exceeds LS_MAX_TOPK={LS_MAX_TOPK}")
    idx = torch.empty(G, total_q, take, dtype=torch.int32, device=dev)
    if take == 0 or total_q == 0:
        return idx
    cu_q, cu_c = _i32(cu_seqlens_q), _i32(cu_seqlens_c)
    nbytes = _native.load().ls_select_pages_f32_workspace_bytes(total_q, total_c, G,
                                                                int(max_seqlen_q))
    ws = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)
    _call(dev, "ls_select_pages_f32", qf.data_ptr(), wq.data_ptr(),
          kcf.data_ptr() if total_c else None, wk.data_ptr(), cu_q.data_ptr(), cu_c.data_ptr(),
          cu_q.numel() - 1, int(max_seqlen_q), total_q, total_c, H, G, D, wq.shape[-1], int(take),
          int(init_blocks), int(local_blocks), block_size, kernel_stride, idx.data_ptr(),
          ws.data_ptr(), ws.numel(), status_word(dev).data_ptr(), _stream(dev))
    return idx


def uniform_select_pages(q: torch.Tensor, kc: torch.Tensor, cu_seqlens_q: torch.Tensor,
                         cu_seqlens_c: torch.Tensor, max_seqlen_q: int, *, take: int,
                         init_blocks: int = 1, local_blocks: int = 2, block_size: int = 64,
                         kernel_stride: int = 16,
                         softmax_scale: float | None = None) -> torch.Tensor:
    """Uniform-method selection (ops/uniform.py:185-320): ``[G, total_q, take]`` int32.

    ``kc [total_c, G, D]`` are the compressed keys themselves.
    """
    dev = _require_cuda(q, kc, cu_seqlens_q, cu_seqlens_c)
    qb, kcb = _bf16(q), _bf16(kc)
    total_q, H, D = qb.shape
    total_c, G = kcb.shape[0], kcb.shape[1]
    if take > LS_MAX_TOPK:
        raise ValueError(f"take={take} exceeds LS_MAX_TOPK={LS_MAX_TOPK}")
    idx = torch.empty(G, total_q, take, dtype=torch.int32, device=dev)
    if take == 0 or total_q == 0:
        return idx
    cu_q, cu_c = _i32(cu_seqlens_q), _i32(cu_seqlens_c)
    nbytes = _native.load().ls_uniform_select_workspace_bytes(total_q, total_c, H, G,
                                                              int(max_seqlen_q))
    ws = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)
    _call(dev, "ls_uniform_select_pages", qb.data_ptr(), kcb.data_ptr() if total_c else None,
               cu_q.data_ptr(), cu_c.data_ptr(), cu_q.numel() - 1, int(max_seqlen_q), total_q,
               total_c, H, G, D, int(take), int(init_blocks), int(local_blocks), block_size,
               kernel_stride, float(softmax_scale or 0.0), idx.data_ptr(), ws.data_ptr(),
               ws.numel(), status_word(dev).data_ptr(), _stream(dev))
    return idx


def _workspace(dev: torch.device, rows: int, groups: int, seq_len: int) -> torch.Tensor:
    """Scratch for the selection kernels, from PyTorch's caching allocator."""
    nbytes = _native.load().ls_select_pages_workspace_bytes(rows, groups, seq_len)
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)


def select_pages_chunk(q: torch.Tensor, weights: FoldedWeights, ks: torch.Tensor, *,
                       q_position: int, seq_len: int, take: int, init_blocks: int = 1,
                       local_blocks: int = 2, block_size: int = 64,
                       kernel_stride: int = 16) -> torch.Tensor:
    """Selection for query rows at ``[q_position, q_position + len(q))`` of one sequence.

    ``ks [G, A, F]`` holds the atoms of the whole sequence (sequence-parallel
    prefill: each rank selects for its own query chunks).
    """
    dev = _require_cuda(q, ks)
    qb = _bf16(q)
    n = qb.shape[0]
    G = weights.num_kv_heads
    total_c = ks.shape[1]
    if take > LS_MAX_TOPK:
        raise ValueError(f"take={take} exceeds LS_MAX_TOPK={LS_MAX_TOPK}")
    idx = torch.empty(G, n, take, dtype=torch.int32, device=dev)
    if take == 0 or n == 0:
        return idx
    ws = _workspace(dev, n, G, int(seq_len))
    _call(dev, "ls_select_pages_chunk", qb.data_ptr(), weights.wq_t.data_ptr(),
               _ptr(ks) if total_c else None, n, int(q_position), int(seq_len), total_c,
               weights.num_heads, G, weights.head_dim, weights.width, int(take),
               int(init_blocks), int(local_blocks), block_size, kernel_stride, idx.data_ptr(),
               ws.data_ptr(), ws.numel(), status_word(dev).data_ptr(), _stream(dev))
    return idx


# ---------------------------------------------------------------------------
# a9: sparse attention
# ---------------------------------------------------------------------------

def attn_splits(rows: int, max_seqlen_q: int, max_seqlen_k: int, topk: int,
                device: torch.device) -> int:
    """Page-list slices per row for :func:`sparse_attn` (1 = one CTA per row).

    Only decode-shaped calls (one query per sequence) are split: with fewer
    (token, group) rows than SMs, one CTA per row leaves SMs idle, so each
    row's pages are cut into slices of at least 4 pages, up to about one CTA
    per SM (more slices cost more in per-CTA set-up than they gain: measured
    on 128K-token caches, batch 64 runs 70 us unsplit and 79 us in 3 slices).
    Prefill keeps one CTA per row, so its results do not depend on how the
    rows are batched.
    """
    if max_seqlen_q != 1 or rows <= 0:
        return 1
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    pages = min(topk, -(-max(max_seqlen_k, 0) // 64))
    want = sms // rows
    return max(1, min(want, pages // 4, LS_MAX_ATTN_SPLITS))


def sparse_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                topk_idx: torch.Tensor, *, softmax_scale: float | None = None,
                causal: bool = True, return_lse: bool = False, block_size: int = 64,
                out: torch.Tensor | None = None, splits: int | None = None):
    """Block-sparse attention over per-token page lists (minicpm.py:3229-3243).

    ``splits`` cuts each row's page list into that many slices, one CTA each,
    combined by a second kernel (``ls_sparse_attn_split``); ``None`` picks
    it with :func:`attn_splits` (decode calls only).
    """
    dev = _require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, topk_idx)
    qb, kb, vb = _bf16(q), _bf16(k), _bf16(v)
    total_q, H, D = qb.shape
    total_k, G, _ = kb.shape
    idx = _i32(topk_idx)
    if idx.ndim != 3 or idx.shape[0] != G or idx.shape[1] != total_q:
        raise ValueError("topk_idx must be [num_kv_heads, total_q, T]")
    if out is None:
        out = torch.empty(total_q, H, D, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(H, total_q, dtype=torch.float32, device=dev) if return_lse else None
    cu_q, cu_k = _i32(cu_seqlens_q), _i32(cu_seqlens_k)
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    if splits is None:
        splits = attn_splits(total_q * G, int(max_seqlen_q), int(max_seqlen_k), idx.shape[2], dev)
    if splits > 1 and total_q:
        nbytes = _native.load().ls_sparse_attn_split_workspace_bytes(total_q, H, int(splits))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _call(dev, "ls_sparse_attn_split", qb.data_ptr(), kb.data_ptr(), vb.data_ptr(),
              cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, int(max_seqlen_q),
              int(max_seqlen_k), total_q, total_k, H, G, D, idx.data_ptr(), idx.shape[2],
              block_size, scale, 1 if causal else 0, int(splits), ws.data_ptr(), nbytes,
              out.data_ptr(), _ptr(lse), status_word(dev).data_ptr(), _stream(dev))
    else:
        _call(dev, "ls_sparse_attn", qb.data_ptr(), kb.data_ptr(), vb.data_ptr(),
              cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, int(max_seqlen_q),
              int(max_seqlen_k), total_q, total_k, H, G, D, idx.data_ptr(), idx.shape[2],
              block_size, scale, 1 if causal else 0, out.data_ptr(), _ptr(lse),
              status_word(dev).data_ptr(), _stream(dev))
    if q.dtype != torch.bfloat16:
        out = out.to(q.dtype)
    return (out, lse) if return_lse else out


def sparse_attn_gather_only(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                            max_seqlen_q: int, max_seqlen_k: int, topk_idx: torch.Tensor, *,
                            causal: bool = True, block_size: int = 64) -> None:
    """The data movement of :func:`sparse_attn` alone (measured gather roofline).

    Same launch geometry, page lists and TMA ring; no math, no output.  Its
    duration is the L2 -> shared-memory gather time of that attention call.
    """
    dev = _require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, topk_idx)
    qb, kb, vb = _bf16(q), _bf16(k), _bf16(v)
    total_q, H, D = qb.shape
    total_k, G, _ = kb.shape
    idx = _i32(topk_idx)
    if idx.ndim != 3 or idx.shape[0] != G or idx.shape[1] != total_q:
        raise ValueError("topk_idx must be [num_kv_heads, total_q, T]")
    cu_q, cu_k = _i32(cu_seqlens_q), _i32(cu_seqlens_k)
    _call(dev, "ls_sparse_attn_gather_only", qb.data_ptr(), kb.data_ptr(), vb.data_ptr(),
               cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, int(max_seqlen_q),
               int(max_seqlen_k), total_q, total_k, H, G, D, idx.data_ptr(), idx.shape[2],
               block_size, 1 if causal else 0, status_word(dev).data_ptr(), _stream(dev))


# ---------------------------------------------------------------------------
# the 8-bit paged key/value cache
# ---------------------------------------------------------------------------

@dataclass
class PagePlan:
    """One step of a batch over the paged cache (:func:`plan_pages`)."""

    context_lens: torch.Tensor   # [B] int32, tokens cached before the step
    seq_lens: torch.Tensor       # [B] int32, with the step's tokens
    cu_seqlens_q: torch.Tensor   # [B+1] int32, the step's packed rows
    cu_blocks: torch.Tensor      # [B+1] int32, pages each request writes
    slots: torch.Tensor          # [total_new] int64, page * 64 + offset (-1: no page)
    positions: torch.Tensor      # [total_new] int64
    free_head: torch.Tensor | None = None  # [1] int32, the free list after the step


def _exact_tensor(t: torch.Tensor, name: str, dtype: torch.dtype, shape) -> None:
    """A tensor the kernels use in place: its own type and layout, no copies."""
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def plan_pages(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
               free_pages: torch.Tensor, free_head: torch.Tensor, total_new: int) -> PagePlan:
    """Pages, slots and positions of one step, on the GPU (``ls_plan_pages``).

    Request ``b`` holds ``context_lens[b]`` tokens and adds ``new_lens[b]``.
    Blocks that begin in this step take the next entries of ``free_pages``
    behind ``free_head [1]``; ``block_table [B, max_blocks]`` is updated in
    place.  ``total_new`` is the packed row count the caller knows (rows behind
    the last request get slot -1).  The next step passes ``plan.seq_lens`` and
    ``plan.free_head`` on; nothing here reads the device back.
    """
    if context_lens.is_cuda:
        got = _native.binding().plan_pages(context_lens, new_lens, block_table, free_pages,
                                           free_head, int(total_new),
                                           status_word(context_lens.device))
        if got is not None:
            _native.raise_for("ls_plan_pages", got[0])
            return PagePlan(context_lens, *got[1:])
    dev = _require_cuda(context_lens, new_lens, block_table, free_pages, free_head)
    ctx, new = _i32(context_lens), _i32(new_lens)
    if ctx.ndim != 1 or new.shape != ctx.shape or ctx.numel() == 0:
        raise ValueError("context_lens and new_lens must be vectors of the same batch")
    batch = ctx.numel()
    if block_table.ndim != 2 or block_table.shape[0] != batch or block_table.shape[1] == 0:
        raise ValueError("block_table must be [batch, max_blocks]")
    _exact_tensor(block_table, "block_table", torch.int32, block_table.shape)
    free, head = _i32(free_pages), _i32(free_head)
    if free.ndim != 1 or head.numel() != 1:
        raise ValueError("free_pages must be a vector and free_head one number")
    total_new = int(total_new)
    if not 0 <= total_new < 1 << 31:
        raise ValueError("total_new must lie in [0, 2^31)")
    # The five int32 results share one allocation.
    ints = torch.empty(3 * batch + 3, dtype=torch.int32, device=dev)
    seq, cu_q, cu_blocks, head_out = ints.split([batch, batch + 1, batch + 1, 1])
    slots, positions = torch.empty(2, total_new, dtype=torch.int64, device=dev).unbind(0)
    _call(dev, "ls_plan_pages", ctx.data_ptr(), new.data_ptr(), batch, block_table.data_ptr(),
          block_table.shape[1], _ptr(free) if free.numel() else None, free.numel(),
          head.data_ptr(), total_new, seq.data_ptr(), cu_q.data_ptr(), cu_blocks.data_ptr(),
          _ptr(slots) if total_new else None, _ptr(positions) if total_new else None,
          head_out.data_ptr(), status_word(dev).data_ptr(), _stream(dev))
    return PagePlan(ctx, seq, cu_q, cu_blocks, slots, positions, head_out)


def _check_cache(k_pages, v_pages, k_scale, v_scale):
    """The cache's tensors, used in place: ``[num_pages, G, 64, 128]`` e4m3, ``[num_pages, G]``."""
    if k_pages.ndim != 4 or k_pages.shape[2] != _native.LS_PAGE_TOKENS:
        raise ValueError("k_pages must be [num_pages, num_kv_heads, 64, head_dim]")
    _exact_tensor(k_pages, "k_pages", torch.float8_e4m3fn, k_pages.shape)
    _exact_tensor(v_pages, "v_pages", torch.float8_e4m3fn, k_pages.shape)
    _exact_tensor(k_scale, "k_scale", torch.float32, k_pages.shape[:2])
    _exact_tensor(v_scale, "v_scale", torch.float32, k_pages.shape[:2])
    return k_pages.shape[0], k_pages.shape[1], k_pages.shape[3]


def _token_rows(t: torch.Tensor) -> torch.Tensor:
    """bf16 ``[N, G, D]`` whose heads are contiguous and tokens 16-byte aligned (a
    view into a fused projection passes as it is)."""
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    if (t.stride(2) == 1 and t.stride(1) == t.shape[2] and t.stride(0) % 8 == 0
            and t.stride(0) >= t.shape[1] * t.shape[2] and t.data_ptr() % 16 == 0):
        return t
    # Not contiguous(): it returns a single token with any stride, and any alignment, as it is.
    return t.clone(memory_format=torch.contiguous_format)


def append_kv(k: torch.Tensor, v: torch.Tensor, plan: PagePlan, k_pages: torch.Tensor,
              v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Round a step's ``k``, ``v`` ``[total_new, G, 128]`` into the 8-bit cache (``ls_append_kv``).

    ``k_pages``/``v_pages [num_pages, G, 64, 128]`` (e4m3) and
    ``k_scale``/``v_scale [num_pages, G]`` (fp32, powers of two) are updated in
    place.  A (page, head) scale covers the page's largest value and only
    grows while the page fills; older codes are rescaled with it.
    """
    if k.is_cuda:
        rc = _native.binding().append_kv(k, v, plan.context_lens, plan.seq_lens,
                                         plan.cu_seqlens_q, plan.cu_blocks, plan.slots, k_pages,
                                         v_pages, k_scale, v_scale, status_word(k.device))
        if rc is not None:
            _native.raise_for("ls_append_kv", rc)
            return
    dev = _require_cuda(k, v, plan.context_lens, plan.seq_lens, plan.cu_seqlens_q, plan.cu_blocks,
                        plan.slots, k_pages, v_pages, k_scale, v_scale)
    num_pages, G, D = _check_cache(k_pages, v_pages, k_scale, v_scale)
    if k.ndim != 3 or tuple(k.shape[1:]) != (G, D) or v.shape != k.shape:
        raise ValueError("k and v must be [total_new, num_kv_heads, head_dim] of the cache")
    n, batch = k.shape[0], plan.context_lens.numel()
    _exact_tensor(plan.context_lens, "plan.context_lens", torch.int32, (batch,))
    _exact_tensor(plan.seq_lens, "plan.seq_lens", torch.int32, (batch,))
    _exact_tensor(plan.cu_seqlens_q, "plan.cu_seqlens_q", torch.int32, (batch + 1,))
    _exact_tensor(plan.cu_blocks, "plan.cu_blocks", torch.int32, (batch + 1,))
    _exact_tensor(plan.slots, "plan.slots", torch.int64, (n,))
    if n == 0:
        return
    kb, vb = _token_rows(k), _token_rows(v)
    _call(dev, "ls_append_kv", kb.data_ptr(), vb.data_ptr(), kb.stride(0), vb.stride(0), n, batch,
          G, D, plan.context_lens.data_ptr(), plan.seq_lens.data_ptr(),
          plan.cu_seqlens_q.data_ptr(), plan.cu_blocks.data_ptr(), plan.slots.data_ptr(),
          k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
          num_pages, status_word(dev).data_ptr(), _stream(dev))


def paged_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
               seq_lens: torch.Tensor, cu_seqlens_q: torch.Tensor, max_seqlen_q: int,
               max_seqlen_k: int, *, topk_idx: torch.Tensor | None = None,
               softmax_scale: float | None = None, causal: bool = True,
               return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention over the 8-bit paged cache (``ls_paged_attn``).

    The counterpart of :func:`sparse_attn` for decode steps, drafts of a few
    tokens and page-listed chunks: query row ``i`` of request ``b`` stands at
    position ``seq_lens[b] - nq + i`` (its own keys are already cached).
    ``topk_idx [G, total_q, T]`` lists each row's pages as the selection writes
    them; ``None`` attends to every page.  Rows behind the last request are left
    as they were in ``out``.
    """
    if q.is_cuda:
        got = _native.binding().paged_attn(
            q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q,
            int(max_seqlen_q), int(max_seqlen_k), topk_idx, softmax_scale or 0.0, bool(causal),
            bool(return_lse), out, status_word(q.device))
        if got is not None:
            _native.raise_for("ls_paged_attn", got[0])
            return got[1:] if return_lse else got[1]
    dev = _require_cuda(q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens,
                        cu_seqlens_q, topk_idx)
    num_pages, G, D = _check_cache(k_pages, v_pages, k_scale, v_scale)
    if q.ndim != 3 or q.shape[2] != D or q.shape[1] % G:
        raise ValueError("q must be [total_q, num_heads, head_dim], num_heads a multiple of the "
                         "cache's heads")
    qb = _bf16(q)
    total_q, H, _ = qb.shape
    table, seq, cu_q = _i32(block_table), _i32(seq_lens), _i32(cu_seqlens_q)
    batch = seq.numel()
    if seq.ndim != 1 or cu_q.shape != (batch + 1,) or table.ndim != 2 or table.shape[0] != batch:
        raise ValueError("block_table [B, max_blocks], seq_lens [B] and cu_seqlens_q [B+1] must "
                         "agree on the batch")
    topk, idx = 0, None
    if topk_idx is not None:
        idx = _i32(topk_idx)
        if idx.ndim != 3 or idx.shape[0] != G or idx.shape[1] != total_q or idx.shape[2] == 0:
            raise ValueError("topk_idx must be [num_kv_heads, total_q, T] with T > 0")
        topk = idx.shape[2]
    direct = out if out is not None and q.dtype == torch.bfloat16 else None
    if out is not None:
        _exact_tensor(out, "out", q.dtype, q.shape)
        if out.device != dev:
            raise ValueError("all tensors must be on the same CUDA device")
    if direct is None:
        direct = torch.empty(total_q, H, D, dtype=torch.bfloat16, device=dev)
        if out is not None:
            direct.copy_(out)  # rows behind the last request keep their values
    lse = torch.empty(H, total_q, dtype=torch.float32, device=dev) if return_lse else None
    scale = float(softmax_scale or 0.0)  # 0 selects D^-0.5
    nbytes = _native.load().ls_paged_attn_workspace_bytes()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, "ls_paged_attn", qb.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
          k_scale.data_ptr(), v_scale.data_ptr(), num_pages, table.data_ptr(), table.shape[1],
          seq.data_ptr(), cu_q.data_ptr(), batch, int(max_seqlen_q), int(max_seqlen_k), total_q, H,
          G, D, _ptr(idx), topk, scale, 1 if causal else 0, ws.data_ptr(), nbytes,
          direct.data_ptr(), _ptr(lse), status_word(dev).data_ptr(), _stream(dev))
    if out is None:
        out = direct if q.dtype == torch.bfloat16 else direct.to(q.dtype)
    elif direct is not out:
        out.copy_(direct)
    return (out, lse) if return_lse else out
