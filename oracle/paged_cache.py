"""The 8-bit paged cache in plain 64-bit torch on the CPU: planning, cache write, attention.

Written from the definitions in ``include/leanselect_b200.h``, one request,
page and row at a time.  ``attend`` also returns what a tolerance needs: the
softmax-weighted sum of |v|, the largest sum |q||k| of a row, and the largest
weight times value scale of a row multiplied with its sum of |value codes|.
"""
from __future__ import annotations

import math

import torch

PAGE = 64
E_MIN, E_MAX = -40, 48


def plan(context, new, table, free, head, total_new):
    """Lists in, dict of lists out; ``table`` (list of lists) is updated."""
    out = dict(seq=[], cu_q=[0], cu_blocks=[0], slots=[], positions=[])
    for b, (c, n) in enumerate(zip(context, new)):
        for p in range(c, c + n):
            j = p // PAGE
            if p % PAGE == 0:
                table[b][j] = free[head] if head < len(free) else -1
                head += 1
            page = table[b][j]
            out["slots"].append(page * PAGE + p % PAGE if page >= 0 else -1)
            out["positions"].append(p)
        out["seq"].append(c + n)
        out["cu_q"].append(out["cu_q"][-1] + n)
        out["cu_blocks"].append(out["cu_blocks"][-1]
                                + (-(-(c + n) // PAGE) - c // PAGE if n else 0))
    pad = total_new - len(out["slots"])
    out["slots"] += [-1] * pad
    out["positions"] += [0] * pad
    out["head"] = min(head, len(free))
    return out


def scale_exponent(amax: float) -> int:
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even, saturating; NaN stays NaN.  float64 in and out."""
    mag = x.abs().clamp(max=448.0)
    _, e = torch.frexp(mag)                    # mag in [2^(e-1), 2^e)
    step = torch.exp2((e - 4).clamp(min=-9).double())  # 4 significant bits, subnormals of 2^-9
    return torch.copysign((torch.round(mag / step) * step).clamp(max=448.0), x)


def append(x, context, new, table, codes, scale):
    """Writes packed rows ``x [N, G, D]`` into ``codes`` (values, float64) and ``scale``."""
    t = 0
    for b, (c, n) in enumerate(zip(context, new)):
        p = c
        while p < c + n:
            j, r0 = p // PAGE, p % PAGE
            rows = min(PAGE - r0, c + n - p)
            page = table[b][j]
            if page >= 0:
                for g in range(codes.shape[1]):
                    block = x[t:t + rows, g].double()
                    finite = block[~block.isnan()]
                    s = 2.0 ** scale_exponent(float(finite.abs().max()) if finite.numel() else 0.0)
                    if r0 > 0:
                        held = float(scale[page, g])
                        s = min(max(s, held), 2.0 ** E_MAX)
                        codes[page, g, :r0] = e4m3(codes[page, g, :r0] * (held / s))
                    codes[page, g, r0:r0 + rows] = e4m3(block / s)
                    scale[page, g] = s
            p += rows
            t += rows


def attend(q, k_codes, v_codes, k_scale, v_scale, table, seq, cu_q, idx=None, scale=None,
           causal=True, out=None):
    """``(out, lse, (weighted |v|, max sum |q||k| scale, max(w vs) sum |code|))`` in float64.

    Rows outside the requests stay as ``out`` has them.
    """
    N, H, D = q.shape
    G = k_codes.shape[1]
    scale = scale or 1.0 / math.sqrt(D)
    out = torch.zeros(N, H, D, dtype=torch.float64) if out is None else out.double().clone()
    lse = torch.full((H, N), math.inf, dtype=torch.float64)
    mass = torch.zeros(N, H, D, dtype=torch.float64)
    reach = torch.zeros(N, H, dtype=torch.float64)
    grain = torch.zeros(N, H, D, dtype=torch.float64)
    for b in range(len(seq)):
        length, nq = seq[b], cu_q[b + 1] - cu_q[b]
        for i in range(nq):
            t = cu_q[b] + i
            last = length - nq + i if causal else length - 1
            for g in range(G):
                blocks = range(-(-length // PAGE)) if idx is None else sorted(
                    {int(p) for p in idx[g, t] if 0 <= int(p) < -(-length // PAGE)})
                ks, vs, scales = [], [], []
                for j in blocks:
                    page, rows = table[b][j], min(PAGE, last + 1 - j * PAGE, length - j * PAGE)
                    if rows <= 0 or not 0 <= page < k_codes.shape[0]:
                        continue
                    ks.append(k_codes[page, g, :rows].double() * float(k_scale[page, g]))
                    vs.append(v_codes[page, g, :rows].double() * float(v_scale[page, g]))
                    scales.append(torch.full((rows,), float(v_scale[page, g]), dtype=torch.float64))
                heads = slice(g * (H // G), (g + 1) * (H // G))
                out[t, heads] = 0.0
                if not ks:
                    continue
                k, v = torch.cat(ks), torch.cat(vs)
                qr = q[t, heads].double()
                x = qr @ k.T * scale
                w = torch.softmax(x, -1)
                out[t, heads] = w @ v
                mass[t, heads] = w @ v.abs()
                reach[t, heads] = (qr.abs() @ k.abs().T).amax(-1) * scale
                sv = torch.cat(scales)
                grain[t, heads] = (w * sv).amax(-1, keepdim=True) * (v.abs() / sv[:, None]).sum(0)
                lse[heads, t] = torch.logsumexp(x, -1)
    return out, lse, (mass, reach, grain)
