"""Plain 64-bit forms of the quantised-cache operators, for the tests."""
import math

import torch

QMAX = {"fp8": 448.0, "int8": 127.0, "int4": 7.0}
KV_DTYPE = {"fp8": 1, "int8": 2, "int4": 3}


def quantise(x, kind):
    """(codes as float64, scales as float32) of rows x [..., dim]."""
    x = x.double()
    amax = x.abs().amax(-1)
    odd = ~torch.isfinite(amax)
    fine = (amax >= 2.0 ** -100) & ~odd
    safe = torch.where(fine, amax, torch.ones_like(amax))
    scale = torch.where(fine, safe / torch.full_like(safe, QMAX[kind]), torch.zeros_like(safe)).float()
    inv = torch.where(fine, torch.full_like(safe, QMAX[kind]) / safe, torch.zeros_like(safe)).float()
    y = torch.where(odd.unsqueeze(-1), 0.0, x) * inv.double().unsqueeze(-1)
    if kind == "fp8":
        step = torch.exp2(torch.clamp(torch.frexp(y)[1].double() - 1, min=-6) - 3)
        codes = torch.round(y / step) * step
    else:
        codes = torch.round(y)
    return codes, torch.where(odd, math.nan, scale)


def pack(codes, kind):
    if kind == "fp8":
        return codes.float().to(torch.float8_e4m3fn)
    c = codes.to(torch.int8)
    if kind == "int8":
        return c.contiguous()
    return ((c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)).contiguous().view(torch.uint8)


def unpack(cache, kind):
    if kind != "int4":
        return cache.double()
    lo, hi = (cache << 4).view(torch.int8) >> 4, cache.view(torch.int8) >> 4
    return torch.stack((lo, hi), -1).flatten(-2).double()


def attend(q, ks, vs, alibi=False, softmax_scale=None):
    """One sequence: q [head_q, dim], ks / vs [n, head_k, dim] in 64 bits -> o, lse, and what bounds the error:
    (sum_j p_j |v_j| per element, the largest sum_d |q_d k_d| * scale of a head, the largest |v|)."""
    hq, dim = q.shape
    n, hk = ks.shape[0], ks.shape[1]
    o = torch.zeros(hq, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((hq,), -math.inf, dtype=torch.float64, device=q.device)
    spread, scores, top = torch.zeros_like(o), torch.zeros_like(lse), 0.0
    if n == 0:
        return o, lse, spread, scores, top
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(dim)
    group = hq // hk
    k = ks.repeat_interleave(group, 1).double()
    v = vs.repeat_interleave(group, 1).double()
    qd = q.double()
    s = torch.einsum("hd,nhd->hn", qd, k) * scale
    scores = (torch.einsum("hd,nhd->hn", qd.abs(), k.abs()) * scale).amax(1)
    if alibi:
        slope = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=q.device, dtype=torch.float64) / hq)
        s = s + slope[:, None] * (torch.arange(n, device=q.device, dtype=torch.float64) - (n - 1))
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    return torch.einsum("hn,nhd->hd", p, v), lse, torch.einsum("hn,nhd->hd", p, v.abs()), scores, v.abs().max().item()


def bounds(o, lse, spread, scores, top, n, weight_bits, out_dtype):
    """Tolerances of o and lse.  Softmax weights rounded to `weight_bits` bits: half a step, 2^-weight_bits relative, or
    2^-25 of the largest weight where fp16 runs into its subnormals, 2^-23 of it where weights are fixed-point numbers of
    22 bits behind the largest one (n of them at worst; the largest weight times its largest code is at most `top`).  Scores: a chain of fp32
    accumulations, 2^-19 of the sum of magnitudes, which moves every weight and the sum alike; exp2 and the
    sums: 2^-19.  Output: half a step of its type."""
    drift = 2.0 ** -19 * (1.0 + scores)
    tol_o = spread * (2.0 ** -weight_bits + 2 * drift[:, None]) + n * 2.0 ** -23 * top
    tol_o = tol_o + (o.abs() + tol_o) * torch.finfo(out_dtype).eps / 2 + 2.0 ** -25
    return tol_o, drift + 2.0 ** -21 * torch.nan_to_num(lse.abs(), posinf=0.0)
