"""Bounds of decode attention that follow the softmax weights of each head, for the tests.

What the kernels may lose, besides half a step of the output's type, per head and element of o:

* a weight w_j = p_j vs_j is rounded to `bits` bits, half a step, 2^-bits of itself, or to a fixed quantum, half of
  which is at most 2^-28 of the head's largest weight: sum_j min(w_j, 2^-28 max w) |code_j|;
* a probability or a weight below 2^-120 of the largest probability may count as zero (fp32's own numbers end at 2^-126,
  and the references that weights are kept against need some room);
* scores: fp32 chains, 2^-19 of the sum of magnitudes, which moves a weight and the sum of the weights alike;
* sums of n keys in fp32: 16 keys at a time (2^-23 of the running sum where the tensor core cuts the sum off) in one
  place, and 8 lanes that add one weight at a time (2^-24): 2^-27 n each.

Nothing in it grows with the largest |v| of other heads or elements.  `bounds` adds the keys' errors up as if they all
pointed the same way; `random_bounds` is for V rows drawn independently of the scores, where they add up like the steps
of a walk, so that a single tile of V that is left out shows among 40 000 keys."""
import math

import torch

QUANTUM = 2.0 ** -28
TINY = 2.0 ** -120


def attend(q, k_code, k_scale, v_code, v_scale, alibi=False, softmax_scale=None):
    """One sequence in 64 bits.  q [head_q, dim], codes [n, head_k, dim], scales [n, head_k] -> o and lse; of w_j |code_j|
    the sum and the root of the sum of squares; what the quantum takes, at most; the drift of a score [head_q]."""
    hq, dim = q.shape
    group = hq // k_code.shape[1]
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(dim)
    k = (k_code.double() * k_scale.double().unsqueeze(-1)).repeat_interleave(group, 1)
    code = v_code.double().repeat_interleave(group, 1)
    vs = v_scale.double().repeat_interleave(group, 1).T
    s = torch.einsum("hd,nhd->hn", q.double(), k) * scale
    reach = (torch.einsum("hd,nhd->hn", q.double().abs(), k.abs()) * scale).amax(1)
    if alibi:
        slope = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=q.device, dtype=torch.float64) / hq)
        bias = slope[:, None] * (torch.arange(len(k), device=q.device, dtype=torch.float64) - (len(k) - 1))
        s, reach = s + bias, reach + bias.abs().amax(1)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    w = p * vs
    least = torch.minimum(w, QUANTUM * w.amax(1, keepdim=True)) + torch.where(torch.minimum(p, w) < TINY * p.amax(1, keepdim=True), w, 0.0)
    o = torch.einsum("hn,nhd->hd", w, code)
    return dict(o=o, lse=lse, spread=torch.einsum("hn,nhd->hd", w, code.abs()), walk=torch.einsum("hn,nhd->hd", w ** 2, code ** 2).sqrt(),
                least=torch.einsum("hn,nhd->hd", least, code.abs()), drift=2.0 ** -19 * (1.0 + reach))


def rounded(tol, o, out_dtype):
    # (half a step of fp16's subnormal numbers; those of fp32, and so of bf16, become zeros)
    fin = torch.finfo(out_dtype)
    return tol + (o.abs() + tol) * fin.eps / 2 + max(fin.smallest_normal * fin.eps / 2, 2.0 ** -126)


def lse_bound(found, n):
    return found["drift"] + n * 2.0 ** -27 + 2.0 ** -21 * found["lse"].abs()


def bounds(found, n, bits, out_dtype):
    """Tolerances of o and lse."""
    tol = found["spread"] * (2.0 ** -bits + 2 * found["drift"][:, None] + n * 2.0 ** -26) + found["least"]
    return rounded(tol, found["o"], out_dtype), lse_bound(found, n)


def random_bounds(found, n, bits, out_dtype):
    """The same where the signs of V are random: a key's error is at most (2^-bits + 2 drift) w |code| and, being spread
    evenly over that, 0.58 of it on average; five times the walk is eight standard deviations and more.  The running sum
    stays within six walks of its end."""
    walk = found["walk"]
    tol = 5 * walk * (2.0 ** -bits + 2 * found["drift"][:, None]) + n * 2.0 ** -26 * (found["o"].abs() + 6 * walk) + found["least"]
    return rounded(tol, found["o"], out_dtype), lse_bound(found, n)
