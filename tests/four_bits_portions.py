"""What portions of prompts over a cache held in four bits are to give, in 64 bits, and how far half-precision kernels may be from it.

An output o = sum_j p_j v_j is moved by
* keys rounded to half precision (2^-11 of each product's magnitude; queries are bfloat16 numbers, which half precision holds) and float32 sums: a score by d_j = 2^-10.9 scale sum_f |q_f k_jf|, and so
  the output by sum_j p_j d_j |v_j - o| (a tenth more for what is not linear);
* weights and values rounded to half precision: 2^-11 sum_j p_j |v_j| each, and weights that are subnormal there (from 2^-14 on where the largest is 2^6 at least): 2^-31 of the largest weight each;
* float32 sums (tensor cores cut off what they add: 2^-23 of the sum, some 2^8 times), exponentials and large scores: 2^-14 sum_j p_j |v_j|;
* its rounding to bfloat16: 2^-8 |o|.
The last rounding is all that shows in the whole: an error evenly spread over +-2^-8 2^e has the mean square 2^-16 / 3 4^e, numbers of that binade 2 4^e or more: 2^-8 / sqrt(6) = 1.6e-3 of the outputs'
norm, where the others give 2e-4 each; 2^-9 is asked for.  (Keys, weights or values in bfloat16 would have 1.6e-3 of their own: 2.3e-3.)"""

import math

import torch

import four_bits as fb
from four_bits import BF16, HALF

NORM = 2.0 ** -9


def want(q, kv, table, spans, nq, nkv, d, page, scale):
    """(outputs, their bounds) in 64 bits of ``spans`` [(new, cached)], [tokens, nq * d]."""
    group, q = nq // nkv, q.double().view(-1, nq, d)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    t0 = 0
    for r, (n, cached) in enumerate(spans):
        total = n + cached
        if n == 0:
            continue
        pages = table[r].long()[:-(-total // page)]
        hidden = torch.arange(total, device=q.device)[None] > torch.arange(cached, total, device=q.device)[:, None]
        for kvh in range(nkv):
            k, v = (lo + s * c for c, s, lo in ([t.reshape(-1, d)[:total] for t in fb.read_rows(kv[pages, kvh, i], page, d, bool(i))] for i in range(2)))
            for h in range(kvh * group, (kvh + 1) * group):
                x = q[t0:t0 + n, h]
                p = torch.softmax((x @ k.T * scale).masked_fill(hidden, -math.inf), -1)
                o = p @ v
                moved = p * (2.0 ** -10.9 * scale * (x.abs() @ k.abs().T))
                size = p @ v.abs()
                # sum_j m_j |v_j - o| <= sum_j m_j |v_j| + |o| sum_j m_j
                bound[t0:t0 + n, h] = 1.1 * (moved @ v.abs() + moved.sum(-1, keepdim=True) * o.abs()) + (2 * 2.0 ** -11 + 2.0 ** -14) * size + HALF[BF16] * o.abs() \
                    + 2.0 ** -31 * p.amax(-1, keepdim=True) * v.abs().sum(0) + 1e-30
                out[t0:t0 + n, h] = o
        t0 += n
    return out.view(-1, nq * d), bound.view(-1, nq * d)


def faults(got, out, bound):
    """What is wrong with outputs, in words; nothing where they are near enough."""
    got, said = got.double(), []
    over = (got - out).abs() - bound
    if not bool((over <= 0).all()):
        said.append(f"{int((~(over <= 0)).sum())} of {over.numel()} beyond their bounds")
    off = float((got - out).norm() / out.norm())
    if not off <= NORM:
        said.append(f"{off:.3g} of the outputs' norm")
    return said
