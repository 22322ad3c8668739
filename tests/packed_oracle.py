"""Attention over packed sequences in float64, head by head, with bounds of what bf16 operands and results may be off."""
import math

import torch

BF16 = 2.0 ** -8          # half a step of bf16, relative to the value
FP32 = 2.0 ** -12         # scores, exponentials and sums in fp32: D products of a score, 2^-24 each and up to 8 in size, and what follows


def packed(q, k, v, ends, causal, do=None, scale=None):
    """``{"o": (value, bound), ...}``; with ``do`` also dq, dk, dv.  The bound of an element counts the roundings to bf16 on its way:
    forward the weights and the result; backward also the result inside Delta, the score gradients and the gradients."""
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    T, H, D = q.shape
    G = k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    do = None if do is None else do.double()
    for a, b in zip(ends, ends[1:]):
        for h in range(H if b > a else 0):
            g = h // (H // G)
            Q, K, V = q[a:b, h], k[a:b, g], v[a:b, g]
            S = Q @ K.T * scale
            if causal:
                S = S.masked_fill(torch.ones_like(S).triu(1) > 0, -math.inf)
            P = torch.softmax(S, -1)
            O = P @ V
            o_err = (BF16 + FP32) * (P @ V.abs()) + BF16 * O.abs()
            out["o"][0][a:b, h], out["o"][1][a:b, h] = O, o_err
            if do is None:
                continue
            dO = do[a:b, h]
            dP, Delta = dO @ V.T, (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - Delta)
            dS_err = BF16 * dS.abs() + P * (dO.abs() * o_err).sum(-1, keepdim=True) + FP32 * P * (dO.abs() @ V.abs().T + Delta.abs())
            out["dv"][0][a:b, g] += P.T @ dO
            out["dv"][1][a:b, g] += (BF16 + FP32) * (P.T @ dO.abs())
            out["dk"][0][a:b, g] += scale * dS.T @ Q
            out["dk"][1][a:b, g] += scale * (dS_err.T + FP32 * dS.T.abs()) @ Q.abs()
            out["dq"][0][a:b, h] = scale * dS @ K
            out["dq"][1][a:b, h] = scale * (dS_err + FP32 * dS.abs()) @ K.abs()
    for n in ("dq", "dk", "dv"):
        value, bound = out[n]
        bound += BF16 * (value.abs() + bound)
    return out


def check(got, want, name):
    value, bound = want[name]
    off = (got.double() - value).abs()
    worst = (off / (bound + 1e-30)).max().item() if off.numel() else 0.0
    assert (off <= bound + 1e-30).all(), f"{name}: {worst:.2f} of the bound, at {(off / (bound + 1e-30)).argmax().item()}"
