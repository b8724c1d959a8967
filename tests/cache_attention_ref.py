"""64-bit definition of the attentions over a cache, and the error bound their kernels are held to."""
import math

import torch


def reference(q, k, v, *, window=None, sinks=0, lengths=None, scale=None, prefix=None):
    """(out, bound) in fp64, both shaped like q: row by row from the definition, and how far a kernel may be off.

    The bound counts every rounding the kernels are allowed (eps = half a step of the 16-bit type,
    relative): each weight is rounded to the type before the second product, which moves the output by at
    most eps * A with A = sum_j p_j |v_j|; the output is rounded once more, eps * |out|.  A score is an fp32 dot
    product, so it is off by at most (D + 8) * 2^-24 * scale * sum_d |q_d k_d|, which moves a weight and the sum of
    weights by that relative amount each.  Weights are kept relative to a reference that some key attains, so
    the sum is at least 1 in those units, and an f16 weight below 2^-14 is rounded absolutely, by 2^-25
    (bf16 has the exponents of fp32).  fp32 accumulation in steps of 16 keys: (n / 16 + 32) * 2^-22 * A."""
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    eps = torch.finfo(q.dtype).eps / 2
    out = torch.zeros((B, Hq, Sq, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lens = [Skv] * B if lengths is None else [min(max(int(n), 0), Skv) for n in lengths.tolist()]
    for b, L in enumerate(lens):
        pos = torch.arange(L - Sq, L, device=q.device)[:, None]
        key = torch.arange(L, device=q.device)[None, :]
        seen = key <= pos
        if window is not None:
            seen &= (key > pos - window) | (key < sinks)
        if prefix is not None:
            seen = torch.cat([(pos >= 0).expand(Sq, prefix[0].shape[1]), seen], 1)
        for h in range(Hq):
            kk, vv = k[b, h // G, :L].double(), v[b, h // G, :L].double()
            if prefix is not None:
                kk, vv = torch.cat([prefix[0][h // G].double(), kk]), torch.cat([prefix[1][h // G].double(), vv])
            if kk.shape[0] == 0:
                continue
            qq = q[b, h].double()
            s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True).nan_to_num(neginf=0.0)
            w = torch.where(seen, (s - top).exp(), 0.0)
            total = w.sum(1, keepdim=True)
            p = torch.where(total > 0, w / total.clamp_min(1e-300), 0.0)
            out[b, h] = p @ vv
            A = p @ vv.abs()
            score = (D + 8) * 2.0 ** -24 * scale * torch.where(seen, qq.abs() @ kk.abs().T, 0.0).amax(1, keepdim=True)
            n = seen.sum(1, keepdim=True)
            bound[b, h] = eps * (A + out[b, h].abs()) * (1 + 2 * eps) + (2 * score + (n / 16 + 32) * 2.0 ** -22) * A + 1e-30
            if q.dtype == torch.float16:
                # subnormal weights, and outputs below the type's smallest normal
                bound[b, h] += 2.0 ** -25 * (seen.double() @ vv.abs()) + 2.0 ** -25
    return out, bound


def check(got, want, what=""):
    out, bound = want
    assert got.shape == out.shape, (what, got.shape, out.shape)
    off = (got.double() - out).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst {(off / bound).nan_to_num(1e9).max().item():.3f} of it at {bad.nonzero()[0].tolist()}"
