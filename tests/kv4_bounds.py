"""The attention over a q4_0 cache in 64 bits with torch, where numpy takes long, and how far f32 outputs may be from it.

Bound of an f32 output, relative to sum p |v| of its channel (e = 2^-24):
  scores   q in two fp16 terms, 2^-22; the product of the two small terms left out, 2^-22; D / 16 tensor-core steps for each of
           three products, cut by 2 e of the running sum of magnitudes, and a few f32 steps: |ds| <= (2^-21 + (6 D / 16 + 16) e) A,
           A = scale * max_c sum |q||k|; where a mask is added, 4 e of the spread of its values besides (its change of base and
           its addition, in f32);
  weights  2 |ds|, 2^-20 for the exponentials, 2^-21 for the two terms and the product left out;
  sums     tensor-core steps that are added up without an ordinary f32 addition between them, cut by 2 e each, and the f32 steps of
           the joins: many rows 4 tiles x 12 products, a total of n / 256 additions; few rows two products for 16 cells of a warp's
           share, a quarter of the cells and a tile's rest.
"""
import numpy as np

import kv4_plain as P

E = 2.0 ** -24


def chain_many(n):
    """Units of e that the sums of the kernel for many rows may be off, n visible cells."""
    return 2 * 48 + n / 256 + 32


def chain_few(n):
    return 2 * 2 * (n / 64 + 2) + 64


def bound_f32(pv, A, D, chain, spread=0.0):
    ds = (2.0 ** -21 + (6 * D / 16 + 16) * E) * A + 4 * E * spread
    return (2 * ds + 2.0 ** -20 + 2.0 ** -21 + chain * E) * pv


def attend64(q, kb, vb, Hk, scale, ranges, mask=None):
    """q: torch [T, H, D]; kb, vb: ggml rows; -> (out, sum p |v|, largest scale sum |q||k|) as numpy f64."""
    import torch
    T, H, D = q.shape
    n, dev = len(kb), q.device
    k, v = (torch.from_numpy(P.unpack(b)).to(dev).view(n, Hk, D) for b in (kb, vb))
    r = torch.as_tensor(np.asarray(ranges), device=dev)
    at = torch.arange(n, device=dev)
    seen = (at >= r[:, :1].clamp_min(0)) & (at < r[:, 1:])
    if mask is not None:
        m = torch.from_numpy(mask.astype(np.float64)).to(dev)
        seen &= ~torch.isneginf(m)
    out, pv = (np.zeros((T, H, D)) for _ in range(2))
    A = np.zeros((T, H, 1))
    for h in range(H):
        qh, kh, vh = q[:, h].double(), k[:, h // (H // Hk)], v[:, h // (H // Hk)]
        s = qh @ kh.T * scale
        if mask is not None:
            s = s + torch.where(seen, m, 0.0)
        s = torch.where(seen, s, -torch.inf)
        p = torch.where(seen, torch.exp(s - s.amax(1, keepdim=True).nan_to_num(neginf=0.0)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        out[:, h], pv[:, h] = (p @ vh).cpu().numpy(), (p @ vh.abs()).cpu().numpy()
        A[:, h, 0] = torch.where(seen, abs(scale) * (qh.abs() @ kh.abs().T), 0.0).amax(1).cpu().numpy()
    return out, pv, A
