"""The recurrence of linear attention as it is written, token by token in 64 bits, and the norms' formula."""
import numpy as np
import torch


def recurrence(q, k, v, g, S, scale):
    """One sequence: q, k [T, Hk, dk], v [T, H, dv], g [T, H], S [H, dk, dv], all float64.  Returns (out, S)."""
    T, H = v.shape[:2]
    r = H // q.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    out = torch.zeros_like(v)
    S = S.clone()
    for t in range(T):
        decay = torch.exp(g[t])[:, None, None]
        S = torch.where(decay == 0, torch.zeros_like(S), decay * S) + k[t][:, :, None] * v[t][:, None, :]
        out[t] = scale * torch.einsum("hk,hkv->hv", q[t], S)
    return out, S


def norm2(x, mode, groups, weight, bias, eps):
    rows = x.reshape(x.shape[0], groups, -1)
    if mode == "none":
        out = x.clone()
    else:
        if mode == "layer":
            rows = rows - rows.mean(-1, keepdim=True)
        out = (rows / torch.sqrt((rows ** 2).mean(-1, keepdim=True) + eps)).reshape(x.shape)
    out = out * (1 if weight is None else weight)
    return out if bias is None else out + bias


def rel(a, b):
    """2-norm of the difference over the 2-norm of the reference."""
    a, b = a.detach().double().cpu().numpy().ravel(), b.detach().double().cpu().numpy().ravel()
    assert a.shape == b.shape and np.isfinite(a).all()
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)) if np.linalg.norm(b) else float(np.linalg.norm(a))
