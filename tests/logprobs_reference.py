"""Token log probabilities in plain 64-bit arithmetic: the definition that the device tests compare with."""
import torch

NINF, INF = -float("inf"), float("inf")


def logprobs(z):
    """[rows, V] 64-bit -> log p [rows, V], entropy [rows] (rows with +inf are shared by them; nothing but -inf: -inf and 0; NaN: NaN)."""
    forced = z == INF
    z = torch.where(forced.any(-1, keepdim=True), torch.where(forced, torch.zeros_like(z), torch.full_like(z, NINF)), z)
    lp = torch.log_softmax(z, -1)
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    empty = (z == NINF).all(-1)
    nan = torch.isnan(z).any(-1)
    lp = torch.where(empty[:, None], torch.full_like(lp, NINF), lp)
    ent = torch.where(empty, torch.zeros_like(ent), ent)
    return torch.where(nan[:, None], torch.full_like(lp, float("nan")), lp), torch.where(nan, torch.full_like(ent, float("nan")), ent)


def pick(lp, targets, sub):
    T, rows = targets.shape
    out = torch.zeros(T, rows, dtype=lp.dtype)
    for i in range(T):
        for r in range(rows):
            t = int(targets[i, r])
            out[i, r] = 0.0 if t < 0 else (lp[r, t - sub] if 0 <= t - sub < lp.shape[1] else (lp[r, 0] if torch.isnan(lp[r, 0]) else NINF))
    return out


def order(z, top):
    """Larger first, equal ones by the smaller column, NaN last."""
    key = torch.where(torch.isnan(z), torch.full_like(z, NINF), z)
    behind = torch.isnan(z)
    rows = []
    for r in range(z.shape[0]):
        idx = sorted(range(z.shape[1]), key=lambda v: (bool(behind[r, v]), -float(key[r, v]), v))
        rows.append(idx[:top])
    return torch.tensor(rows, dtype=torch.int64).view(z.shape[0], top)


def gradient(z, targets, sub, g_lp, g_ent):
    lp, ent = logprobs(z)
    p = torch.exp(lp)
    dz = -g_ent[:, None] * torch.where(p > 0, p * (lp + ent[:, None]), torch.zeros_like(p))
    for i in range(targets.shape[0]):
        for r in range(z.shape[0]):
            t = int(targets[i, r])
            if t >= 0:
                dz[r] -= g_lp[i, r] * p[r]
                if 0 <= t - sub < z.shape[1]:
                    dz[r, t - sub] += g_lp[i, r]
    flat = torch.isinf(z.amax(-1))
    return torch.where(flat[:, None], torch.zeros_like(dz), dz)
