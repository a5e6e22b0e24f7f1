"""The 8-bit K/V cache in plain 64-bit arithmetic on the host: the definition that the device tests compare with."""
import torch

F64 = torch.float64
GRID = torch.tensor([k * 2.0 ** -9 for k in range(8)] + [(8 + k) * 2.0 ** (e - 10) for e in range(1, 16) for k in range(8)][:-1], dtype=F64)


def to_grid(y):
    """Nearest e4m3 number (ties: even code), +-448 beyond, NaN kept."""
    a = y.abs().clamp(max=448.0)
    hi = torch.searchsorted(GRID, torch.nan_to_num(a)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = a - GRID[lo], GRID[hi] - a
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return torch.where(torch.isnan(y), y, torch.copysign(GRID[code], y))


def values(codes):
    grid = torch.cat([GRID, torch.tensor([float("nan")], dtype=F64)])
    c = codes.cpu().long()
    return torch.where(c < 128, grid[c & 127], -grid[c & 127])


def shift(x, dims):
    """log2 of the scale of blocks of x: over the finite values; -126 where there is none."""
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)
    return torch.where(a > 0, torch.ceil(torch.log2(a.clamp_min(1e-300) / 448)), torch.full_like(a, -126.0)).clamp_min(-126)


def empty(B, H, cap, block):
    return torch.zeros(4, B, H, cap, 128, dtype=F64), torch.full((4, B, H, cap // block), -126.0, dtype=F64)


def fill(rows, vals, exps, S, block, start=None):
    """rows: four [B*S, H*128]; vals: code values, exps: log2 of the scales (both written in place)."""
    B, H = vals.shape[1:3]
    for i, r in enumerate(rows):
        x = r.cpu().to(F64).view(B, S, H, 128).transpose(1, 2).clone()
        for b in range(B):
            if start is not None:
                x[b, :, :max(0, int(start[b]))] = 0
        for j in range((S + block - 1) // block):
            w = slice(j * block, min(S, (j + 1) * block))
            e = shift(x[:, :, w], (2, 3))
            vals[i, :, :, w] = to_grid(x[:, :, w] * torch.exp2(-e)[..., None, None])
            exps[i, :, :, j] = e


def append(rows, vals, exps, slot, block):
    B, H = vals.shape[1:3]
    j = slot // block
    for i, r in enumerate(rows):
        x = r.cpu().to(F64).view(B, H, 128)
        e = shift(x, (2,))
        if slot % block:
            old = exps[i, :, :, j]
            e = torch.maximum(e, old)
            w = slice(j * block, slot)
            vals[i, :, :, w] = to_grid(vals[i, :, :, w] * torch.exp2(old - e)[..., None, None])
        vals[i, :, :, slot] = to_grid(x * torch.exp2(-e)[..., None])
        exps[i, :, :, j] = e


def dense(vals, exps, block):
    return vals * torch.exp2(exps).repeat_interleave(block, -1)[..., None]


def attention(q, full, key_flag, query_flag, kv_len, kv_start, scale):
    """q [B, H*128], full [4, B, H, cap, 128] (64-bit) -> (o [B, H, 128], the largest score error factor sum |q||k| scale [B, H])."""
    B, H, cap = full.shape[1:4]
    o, reach = torch.zeros(B, H, 128, dtype=F64), torch.zeros(B, H, dtype=F64)
    for b in range(B):
        i, n = max(0, int(kv_start[b]) if kv_start is not None else 0), min(cap, int(kv_len[b]))
        if n <= i:
            continue
        cross = (key_flag[b, i:n].cpu() != 0) != bool(query_flag[b])
        k = torch.where(cross[None, :, None], full[1, b, :, i:n], full[0, b, :, i:n])
        v = torch.where(cross[None, :, None], full[3, b, :, i:n], full[2, b, :, i:n])
        qb = q[b].cpu().to(F64).view(H, 1, 128)
        o[b] = (torch.softmax((k * qb).sum(-1) * scale, -1)[..., None] * v).sum(-2)
        reach[b] = (k.abs() * qb.abs()).sum(-1).amax(-1) * scale
    return o, reach
