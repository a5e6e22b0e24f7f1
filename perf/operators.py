"""What the 8-bit cache operators and the token log-probability operators are measured by.

The decoder caches four rows a token and layer (K_same, K_cross, V_same, V_cross; modality-routed attention reads one K and one V row of
every key).  In the 8-bit form a buffer is uint8 codes [4, B, H, capacity, 128] (e4m3 values) and uint8 scales [4, B, H, capacity / block]:
the value is code * 2^(scale - 127), one scale for each block of tokens and head.
"""
import math

import torch

own = False            # set from outside: run() makes the framework's calls instead of the plain form

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
D = 128                # channels of a head
NEWLINE, TEXT, CODES = 13, 32000, 514      # the decoder's newline id, text vocabulary and image codes (512 + begin + end of image)


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one generation step of a single conversation: one layer's four rows of one token
        dict(name="append_1x32", op="append", B=1, H=32, cap=2048, block=16, slot=1029),
        # one generation step of a serving batch
        dict(name="append_64x32", op="append", B=64, H=32, cap=1024, block=16, slot=776),
        # prompts of uneven lengths, padded on the left to the longest (an image is 578 tokens, a sentence follows)
        dict(name="fill_3x611_padded", op="fill", B=3, S=611, H=32, cap=768, block=16, padded=True),
        # the full context of the training recipe as a prompt
        dict(name="fill_8x2048", op="fill", B=8, S=2048, H=32, cap=2048, block=16, padded=False),
        # one image's tokens read back from the middle of a cache, begin and end inside a block
        dict(name="read_1x577", op="read", B=1, n=577, first=33, H=32, cap=1024, block=16),
        # a whole cache read back, a scale for each token
        dict(name="read_8x1024", op="read", B=8, n=1024, first=0, H=32, cap=1024, block=1),
        # a step of one conversation with a long context
        dict(name="attn_1x8191", op="attn", B=1, L=8191, H=32, cap=8192, block=16, ragged=False, image=578),
        # the step that the generation benchmark times: 8 sequences, a context of 1024 with one image
        dict(name="attn_8x1024", op="attn", B=8, L=1024, H=32, cap=1088, block=16, ragged=False, image=578),
        # a serving batch of uneven contexts, left-padded prompts
        dict(name="attn_48x2048_ragged", op="attn", B=48, L=2048, H=32, cap=2048, block=32, ragged=True, image=578),
        # what a step answers with: 8 sequences x 2 codebooks over the padded vocabulary, 20 alternatives
        dict(name="logp_step_16x32514", op="logp", rows=16, V=TEXT + CODES, T=1, top=20, half=True, grad=False, f32=False),
        # the image tokens of a batch of 16 under one codebook's head: log probabilities and entropies with their gradient
        dict(name="logp_train_9248x514", op="logp", rows=9248, V=CODES, T=1, top=0, half=False, grad=True, f32=False),
        # the text tokens of a batch of 4 x 2047 under the language head, the two codebooks' targets, with the gradient
        dict(name="logp_train_8188x32000", op="logp", rows=8188, V=TEXT, T=2, top=0, half=False, grad=True, f32=False),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "fill", "read", "attn", "attn", "logp", "logp"])
    H = rng.choice([2, 5, 7, 16, 32, 32])
    block = rng.choice([1, 4, 16, 16, 32, 64])
    up = lambda n: (n + block - 1) // block * block  # noqa: E731
    if op == "append":
        cap = up(_log(rng, 64, 4096))
        return dict(op=op, B=_log(rng, 1, 64), H=H, cap=cap, block=block, slot=rng.randrange(cap))
    if op == "fill":
        S = _log(rng, 1, 2048)
        return dict(op=op, B=_log(rng, 1, 8), S=S, H=H, cap=up(S + rng.randrange(1, 200)), block=block, padded=rng.random() < 0.5)
    if op == "read":
        n = _log(rng, 1, 2048)
        first = rng.randrange(0, 100)
        return dict(op=op, B=_log(rng, 1, 8), n=n, first=first, H=H, cap=up(first + n), block=block)
    if op == "attn":
        L = _log(rng, 1, 8192)
        B = _log(rng, 1, max(1, min(48, 48 * 2048 // L)))
        return dict(op=op, B=B, L=L, H=H, cap=up(L + rng.randrange(0, 64)), block=block, ragged=rng.random() < 0.5,
                    image=rng.choice([0, 18, 578]))
    half = rng.random() < 0.25
    V = TEXT + CODES if half else _log(rng, 3, 40000)
    grad = not half and rng.random() < 0.5
    top = 0 if grad else rng.choice([0, 1, 5, 20])
    rows = _log(rng, 1, max(2, min(16384, (64 << 20) // V)))
    return dict(op="logp", rows=rows, V=V, T=rng.choice([1, 1, 2]), top=min(top, V), half=half, grad=grad,
                f32=not half and rng.random() < 0.3)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _lens(case):
    """(first valid key, end of the valid keys) of every sequence: a function of the case alone, so that work() knows them."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [0] * B, [L] * B
    end = [max(1, L - (b * L) // (2 * B)) for b in range(B)]
    return [(b * 37) % max(1, end[b] // 3 + 1) if b % 2 else 0 for b in range(B)], end


def _activations(g, shape, dev, outlier):
    """bf16 rows like a decoder's: some channels of a head many times wider than the others, tokens of uneven size."""
    x = torch.randn(shape, generator=g, device=dev)
    x = x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device=dev))
    if outlier:
        x = x * (1 + 7 * (torch.rand(shape[-1], generator=g, device=dev) < 0.05))
    return x.to(BF16)


def _four_rows(g, n, H, dev):
    """K_same, K_cross, V_same, V_cross of n tokens as the decoder holds them: K_same and V_same are columns of its fused q|k|v rows."""
    fused = torch.cat([_activations(g, (n, H * D), dev, i < 2) for i in range(3)], 1)
    return [fused[:, H * D:2 * H * D], _activations(g, (n, H * D), dev, True), fused[:, 2 * H * D:], _activations(g, (n, H * D), dev, False)]


def _filled(g, B, H, cap, block, dev):
    """Codes and scales of a cache in use: values over the whole of e4m3 without its two NaNs, scales of uneven blocks."""
    x = torch.randn((4, B, H, cap, D), generator=g, device=dev).clamp_(-4.4, 4.4).mul_(100)
    codes = x.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.randint(117, 122, (4, B, H, cap // block), generator=g, device=dev, dtype=torch.uint8)
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    s = dict(case=case)
    op = case["op"]
    if op == "logp":
        rows, V, T = case["rows"], case["V"], case["T"]
        z = torch.empty((rows, V), dtype=F32 if case["f32"] else BF16, device=dev)
        for r in range(0, rows, 1024):
            z[r:r + 1024] = 2.5 * torch.randn(z[r:r + 1024].shape, generator=g, device=dev)
        t = torch.randint(0, V, (T, rows), generator=g, device=dev)
        if case["half"]:         # every other row speaks text, the others image codes; the foreign half of the columns is masked
            z[::2, TEXT:] = -math.inf
            z[1::2, :TEXT] = -math.inf
            t[:, ::2] %= TEXT
            t[:, 1::2] = TEXT + t[:, 1::2] % CODES
            if rows >= 8:        # behind an image's end a newline is forced
                z[6] = -math.inf
                z[6, NEWLINE] = math.inf
                t[:, 6] = NEWLINE
        likely = torch.rand((T, rows), generator=g, device=dev) < 0.7          # most given tokens are likely ones
        for i in range(T):
            at = torch.nonzero(likely[i]).squeeze(1)
            z[at, t[i, at]] += 9
        t[torch.rand((T, rows), generator=g, device=dev) < 0.1] = -100         # positions that are not scored
        s.update(z=z, t=t)
        if case["grad"]:
            s.update(g_lp=torch.randn((T, rows), generator=g, device=dev) / rows,
                     g_ent=0.01 * torch.randn(rows, generator=g, device=dev) / rows)
        return s
    B, H, cap, block = case["B"], case["H"], case["cap"], case["block"]
    if op == "fill":
        s["rows"] = _four_rows(g, B * case["S"], H, dev)
        s["start"] = None
        if case["padded"]:
            s["start"] = torch.randint(0, case["S"] // 2 + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            s["start"][B - 1] = 0
        s["codes"] = torch.zeros((4, B, H, cap, D), dtype=torch.uint8, device=dev)
        s["scales"] = torch.zeros((4, B, H, cap // block), dtype=torch.uint8, device=dev)
        return s
    s["codes"], s["scales"] = _filled(g, B, H, cap, block, dev)
    if op == "append":
        s["rows"] = _four_rows(g, B, H, dev)
        s["slot"] = torch.tensor([case["slot"]], device=dev)
    elif op == "attn":
        start, end = (torch.tensor(v, dtype=torch.int32, device=dev) for v in _lens(case))
        turn = torch.randperm(B, generator=g, device=dev)
        s["start"], s["end"] = (start[turn].contiguous() if case["ragged"] else None), end[turn].contiguous()
        s["q"] = _activations(g, (B, 3 * H * D), dev, False)[:, :H * D]                     # the q columns of the fused rows
        at = torch.randint(0, max(1, cap // 3), (B, 1), generator=g, device=dev)            # where the image lies in the context
        pos = torch.arange(cap, device=dev)[None]
        s["key_flag"] = ((pos >= at) & (pos < at + case["image"])).to(torch.uint8)
        s["query_flag"] = (torch.rand(B, generator=g, device=dev) < 0.3).to(torch.uint8)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        from libra_amd import kernels as K
        if case["op"] == "append":
            K.kv8_append(s["rows"], s["codes"], s["scales"], s["slot"])
            return _cache(s)
        if case["op"] == "fill":
            K.kv8_fill(s["rows"], s["codes"], s["scales"], case["S"], kv_start=s["start"])
            return _cache(s)
        if case["op"] == "read":
            return K.kv8_read(s["codes"], s["scales"], case["first"], case["n"])
        if case["op"] == "attn":
            return K.bridge_attn_decode8(s["q"], s["codes"], s["scales"], s["key_flag"], s["query_flag"], s["end"], D ** -0.5,
                                         kv_start=s["start"])
        out = K.token_logprobs(s["z"], s["t"], top=case["top"])
        if case["grad"]:
            dz = K.token_logprobs_bwd(s["z"], s["t"], out.stats, s["g_lp"], s["g_ent"])
            return dict(logprobs=out.logprobs, entropy=out.entropy, dlogits=dz)
        return dict(logprobs=out.logprobs, entropy=out.entropy, top_ids=out.top_ids, top_logprobs=out.top_logprobs)
    return dict(append=_append, fill=_fill, read=_read, attn=_attn, logp=_logp)[case["op"]](s)


def _cache(s):
    """The cache as the values it stands for: e4m3 codes and powers of two, its own buffers."""
    return dict(values=s["codes"].view(torch.float8_e4m3fn), scales=s["scales"].view(torch.float8_e8m0fnu))


def _exponent(a):
    """Smallest s >= -126 with a <= 448 * 2^s."""
    m, e = torch.frexp(a)
    return torch.where(a > 0, (e - 9 + (m > 0.875).to(e.dtype)), torch.full_like(e, -126)).clamp_min(-126)


def _e4m3(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _value(codes):
    return codes.view(torch.float8_e4m3fn).to(F32)


def _append(s):
    case = s["case"]
    B, H, slot, block = case["B"], case["H"], case["slot"], case["block"]
    x = torch.stack([r.reshape(B, H, D) for r in s["rows"]]).to(F32)
    e = _exponent(x.abs().amax(-1))
    j = slot // block
    if slot % block:
        old = s["scales"][..., j].to(torch.int32) - 127
        e = torch.maximum(e, old)
        before = s["codes"][..., j * block:slot, :]
        before.copy_(_e4m3(torch.ldexp(_value(before), (old - e)[..., None, None])))
    s["codes"][..., slot, :] = _e4m3(torch.ldexp(x, -e[..., None]))
    s["scales"][..., j] = (e + 127).to(torch.uint8)
    return _cache(s)


def _fill(s):
    case = s["case"]
    B, H, S, block = case["B"], case["H"], case["S"], case["block"]
    n = (S + block - 1) // block
    x = torch.zeros((4, B, H, n * block, D), dtype=F32, device=s["codes"].device)
    x[..., :S, :] = torch.stack([r.reshape(B, S, H, D) for r in s["rows"]]).transpose(2, 3)
    if s["start"] is not None:
        pad = torch.arange(n * block, device=x.device)[None] < s["start"][:, None]
        x.masked_fill_(pad[None, :, None, :, None], 0)
    x = x.view(4, B, H, n, block, D)
    e = _exponent(x.abs().amax((-1, -2)))
    codes = _e4m3(torch.ldexp(x, -e[..., None, None])).view(4, B, H, n * block, D)
    s["codes"][..., :S, :] = codes[..., :S, :]
    s["scales"][..., :n] = (e + 127).to(torch.uint8)
    return _cache(s)


def _read(s):
    case = s["case"]
    B, H, first, n, block = case["B"], case["H"], case["first"], case["n"], case["block"]
    e = (s["scales"].to(torch.int32) - 127).repeat_interleave(block, -1)[..., first:first + n]
    x = torch.ldexp(_value(s["codes"][..., first:first + n, :]), e[..., None])
    return x.transpose(2, 3).reshape(4, B, n, H * D).to(BF16)


def _attn(s):
    case = s["case"]
    B, H, L, block = case["B"], case["H"], case["L"], case["block"]
    e = (s["scales"].to(torch.int32) - 127).repeat_interleave(block, -1)[..., :L]
    cross = (s["key_flag"][:, :L] != s["query_flag"][:, None])[:, None, :, None]
    row = lambda i: torch.ldexp(_value(s["codes"][i, :, :, :L]), e[i][..., None])  # noqa: E731
    k = torch.where(cross, row(1), row(0))
    sc = (k * s["q"].to(F32).view(B, H, 1, D)).sum(-1) * D ** -0.5
    pos = torch.arange(L, device=sc.device)[None]
    ok = pos < s["end"][:, None]
    if s["start"] is not None:
        ok = ok & (pos >= s["start"][:, None])
    sc = sc.masked_fill(~ok[:, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.where(ok[:, None], torch.exp(sc - torch.where(m > -math.inf, m, torch.zeros_like(m))), torch.zeros_like(sc))
    v = torch.where(cross, row(3), row(2))
    total = p.sum(-1, keepdim=True)
    o = (p[..., None] * v).sum(-2) / torch.where(total > 0, total, torch.ones_like(total))
    return o.reshape(B, H * D).to(BF16)


def _logp(s):
    case, z, t = s["case"], s["z"].to(F32), s["t"]
    m = z.amax(-1, keepdim=True)
    d = torch.where(z == m, torch.zeros_like(z), z - m)                  # (a row whose largest is infinite: 0 there, -inf elsewhere)
    e = torch.exp(d)
    rest = e.scatter(1, z.argmax(-1, keepdim=True), 0).sum(-1, keepdim=True)      # beside the largest: a sure token's log p is log1p of this
    log_sum = torch.log1p(rest)
    logp = d - log_sum
    entropy = (log_sum - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(-1, keepdim=True) / (1 + rest)).squeeze(-1)
    given = torch.gather(logp, 1, t.clamp_min(0).t()).t()
    out = dict(logprobs=torch.where(t < 0, torch.zeros_like(given), given), entropy=entropy)
    if case["grad"]:
        p = torch.exp(logp)
        g_lp = torch.where(t < 0, torch.zeros_like(s["g_lp"]), s["g_lp"])
        dz = -p * torch.where(p > 0, logp + entropy[:, None], torch.zeros_like(p)) * s["g_ent"][:, None]
        for i in range(t.shape[0]):                                      # [v = t] - p, at v = t as 1 - p without the loss of a sure token
            one_less = (-p).scatter(1, t[i].clamp_min(0)[:, None], -torch.expm1(given[i])[:, None])
            dz += g_lp[i][:, None] * one_less
        out["dlogits"] = dz.to(s["z"].dtype)
        return out
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top"]] if case["top"] else torch.zeros((z.shape[0], 0), dtype=torch.int64, device=z.device)
    return dict(out, top_ids=order, top_logprobs=torch.gather(logp, 1, order))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "logp":
        n = case["rows"] * case["V"]
        size = 4 if case["f32"] else 2
        per_row = case["rows"] * (case["T"] * 12 + 4 + case["top"] * 12 + (case["T"] * 4 + 4 if case["grad"] else 0))
        return dict(bytes=n * size * (2 if case["grad"] else 1) + per_row, flops=n * (10 if case["grad"] else 5))
    B, H, block = case["B"], case["H"], case["block"]
    if op == "attn":
        start, end = _lens(case)
        keys = sum(b - a for a, b in zip(start, end))
        return dict(bytes=keys * (H * (2 * D + 2 / block) + 1) + 4 * B * H * D, flops=keys * H * 4 * D)
    n = dict(append=1, fill=case.get("S"), read=case.get("n"))[op]
    tokens = 4 * B * H * n
    return dict(bytes=tokens * D * 3 + 4 * B * H * ((n + block - 1) // block), flops=tokens * D * 2)


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------------------------
def _grid(dev):
    """The 127 non-negative e4m3 numbers (4 exponent bits of bias 7, 3 of mantissa, no infinities; the 128th is NaN)."""
    low = [k * 2.0 ** -9 for k in range(8)]
    return torch.tensor((low + [(8 + k) * 2.0 ** (e - 10) for e in range(1, 16) for k in range(8)])[:127], dtype=F64, device=dev)


def _to_grid(y):
    """y (|y| <= 448) to the nearest e4m3 number, the even code where two are as near."""
    grid = _grid(y.device)
    a = y.abs()
    hi = torch.searchsorted(grid, a).clamp_(max=126)
    lo = (hi - 1).clamp_(min=0)
    below, above = a - grid[lo], grid[hi] - a
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(grid[code], y)


def _shift(a):
    """log2 of a block's scale: of the powers of two that bring a to 448 or less, the smallest, not below 2^-126."""
    return torch.where(a > 0, torch.ceil(torch.log2(a.clamp_min(1e-300) / 448)), torch.full_like(a, -126)).clamp_min(-126)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logp":
        parts = [_exact_logp(case, s, r, min(case["rows"], r + 512)) for r in range(0, case["rows"], 512)]
        return {k: torch.cat([p[k] for p in parts], 1 if k == "logprobs" else 0) for k in parts[0]}
    B, H, block = case["B"], case["H"], case["block"]
    dev = s["codes"].device
    grid = torch.cat([_grid(dev), torch.full((1,), math.nan, dtype=F64, device=dev)])
    value = lambda c: torch.where(c < 128, grid[(c & 127).long()], -grid[(c & 127).long()])  # noqa: E731
    if op == "read":
        w = slice(case["first"], case["first"] + case["n"])
        at = torch.arange(case["cap"], device=dev)[w] // block
        x = value(s["codes"][..., w, :]) * torch.exp2(s["scales"].to(F64) - 127)[..., at][..., None]
        return x.permute(0, 1, 3, 2, 4).reshape(4, B, case["n"], H * D)
    if op == "attn":
        out = torch.zeros((B, H, D), dtype=F64, device=dev)
        for b in range(B):
            i, n = (int(s["start"][b]) if s["start"] is not None else 0), int(s["end"][b])
            if n <= i:
                continue
            cross = (s["key_flag"][b, i:n] != s["query_flag"][b]).long()
            j = torch.arange(i, n, device=dev)
            scale = torch.exp2(s["scales"][:, b].to(F64) - 127)
            k = value(s["codes"][cross, b, :, j]) * scale[cross, :, j // block][..., None]              # [n, H, D]
            v = value(s["codes"][2 + cross, b, :, j]) * scale[2 + cross, :, j // block][..., None]
            a = torch.einsum("nhd,hd->hn", k, s["q"][b].to(F64).view(H, D)) / math.sqrt(D)
            out[b] = torch.einsum("hn,nhd->hd", torch.softmax(a, -1), v)
        return out.reshape(B, H * D)
    values, scales = value(s["codes"]), torch.exp2(s["scales"].to(F64) - 127)
    if op == "append":
        slot, j = case["slot"], case["slot"] // block
        for i in range(4):
            x = s["rows"][i].to(F64).reshape(B, H, D)
            e = _shift(x.abs().amax(-1))
            if slot % block:
                old = torch.log2(scales[i, :, :, j])
                e = torch.maximum(e, old)
                w = slice(j * block, slot)
                values[i, :, :, w] = _to_grid(values[i, :, :, w] * torch.exp2(old - e)[..., None, None])
            values[i, :, :, slot] = _to_grid(x * torch.exp2(-e)[..., None])
            scales[i, :, :, j] = torch.exp2(e)
        return dict(values=values, scales=scales)
    S = case["S"]                                                       # fill
    scales = torch.exp2(torch.full_like(scales, -127))
    for i in range(4):
        x = s["rows"][i].to(F64).reshape(B, S, H, D).permute(0, 2, 1, 3).contiguous()
        if s["start"] is not None:
            for b in range(B):
                x[b, :, :int(s["start"][b])] = 0
        for j in range((S + block - 1) // block):
            w = slice(j * block, min(S, (j + 1) * block))
            e = _shift(x[:, :, w].abs().amax((2, 3)))
            values[i, :, :, w] = _to_grid(x[:, :, w] * torch.exp2(-e)[..., None, None])
            scales[i, :, :, j] = torch.exp2(e)
    return dict(values=values, scales=scales)


def _exact_logp(case, s, r0, r1):
    z, t = s["z"][r0:r1].to(F64), s["t"][:, r0:r1]
    forced = torch.isinf(z) & (z > 0)
    z = torch.where(forced.any(-1, keepdim=True), torch.where(forced, torch.zeros_like(z), torch.full_like(z, -math.inf)), z)
    logp = torch.log_softmax(z, -1)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    scored = t >= 0
    col = torch.where(scored, t, torch.zeros_like(t))
    rows = torch.arange(r1 - r0, device=z.device)
    lp = torch.stack([torch.where(scored[i], logp[rows, col[i]], torch.zeros_like(entropy)) for i in range(case["T"])])
    out = dict(logprobs=lp, entropy=entropy)
    if case["grad"]:
        g_ent = s["g_ent"][r0:r1].to(F64)
        dz = g_ent[:, None] * -p * (torch.where(p > 0, logp, torch.zeros_like(p)) + entropy[:, None])
        for i in range(case["T"]):
            gi = torch.where(scored[i], s["g_lp"][i, r0:r1].to(F64), torch.zeros_like(g_ent))
            hit = torch.zeros_like(z)
            hit[rows, col[i]] = 1
            dz = dz + gi[:, None] * (hit - p)
        return dict(out, dlogits=dz)
    # (the alternatives' order is the inputs' own and compared with the plain form's; their values are these)
    shown = s["z"][r0:r1].to(F64)
    ids = torch.argsort(shown, dim=-1, descending=True, stable=True)[:, :case["top"]]
    return dict(out, top_ids=ids, top_logprobs=logp.gather(1, ids))
