"""The 8-bit K/V cache on the device: written (prompt, single tokens), read back, attended over - against the 64-bit definition
(kv8_reference.py).  Writing and reading are exact: every rounding is defined.  Attention: fp32 arithmetic and one rounding to bf16 at the
end, i.e. 2^-8 |o| plus what fp32 leaves: a score of 128 products is off by at most 130 * 2^-24 * sum |q||k| * scale =: d, a probability by
2 d + 2^-20 relative (exp2, and sums of up to L / 32 + 64 terms in fp32: (L / 32 + 64) 2^-24), and o by that times 2 max |v|."""
import pytest
import torch

import kv8_reference as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from libra_amd import kernels
    return kernels


def rows4(n, H, seed, wild=False):
    """K_same, K_cross, V_same, V_cross as the engine holds them (two are column slices of fused rows)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 5 * H * 128, generator=g)
    x *= torch.exp(torch.randn(n, 1, generator=g)) * (1 + 30 * (torch.rand(1, 5 * H * 128, generator=g) < 0.03))
    if wild:                                            # the number format's corners
        special = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 1e-38, 9e-41, 448.0, 464.0, 1.75, 1.76])
        at = torch.randint(0, x.numel(), (x.numel() // 50,), generator=g)
        x.view(-1)[at] = special[torch.randint(0, len(special), (len(at),), generator=g)]
        x[::3] *= 2.0 ** -30
    x = x.to(BF).cuda()
    D = H * 128
    return [x[:, D:2 * D], x[:, 3 * D:4 * D].contiguous(), x[:, 2 * D:3 * D], x[:, 4 * D:].contiguous()]


def same(codes, scales, vals, exps, upto=None):
    got = R.values(codes)
    n = got.shape[3] if upto is None else upto
    assert torch.equal(scales.cpu().double()[..., :] - 127, exps), "scales"
    a, b = got[:, :, :, :n], vals[:, :, :, :n]
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), "codes"


@pytest.mark.parametrize("B,S,H,cap,block,start,wild", [
    (1, 1, 1, 1, 1, None, False), (1, 1, 2, 64, 64, None, False), (2, 17, 3, 32, 16, None, True), (3, 77, 2, 96, 32, [5, 0, 40], True),
    (2, 64, 17, 64, 4, [64, 63], False), (1, 130, 32, 192, 64, [64], False), (2, 33, 5, 36, 2, None, True)])
def test_fill(K, B, S, H, cap, block, start, wild):
    codes, scales = K.kv8_alloc(B, cap, H, "cuda", block)
    codes.fill_(0x11)                                   # what lies behind the prompt stays as it was
    scales.fill_(77)
    rows = rows4(B * S, H, 1, wild)
    st = torch.tensor(start, dtype=torch.int32, device="cuda") if start else None
    K.kv8_fill(rows, codes, scales, S, kv_start=st)
    vals, exps = R.empty(B, H, cap, block)
    n = (S + block - 1) // block
    vals[:] = R.values(torch.tensor([0x11]))
    exps[..., n:] = 77 - 127
    R.fill(rows, vals, exps, S, block, start)
    same(codes, scales, vals, exps)


@pytest.mark.parametrize("B,H,cap,block,slots,wild", [
    (1, 1, 4, 1, range(4), False), (2, 3, 48, 16, range(40), False), (3, 17, 64, 64, range(64), False), (2, 32, 16, 4, range(9), True),
    (1, 2, 32, 32, [0, 1, 1, 2, 1, 2, 3], False)])
def test_append_token_by_token(K, B, H, cap, block, slots, wild):
    """Every step equals the definition (scale of the first token, growth, earlier codes re-expressed), a slot written again included."""
    codes, scales = K.kv8_alloc(B, cap, H, "cuda", block)
    vals, exps = R.empty(B, H, cap, block)
    for step, slot in enumerate(slots):
        rows = rows4(B, H, 100 + step, wild)
        K.kv8_append(rows, codes, scales, torch.tensor([slot], device="cuda"))
        R.append(rows, vals, exps, slot, block)
    used = max(slots) // block + 1
    same(codes, scales[..., :used], vals, exps[..., :used])


def test_append_after_fill_and_bound(K):
    """Tokens appended behind a prompt that ends inside a block; every value within the documented distance of what was written."""
    B, S, H, cap, block = 2, 21, 4, 64, 16
    rows = rows4(B * S, H, 5)
    codes, scales = K.kv8_alloc(B, cap, H, "cuda", block)
    vals, exps = R.empty(B, H, cap, block)
    K.kv8_fill(rows, codes, scales, S)
    R.fill(rows, vals, exps, S, block)
    want = [r.cpu().double().view(B, S, H, 128) for r in rows]
    for t in range(S, 50):
        new = rows4(B, H, 200 + t)
        K.kv8_append(new, codes, scales, torch.tensor([t], device="cuda"))
        R.append(new, vals, exps, t, block)
        want = [torch.cat([w, n.cpu().double().view(B, 1, H, 128)], 1) for w, n in zip(want, new)]
    same(codes, scales[..., :4], vals, exps[..., :4])
    got = K.kv8_read(codes, scales, 0, 50).cpu().double().view(4, B, 50, H, 128)
    unit = torch.exp2(exps).repeat_interleave(block, -1)[..., :50].transpose(2, 3)[..., None]
    x = torch.stack(want)
    assert bool(((got - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -9 * unit)).all())


@pytest.mark.parametrize("slot", [-1, 32, 1 << 40])
def test_append_outside_stores_nothing(K, slot):
    codes, scales = K.kv8_alloc(1, 32, 2, "cuda", 16)
    K.kv8_append(rows4(1, 2, 3), codes, scales, torch.tensor([slot], device="cuda"))
    assert int(codes.max()) == 0 and int(scales.max()) == 0


@pytest.mark.parametrize("B,H,cap,block,first,n", [(1, 1, 1, 1, 0, 1), (2, 3, 64, 16, 5, 37), (2, 32, 128, 64, 127, 1), (1, 5, 96, 32, 0, 96), (1, 2, 8, 8, 3, 0)])
def test_read(K, B, H, cap, block, first, n):
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(0, 256, (4, B, H, cap, 128), generator=g, dtype=torch.uint8)        # all 256 codes, the two NaNs among them
    scales = torch.randint(1, 247, (4, B, H, cap // block), generator=g, dtype=torch.uint8)
    got = K.kv8_read(codes.cuda(), scales.cuda(), first, n)
    full = R.dense(R.values(codes), scales.double() - 127, block)[:, :, :, first:first + n].transpose(2, 3).reshape(4, B, n, H * 128)
    want = full.to(torch.float32).to(BF)                # exact but below bf16's normal range
    assert got.shape == (4, B, n, H * 128) and torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.cpu().float()), torch.nan_to_num(want.float()))
    ok = torch.isfinite(full) & (full.abs() >= 2.0 ** -126)
    assert torch.equal(got.cpu().double()[ok], full[ok])


def attn_case(K, B, H, cap, block, seed=0):
    """A cache written by fill, and a query."""
    rows = rows4(B * cap, H, seed)
    codes, scales = K.kv8_alloc(B, cap, H, "cuda", block)
    K.kv8_fill(rows, codes, scales, cap)
    g = torch.Generator().manual_seed(seed + 9)
    q = torch.randn(B, 3 * H * 128, generator=g).to(BF).cuda()[:, :H * 128]
    return q, codes, scales, g


def attn_check(K, q, codes, scales, kf, qf, ln, st):
    B, H, cap = codes.shape[1:4]
    out = K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5, kv_start=st)
    full = R.dense(R.values(codes), scales.cpu().double() - 127, cap // scales.shape[3])
    ref, reach = R.attention(q, full, kf, qf.cpu(), ln.cpu(), st.cpu() if st is not None else None, 128 ** -0.5)
    rel = 2 * 130 * 2.0 ** -24 * reach + 2.0 ** -20 + (cap / 32 + 64) * 2.0 ** -24
    vmax = torch.nan_to_num(full[2:]).abs().amax((0, 3, 4))
    err = (out.cpu().double().view(B, H, 128) - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + (2 * vmax * rel)[..., None]
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())
    return out


@pytest.mark.parametrize("B,H,cap,block", [(1, 1, 1, 1), (1, 2, 16, 16), (3, 2, 96, 32), (2, 4, 320, 64), (5, 7, 130, 2), (2, 32, 2048, 16), (1, 3, 5000, 8)])
def test_attention(K, B, H, cap, block):
    q, codes, scales, g = attn_case(K, B, H, cap, block)
    kf = (torch.rand(B, cap, generator=g) < 0.4).to(torch.uint8).cuda()
    qf = torch.tensor([i % 2 for i in range(B)], dtype=torch.uint8, device="cuda")
    ln = torch.randint(1, cap + 1, (B,), generator=g).to(torch.int32)
    ln[0] = cap
    if B > 1:
        ln[1] = 1
    attn_check(K, q, codes, scales, kf, qf, ln.cuda(), None)
    st = (torch.rand(B, generator=g) * ln).to(torch.int32)
    attn_check(K, q, codes, scales, kf, qf, ln.cuda(), st.cuda())


def test_attention_lengths(K):
    """Every length around the sizes at which waves, iterations and splits begin, in one batch."""
    ns = [0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 640]
    q, codes, scales, g = attn_case(K, len(ns), 2, 640, 16, 3)
    kf = (torch.rand(len(ns), 640, generator=g) < 0.5).to(torch.uint8).cuda()
    qf = torch.zeros(len(ns), dtype=torch.uint8, device="cuda")
    ln = torch.tensor(ns, dtype=torch.int32, device="cuda")
    out = attn_check(K, q, codes, scales, kf, qf, ln, None)
    assert float(out[0].float().abs().max()) == 0                                            # no key: zeros
    st = torch.tensor([min(n, 3 * i) for i, n in enumerate(ns)], dtype=torch.int32, device="cuda")
    attn_check(K, q, codes, scales, kf, qf, ln, st)
    wide = torch.full((len(ns),), 1 << 20, dtype=torch.int32, device="cuda")                 # limits outside the cache are cut to it
    attn_check(K, q, codes, scales, kf, qf, wide, -wide)
    assert float(K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 1.0, kv_start=ln).float().abs().max()) == 0


def test_attention_reads_valid_keys_only(K):
    """NaN and infinity codes at masked keys (before start, behind the end) and in the buffers that the routing does not select."""
    B, H, cap, block = 3, 2, 200, 8
    q, codes, scales, g = attn_case(K, B, H, cap, block, 4)
    kf = (torch.rand(B, cap, generator=g) < 0.5).to(torch.uint8).cuda()
    qf = torch.tensor([0, 1, 0], dtype=torch.uint8, device="cuda")
    ln = torch.tensor([150, 61, 200], dtype=torch.int32, device="cuda")
    st = torch.tensor([0, 13, 199], dtype=torch.int32, device="cuda")
    clean = K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5, kv_start=st)
    for b in range(B):
        cross = (kf[b] != 0) != bool(qf[b])
        dead = torch.ones(cap, dtype=torch.bool, device="cuda")
        dead[int(st[b]):int(ln[b])] = False
        for w in range(4):
            codes[w, b][:, dead | (~cross if w % 2 else cross)] = 0x7f
    assert torch.equal(clean, K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5, kv_start=st))


def test_attention_large_and_small_scores(K):
    """Scores far from zero: the running maximum carries them; a scale range of 2^60 between keys."""
    q, codes, scales, g = attn_case(K, 2, 2, 256, 16, 6)
    kf = torch.zeros(2, 256, dtype=torch.uint8, device="cuda")
    qf = torch.zeros(2, dtype=torch.uint8, device="cuda")
    ln = torch.tensor([256, 200], dtype=torch.int32, device="cuda")
    scales[:2] += torch.arange(0, 16, dtype=torch.uint8, device="cuda")[:scales.shape[3]] // 4
    scales[2:] -= torch.arange(0, 60, 4, dtype=torch.uint8, device="cuda").repeat(2)[:scales.shape[3]]
    attn_check(K, q * 4, codes, scales, kf, qf, ln, None)


def test_offsets_past_32_bits(K):
    """A cache of more than 4 GiB: the last slots of the last head of every buffer, written, read and attended over."""
    B, H, cap, block = 2, 8, 600064, 64                 # codes: 4 * 2 * 8 * 600064 * 128 = 4.9e9 bytes
    codes, scales = K.kv8_alloc(B, cap, H, "cuda", block)
    vals, exps = R.empty(B, H, 128, block)
    for t in range(cap - 100, cap):
        if t in (cap - 100, cap - 64, cap - 63, cap - 1):
            rows = rows4(B, H, t)
            K.kv8_append(rows, codes, scales, torch.tensor([t], device="cuda"))
            R.append(rows, vals, exps, t - cap + 128, block)
    same(codes[..., cap - 64:, :].contiguous(), scales[..., -1:], vals[..., 64:, :], exps[..., 1:])
    got = K.kv8_read(codes, scales, cap - 64, 64).cpu().double().view(4, B, 64, H, 128).transpose(2, 3)
    assert torch.equal(got, R.dense(vals[..., 64:, :], exps[..., 1:], block))
    kf = torch.zeros(B, cap, dtype=torch.uint8, device="cuda")
    qf = torch.tensor([0, 1], dtype=torch.uint8, device="cuda")
    q = rows4(B, H, 1)[1]
    ln = torch.full((B,), cap, dtype=torch.int32, device="cuda")
    out = K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5, kv_start=ln - 64)
    small_c, small_s = codes[..., cap - 64:, :].contiguous(), scales[..., -1:].contiguous()
    want = K.bridge_attn_decode8(q, small_c, small_s, kf[:, :64].contiguous(), qf, torch.full_like(ln, 64), 128 ** -0.5)
    assert torch.equal(out, want)


def test_deterministic_and_batch_independent(K):
    q, codes, scales, g = attn_case(K, 4, 4, 512, 16, 8)
    kf = (torch.rand(4, 512, generator=g) < 0.4).to(torch.uint8).cuda()
    qf = torch.tensor([0, 1, 1, 0], dtype=torch.uint8, device="cuda")
    ln = torch.tensor([512, 333, 64, 500], dtype=torch.int32, device="cuda")
    a = K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5)
    assert torch.equal(a, K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5))


def test_captured_step_replays(K):
    """Append + attention of a growing cache as one captured graph (slot, lengths on the device), two graphs alive at once, eager work
    between the replays: every replay equals the eager step."""
    B, H, cap, block = 2, 4, 64, 16
    slot = torch.zeros(1, dtype=torch.int64, device="cuda")
    ln = torch.zeros(B, dtype=torch.int32, device="cuda")
    kf = torch.zeros(B, cap, dtype=torch.uint8, device="cuda")
    qf = torch.tensor([0, 1], dtype=torch.uint8, device="cuda")
    buf = [r.clone() for r in rows4(B, H, 0)]
    q = buf[0]
    caches = [K.kv8_alloc(B, cap, H, "cuda", block) for _ in range(3)]

    def step(c):
        K.kv8_append(buf, *c, slot)
        return K.bridge_attn_decode8(q, *c, kf, qf, ln, 128 ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in caches[1:]:
            step(c)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in caches[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for c in caches:
        c[0].zero_(); c[1].zero_()
    for t in range(40):
        for b, r in zip(buf, rows4(B, H, 50 + t)):
            b.copy_(r)
        slot.fill_(t)
        ln.fill_(t + 1)
        want = step(caches[0])
        for g in graphs:
            g.replay()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), t
    assert all(torch.equal(c[0], caches[0][0]) and torch.equal(c[1], caches[0][1]) for c in caches[1:])


@pytest.mark.parametrize("B,H,block,two", [(3, 2, 16, False), (8, 32, 16, True), (1, 5, 64, False), (2, 17, 1, True)])
def test_rope_append_is_rope_then_append(K, B, H, block, two):
    """The fused step == rope_bridge_pos followed by kv8_append, bit for bit, token by token over block borders."""
    from oracle import libra_oracle as LO
    D, cap = H * 128, 64
    cosf, sinf = LO.rope_tables(128, 64)
    cos, sin = cosf.to(BF).cuda(), sinf.to(BF).cuda()
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    w = [0.3 * rnd(D, 8) for _ in range(4)]
    a, b = K.kv8_alloc(B, cap, H, "cuda", block), K.kv8_alloc(B, cap, H, "cuda", block)
    for t in list(range(19)) + [63, 64]:                # (64: outside, stores nothing)
        flag = (torch.rand(B, generator=g) < 0.5).to(torch.uint8).cuda()
        pos = torch.randint(0, 64, (B, 2) if two else (B,), generator=g).to(torch.int32).cuda()
        tb = torch.zeros(B, 64, dtype=BF, device="cuda"); tb[:, :16] = rnd(B, 16)
        qkv = (rnd(B, 3 * D + 64) * (1 + t % 5))[:, :3 * D]
        q2 = qkv.clone()
        slot = torch.tensor([t], device="cuda")
        K.rope_bridge_pos_append8(qkv, tb, *w, flag, cos, sin, pos, H, *a, slot)
        kc, vc = K.rope_bridge_pos(q2, tb, *w, flag, cos, sin, pos, H)
        K.kv8_append((q2[:, D:2 * D], kc, q2[:, 2 * D:], vc), *b, slot)
        assert torch.equal(qkv, q2) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), t
    with pytest.raises(ValueError):
        K.rope_bridge_pos_append8(qkv, tb, *w, flag, cos, sin, pos, H + 1, *a, slot)


def test_other_stream(K):
    """Work enqueued on a side stream runs on that stream."""
    q, codes, scales, g = attn_case(K, 2, 4, 256, 16, 12)
    kf = torch.zeros(2, 256, dtype=torch.uint8, device="cuda")
    qf = torch.zeros(2, dtype=torch.uint8, device="cuda")
    ln = torch.tensor([256, 9], dtype=torch.int32, device="cuda")
    want = K.bridge_attn_decode8(q, codes, scales, kf, qf, ln, 128 ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c2, s2 = torch.zeros_like(codes), torch.zeros_like(scales)
        K.kv8_fill([r.transpose(1, 2).reshape(2 * 256, 4 * 128) for r in K.kv8_read(codes, scales, 0, 256).view(4, 2, 256, 4, 128).transpose(2, 3)], c2, s2, 256)
        got = K.bridge_attn_decode8(q, c2, s2, kf, qf, ln, 128 ** -0.5)
    side.synchronize()
    assert torch.equal(got, want)                       # quantising what was read back changes nothing the attention sees


def test_one_row_of_any_stride(K):
    """A single row's stride says nothing (torch leaves any number there, 1 after a transpose): a batch of one takes every row it is given."""
    H, cap, D = 2, 32, 256
    odd = lambda x: torch.as_strided(x, x.shape, (1, 1))  # noqa: E731
    pair = [K.kv8_alloc(1, cap, H, "cuda", 16) for _ in range(2)]
    kf, qf, ln = torch.zeros(1, cap, dtype=torch.uint8, device="cuda"), torch.ones(1, dtype=torch.uint8, device="cuda"), torch.full((1,), 3, dtype=torch.int32, device="cuda")
    rows = [r.contiguous() for r in rows4(1, H, 21)]
    new = [r.contiguous() for r in rows4(1, H, 22)]
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    w, cos, sin, qkv, tb = [rnd(D, 8) for _ in range(4)], rnd(64, 128), rnd(64, 128), rnd(1, 3 * D), rnd(1, 16)
    outs = []
    for c, f in zip(pair, (lambda x: x, odd)):
        K.kv8_fill([f(r) for r in rows], *c, 1)
        K.kv8_append([f(r) for r in new], *c, torch.tensor([1], device="cuda"))
        x = qkv.clone()
        K.rope_bridge_pos_append8(f(x), f(tb), *w, qf, cos, sin, ln, H, *c, torch.tensor([2], device="cuda"))
        outs.append((x, K.bridge_attn_decode8(f(new[0]), *c, f(kf), qf, ln, 128 ** -0.5)))
    assert all(torch.equal(a, b) for a, b in zip(pair[0] + outs[0], pair[1] + outs[1]))


def attn_parts(K, B, H, cap, lens, seed):
    """Attention of a batch and of each of its sequences alone: (batch, alone, the tolerance of either against the definition)."""
    q, codes, scales, g = attn_case(K, B, H, cap, 16, seed)
    kf = (torch.rand(B, cap, generator=g) < 0.4).to(torch.uint8).cuda()
    qf = torch.tensor([i % 2 for i in range(B)], dtype=torch.uint8, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    whole = attn_check(K, q, codes, scales, kf, qf, ln, None)
    alone = torch.cat([attn_check(K, q[b:b + 1], codes[:, b:b + 1].contiguous(), scales[:, b:b + 1].contiguous(), kf[b:b + 1], qf[b:b + 1],
                                  ln[b:b + 1], None) for b in range(B)])
    return whole, alone


def test_a_sequence_alone_and_in_a_batch_under_one_plan(K):
    """Up to 1024 slots a (sequence, head) is one workgroup's whatever the batch: the same bits alone as in the batch."""
    whole, alone = attn_parts(K, 4, 4, 512, [512, 333, 64, 500], 8)
    assert torch.equal(whole, alone)
    whole, alone = attn_parts(K, 3, 2, 1024, [1024, 1, 700], 9)
    assert torch.equal(whole, alone)


def test_a_sequence_alone_and_in_a_batch_under_two_plans(K):
    """Larger caches split the keys of a small batch: alone a sequence's four heads take several workgroups each and the merge, in a batch of
    64 one each.  Another order of the same fp32 sums: both are within the definition's tolerance (attn_check), so within twice it of each
    other; the split is there to be crossed (other workspace sizes)."""
    B, H, cap = 64, 4, 1552
    L = K._lib.lib().libra_bridge_attn_decode8_workspace_bytes
    assert L(B, H, cap) == 0 and L(1, H, cap) > 0
    lens = [1552, 1537, 1536, 1025, 1024, 1023, 513, 512, 65, 64, 1, 0] + [37 * i % 1553 for i in range(52)]
    attn_parts(K, B, H, cap, lens, 10)
