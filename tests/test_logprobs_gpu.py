"""Log probabilities of given tokens, entropy, alternatives and their gradient on the device against the 64-bit definition.

Tolerances.  z - m is rounded once (2^-24 |z - m|); exp of it is then off by that much plus 2^-22 relative; the sum r of the columns beside
the largest is a sum of positive terms in at most V / 256 + 16 steps: relative error e_r = 2^-21 + D 2^-23 + (V / 256 + 16) 2^-24, with D =
the largest |z - m| that still counts (p > 2^-40: 28).  log p = (z - m) - log1p(r): off by 2^-23 (|z - m| + log1p(r)) + e_r min(1, r).
Entropy: log1p(r) and the weighted mean of |z - m| each to e_r relative.  p = exp(log p): relative error e_p = the error of log p + 2^-22.
The gradient's terms are products with p: |dz| off by e_p times the sum of the terms' sizes, and half a step of the logits' type at the end."""
import pytest
import torch

import logprobs_reference as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def K():
    from libra_amd import kernels
    return kernels


def e_r(V):
    return 2.0 ** -21 + 28 * 2.0 ** -23 + (V / 256 + 16) * 2.0 ** -24


def tol_lp(z, lp):
    """tolerance of log p [rows, V]"""
    m = z.amax(-1, keepdim=True)
    d = torch.nan_to_num((z - m).abs(), nan=0.0, posinf=0.0)
    lsum = torch.nan_to_num(-lp.amax(-1, keepdim=True), nan=0.0, posinf=0.0)
    return 2.0 ** -23 * (d + lsum) + e_r(z.shape[1]) * torch.expm1(lsum).clamp(max=1.0)


def near(got, want, tol, what):
    got, want = got.cpu().double(), want.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    err = (got - want).abs()[fin]
    bad = err > tol.expand_as(want)[fin]
    assert not bool(bad.any()), (what, float((err / tol.expand_as(want)[fin].clamp_min(1e-300)).max()))


def check(K, z, targets, sub, top):
    out = K.token_logprobs(z, targets, target_sub=sub, top=top)
    z64, t = z.cpu().double(), targets.cpu()
    lp, ent = R.logprobs(z64)
    tol = tol_lp(z64, lp)
    at = (t.clamp_min(0) - sub).clamp(0, z64.shape[1] - 1)
    near(out.logprobs, R.pick(lp, t, sub), torch.gather(tol, 1, at.t()).t(), "logprobs")
    d = torch.nan_to_num((z64 - z64.amax(-1, keepdim=True)).abs(), nan=0.0, posinf=0.0)
    p = torch.nan_to_num(torch.exp(lp))
    lsum = torch.nan_to_num(-lp.amax(-1), nan=0.0, posinf=0.0)
    near(out.entropy, ent, 2 * e_r(z64.shape[1]) * (lsum + (p * d).sum(-1)) + 2.0 ** -22 * ent.abs().nan_to_num(), "entropy")
    near(out.lse, torch.where(torch.isnan(ent), ent, torch.logsumexp(z64, -1)), 2.0 ** -23 * (z64.amax(-1).abs().nan_to_num(posinf=0.0, neginf=0.0) + lsum) + e_r(z64.shape[1]), "lse")
    ids = R.order(z64, top)
    assert torch.equal(out.top_ids.cpu(), ids + sub)
    near(out.top_logprobs, torch.gather(lp, 1, ids), torch.gather(tol, 1, ids), "top_logprobs")
    return out


def logits(rows, V, seed, dtype, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = spread * torch.randn(rows, V, generator=g)
    t = torch.randint(0, V, (2, rows), generator=g)
    z[torch.arange(rows), t[0]] += torch.where(torch.rand(rows, generator=g) < 0.5, 12.0, 0.0)
    t[torch.rand(2, rows, generator=g) < 0.15] = -100
    return z.to(dtype).cuda(), t.cuda()


SHAPES = [(1, 1, 1), (3, 2, 2), (2, 7, 5), (5, 8, 8), (4, 64, 20), (7, 513, 20), (3, 514, 64), (2, 2048, 3), (2, 2049, 20), (3, 4097, 1), (2, 32000, 20),
          (3, 32514, 64), (2, 40001, 7), (1, 70003, 5)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V,top", SHAPES)
def test_forward(K, rows, V, top, dtype):
    z, t = logits(rows, V, rows + V, dtype)
    check(K, z, t, 0, top)
    check(K, z, t[:1].contiguous(), 0, 0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [9, 514, 32514, 70003])
def test_masked_and_forced_rows(K, V, dtype):
    """Columns masked with -inf, with the type's lowest value, rows with one or no column left, forced rows, NaN."""
    z, t = logits(12, V, 3, dtype)
    inf = float("inf")
    z[0, V // 2:] = -inf
    z[1, :V // 2] = -inf
    z[2] = -inf
    z[2, 5] = 1.5                                       # one column left
    z[3] = -inf                                         # none
    z[4] = -inf
    z[4, 7] = inf                                       # forced
    z[5, 2] = inf
    z[5, 8] = inf                                       # two share
    z[6] = inf
    z[7, 3] = float("nan")
    z[8, ::2] = torch.finfo(dtype).min
    z[9] = torch.finfo(dtype).min
    z[10] = 0.25                                        # all equal
    z[11, 1:] = -inf
    z[11, 0] = float("nan")
    t[0, 4], t[1, 4], t[0, 2], t[0, 3], t[1, 7], t[0, 5] = 7, 1, 5, 0, 0, 8
    top = min(V, 20)
    out = check(K, z, t, 0, top)
    assert out.top_ids[3].tolist() == list(range(top)) and out.top_ids[10].tolist() == list(range(top))       # ties: the smaller column
    g = torch.Generator().manual_seed(1)
    g_lp, g_ent = torch.randn(2, 12, generator=g).cuda(), torch.randn(12, generator=g).cuda()
    dz = K.token_logprobs_bwd(z, t, out.stats, g_lp, g_ent).float().cpu()
    assert not dz[[3, 4, 5, 6]].any() and bool(torch.isnan(dz[7]).all()) and bool(torch.isnan(dz[11]).all())
    keep = [0, 1, 2, 8, 9, 10]
    grad_check(z[keep], t[:, keep], 0, g_lp[:, keep], g_ent[keep], dz[keep])


def grad_check(z, t, sub, g_lp, g_ent, dz):
    z64 = z.cpu().double()
    want = R.gradient(z64, t.cpu(), sub, g_lp.cpu().double(), g_ent.cpu().double())
    lp, ent = R.logprobs(z64)
    p = torch.exp(lp)
    g = (g_lp.cpu().double().abs() * (t.cpu() >= 0)).sum(0)[:, None]
    # z - m - log_sum from fp32 stats: one more rounding of the row's own numbers
    e_p = tol_lp(z64, lp).nan_to_num() + 2.0 ** -23 * lp.abs().nan_to_num(posinf=0.0) + 2.0 ** -21
    size = p * (g + g_ent.cpu().double().abs()[:, None] * (torch.where(p > 0, lp.abs(), torch.zeros_like(p)) + ent[:, None] + 1))
    tol = e_p * size + (torch.finfo(z.dtype).eps / 2) * want.abs() + 2.0 ** -126
    hit = torch.zeros_like(p)
    for i in range(t.shape[0]):
        for r in range(z.shape[0]):
            v = int(t[i, r]) - sub
            if int(t[i, r]) >= 0 and 0 <= v < z.shape[1]:
                hit[r, v] += abs(float(g_lp[i, r]))
    one = torch.where(hit > 0, -torch.expm1(lp), torch.zeros_like(lp))
    tol = tol + hit * (one * 2.0 ** -21 + e_p * p)      # 1 - p of a given token, as -expm1(log p)
    near(dz, want, tol, "dlogits")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 13), (4, 514), (2, 2049), (3, 32000), (2, 32514), (2, 40001)])
def test_backward(K, rows, V, dtype):
    z, t = logits(rows, V, 7 * rows + V, dtype)
    if rows > 2:
        t[1, 2] = t[0, 2] = 1                           # the same token twice
    g = torch.Generator().manual_seed(V)
    g_lp, g_ent = torch.randn(2, rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    out = K.token_logprobs(z, t)
    grad_check(z, t, 0, g_lp, g_ent, K.token_logprobs_bwd(z, t, out.stats, g_lp, g_ent))
    grad_check(z, t, 0, g_lp, torch.zeros_like(g_ent), K.token_logprobs_bwd(z, t, out.stats, g_lp))
    grad_check(z, t, 0, torch.zeros_like(g_lp), g_ent, K.token_logprobs_bwd(z, t, out.stats, None, g_ent))
    w = z.clone()
    K.token_logprobs_bwd(w, t, out.stats, g_lp, g_ent, out=w)          # in place
    assert torch.equal(w, K.token_logprobs_bwd(z, t, out.stats, g_lp, g_ent))


def test_backward_against_differences(K):
    """Central differences of the 64-bit definition along random directions against the fp32 gradient."""
    z, t = logits(6, 97, 5, F32)
    g = torch.Generator().manual_seed(2)
    g_lp, g_ent = torch.randn(2, 6, generator=g), torch.randn(6, generator=g)
    dz = K.token_logprobs_bwd(z, t, K.token_logprobs(z, t).stats, g_lp.cuda(), g_ent.cuda()).cpu().double()

    def f(x):
        lp, ent = R.logprobs(x)
        return (R.pick(lp, t.cpu(), 0) * g_lp.double()).sum() + (ent * g_ent.double()).sum()
    for seed in range(5):
        u = torch.randn(6, 97, generator=g, dtype=torch.float64)
        h = 1e-5
        num = (f(z.cpu().double() + h * u) - f(z.cpu().double() - h * u)) / (2 * h)
        # differences: h^2 of a third derivative of order 10; the gradient: 97 * 6 terms of fp32
        assert abs(float((dz * u).sum() - num)) <= 1e-8 * 10 + 2.0 ** -18 * float((dz * u).abs().sum())


def test_nearly_certain_token(K):
    """log p of a token that is nearly certain keeps its relative precision (log1p of the others), and so does its gradient."""
    V = 1000
    z = torch.zeros(5, V)
    lead = torch.tensor([10.0, 16.0, 20.0, 30.0, 60.0])
    z[:, 3] = lead
    t = torch.full((1, 5), 3)
    zc, tc = z.cuda(), t.cuda()
    out = K.token_logprobs(zc, tc, top=2)
    want = -torch.log1p((V - 1) * torch.exp(-lead.double()))
    assert bool(((out.logprobs[0].cpu().double() - want).abs() <= 2.0 ** -18 * want.abs()).all())
    assert bool(((out.top_logprobs[:, 0].cpu().double() - want).abs() <= 2.0 ** -18 * want.abs()).all())
    dz = K.token_logprobs_bwd(zc, tc, out.stats, torch.ones(1, 5, device="cuda"))
    one = -torch.expm1(want)
    assert bool(((dz[:, 3].cpu().double() - one).abs() <= 2.0 ** -17 * one).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_and_offsets(K, dtype):
    """Row strides and starts at every alignment, a head's slice of a wider buffer, ids with an offset, targets outside the head."""
    wide, _ = logits(5, 1100, 9, dtype)
    for col in (0, 1, 2, 3, 5, 8):
        for V in (514, 511, 16, 1):
            z = wide[:, col:col + V]
            t = torch.tensor([[32000, 32000 + V - 1, 31999, 32000 + V, -1], [32000, -100, 32000, 7, 32000]], device="cuda")
            out = check(K, z, t, 32000, min(V, 4))
            g_lp, g_ent = torch.linspace(-1, 1, 10).view(2, 5).cuda(), torch.linspace(0.5, 1, 5).cuda()
            buf = torch.full((5, 700), 9.0, dtype=dtype, device="cuda")
            dz = K.token_logprobs_bwd(z, t, out.stats, g_lp, g_ent, target_sub=32000, out=buf[:, 3:3 + V])
            grad_check(z, t, 32000, g_lp, g_ent, dz)
            assert bool((buf[:, :3] == 9).all()) and bool((buf[:, 3 + V:] == 9).all())                # nothing beside it is touched


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_of_targets_below_the_head(K, dtype):
    """Tokens whose column is negative, among them whole multiples of what a workgroup reads at a time: each counts with its -p, no column is
    theirs, and the columns of the other given tokens are as ever."""
    V, sub = 2100, 32000
    z, _ = logits(6, V, 17, dtype)
    t = torch.tensor([[sub - 1, sub - 256, sub - 512, sub - 1024, sub - 2048, 0], [sub, sub + 5, -1, sub - 8, sub + V - 1, sub + 300]], device="cuda")
    g = torch.Generator().manual_seed(6)
    g_lp, g_ent = torch.randn(2, 6, generator=g).cuda(), torch.randn(6, generator=g).cuda()
    for w in (V, 514):
        zw, tw = z[:, :w], t if w == V else t.where(t < sub + w, sub + w - 1)
        out = check(K, zw, tw, sub, 3)
        grad_check(zw, tw, sub, g_lp, g_ent, K.token_logprobs_bwd(zw, tw, out.stats, g_lp, g_ent, target_sub=sub))


def test_many_targets_and_empty_calls(K):
    z, _ = logits(3, 50, 1, BF)
    t = torch.randint(0, 50, (64, 3), generator=torch.Generator().manual_seed(0)).cuda()
    check(K, z, t, 0, 50)
    out = K.token_logprobs(z, t[:0])
    assert out.logprobs.shape == (0, 3) and bool(torch.isfinite(out.entropy).all())
    out = K.token_logprobs(z[:0], t[:, :0].contiguous(), top=3)
    assert out.top_ids.shape == (0, 3)
    assert K.token_logprobs_bwd(z[:0], t[:, :0].contiguous(), out.stats, None).shape == (0, 50)


def test_more_rows_than_a_launch(K):
    """2^21 rows a launch: the rows behind that limit, an odd number of them."""
    rows, V = (1 << 21) + 7, 12
    z = torch.zeros(rows, V, dtype=BF, device="cuda")
    tail, t2 = logits(9, V, 3, BF)
    z[-9:] = tail
    t = torch.zeros((2, rows), dtype=torch.int64, device="cuda")
    t[:, -9:] = t2
    out = K.token_logprobs(z, t, top=2)
    want = check(K, tail, t2, 0, 2)
    assert torch.equal(out.logprobs[:, -9:], want.logprobs) and torch.equal(out.top_ids[-9:], want.top_ids)
    assert bool((out.stats[1, :-9] == out.stats[1, 0]).all())
    g = torch.ones(2, rows, device="cuda")
    dz = K.token_logprobs_bwd(z, t, out.stats, g)
    assert torch.equal(dz[-9:], K.token_logprobs_bwd(tail, t2, want.stats, g[:, :9].contiguous())) and torch.equal(dz[0], dz[rows - 10])


def test_one_row_of_a_column(K):
    """A single row whose stride says nothing (as a transposed column has)."""
    z, t = logits(1, 50, 4, BF)
    col = z.view(-1).as_strided((1, 50), (1, 1))
    assert col.stride(0) == 1
    assert torch.equal(check(K, col, t, 0, 5).logprobs, check(K, z, t, 0, 5).logprobs)


def test_refusals(K):
    z, t = logits(3, 50, 1, BF)
    for bad in (lambda: K.token_logprobs(z, t, top=51), lambda: K.token_logprobs(z, t, top=-1), lambda: K.token_logprobs(z.half(), t),
                lambda: K.token_logprobs(z, t[0]), lambda: K.token_logprobs(z, t.int()), lambda: K.token_logprobs(z.t()[:3], t),
                lambda: K.token_logprobs(z, t.cpu()), lambda: K.token_logprobs(z, torch.zeros(65, 3, dtype=torch.int64, device="cuda")),
                lambda: K.token_logprobs_bwd(z, t, torch.zeros(3, 3, dtype=torch.float64, device="cuda"), None),
                lambda: K.token_logprobs_bwd(z, t, torch.zeros(3, 3, device="cuda"), torch.zeros(1, 3, device="cuda")),
                lambda: K.token_logprobs_bwd(z, t, torch.zeros(3, 3, device="cuda"), None, out=z[:, :49])):
        with pytest.raises(ValueError):
            bad()


def test_offsets_past_32_bits(K):
    """More than 2^32 elements: the last rows are right."""
    rows, V = 135000, 32000
    z = torch.zeros(rows, V, dtype=BF, device="cuda")
    tail, t2 = logits(4, V, 11, BF)
    z[-4:] = tail
    t = torch.full((2, rows), -100, dtype=torch.int64, device="cuda")
    t[:, -4:] = t2
    a, b = K.token_logprobs(z, t, top=3), K.token_logprobs(tail, t2, top=3)
    assert torch.equal(a.logprobs[:, -4:], b.logprobs) and torch.equal(a.stats[:, -4:], b.stats) and torch.equal(a.top_ids[-4:], b.top_ids)
    g_lp = torch.ones(2, rows, device="cuda")
    g_ent = torch.ones(rows, device="cuda")
    K.token_logprobs_bwd(z, t, a.stats, g_lp, g_ent, out=z)
    assert torch.equal(z[-4:], K.token_logprobs_bwd(tail, t2, b.stats, g_lp[:, :4].contiguous(), g_ent[:4]))


def test_deterministic_stream_and_graph(K):
    z, t = logits(33, 514, 2, BF)
    g_lp, g_ent = torch.ones(2, 33, device="cuda"), torch.ones(33, device="cuda")

    def both():
        o = K.token_logprobs(z, t, top=5)
        return o, K.token_logprobs_bwd(z, t, o.stats, g_lp, g_ent)
    first, d0 = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, d = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, o)) and torch.equal(d0, d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, d = both()
    for seed in (2, 3, 4):
        z2, t2 = logits(33, 514, seed, BF)
        z.copy_(z2); t.copy_(t2)
        want, dw = both()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, o)) and torch.equal(dw, d), seed
