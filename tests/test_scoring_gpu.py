"""LibraForCausalLM.token_logprobs (scoring with a gradient), output_logprobs of the generation loop, and generation over the 8-bit KV cache:
the operators as a user of the model calls them, together."""
import pytest
import torch

import logprobs_reference as R
from helpers import load_golden, rel_err, sub, sub_params
from test_f4_variants_gpu import _build, _oracle_logits
from test_logprobs_gpu import e_r, near, tol_lp

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _tiny():
    from libra_amd.libra import LibraConfig, LibraForCausalLM
    t, meta = load_golden("libra_tiny.safetensors")
    m = LibraForCausalLM(LibraConfig(**meta["cfg"]))
    m.load_state_dict(sub(t, "w."), strict=True)
    return m.to(BF).cuda(), sub_params(t, "w."), t, meta["cfg"], {}


def _model(name):
    if name == "default":
        return _tiny()
    m, w, t, t0, meta, over = _build(name)
    return m, w, t0, meta["cfg"], over


def _inputs(t):
    return dict(attention_mask=t["in.attention_mask"].cuda(), vision_indices=t["in.vision_indices"].cuda(),
                contiguous_signal=t["in.signal"].to(BF).cuda())


@pytest.mark.parametrize("name", ["default", "unified", "pred2d", "rope2d"])
def test_scores_are_those_of_the_models_logits(name):
    """Every number against the 64-bit definition on the model's own logits (same kernels, same bits), aligned to the token it is about."""
    m, _, t, c, over = _model(name)
    m.eval()
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    with torch.no_grad():
        z = m(input_ids=ids, **kw).logits.cpu().double()
        out = m.token_logprobs(ids, lab, top=4, **kw)
    Q, B, S, V = z.shape
    assert out.logprobs.shape == (Q, B, S) and out.top_ids.shape == (Q, B, S, 4) and not out.logprobs.requires_grad
    assert float(out.logprobs[:, :, 0].abs().max()) == 0 and bool((out.top_ids[:, :, 0] == -1).all())
    z2 = z[:, :, :-1].reshape(-1, V)
    lp, ent = R.logprobs(z2)
    tol = tol_lp(z2, lp)
    tgt = t["in.labels"][:, :, 1:].reshape(1, -1)
    near(out.logprobs[:, :, 1:].reshape(1, -1), R.pick(lp, tgt, 0), torch.gather(tol, 1, tgt.clamp_min(0).t()).t(), "logprobs")
    near(out.entropy[:, :, 1:].reshape(-1), torch.where(tgt[0] >= 0, ent, torch.zeros_like(ent)), 8 * e_r(V) * (ent + 1), "entropy")
    order = R.order(z2, 4)
    assert torch.equal(out.top_ids[:, :, 1:].reshape(-1, 4).cpu(), order)
    near(out.top_logprobs[:, :, 1:].reshape(-1, 4), torch.gather(lp, 1, order), torch.gather(tol, 1, order), "top_logprobs")
    # default labels: the ids where the mask allows and the row before can express them
    want = ids.masked_fill(kw["attention_mask"][None] == 0, -100)
    if name != "unified":
        vis = kw["vision_indices"] < c["max_vision_token_length"]
        for b in range(B):
            for s in range(1, S):
                for q in range(Q):
                    if bool(vis[b, s - 1]) != bool(ids[q, b, s] >= c["vocab_size"]):
                        want[q, b, s] = -100
    with torch.no_grad():
        own = m.token_logprobs(ids, **kw)
        assert torch.equal(own.logprobs, m.token_logprobs(ids, want, **kw).logprobs) and bool(torch.isfinite(own.logprobs).all())


def test_scoring_one_token():
    """A sequence of a single token: nothing predicts it."""
    m, _, t, c, _ = _model("default")
    m.requires_grad_(True)
    vi = torch.full((1, 1), c["max_vision_token_length"], device="cuda")
    sig = torch.zeros(1, 1, c["contiguous_signal_size"], dtype=BF, device="cuda")
    out = m.token_logprobs(torch.full((2, 1, 1), 7, device="cuda"), vision_indices=vi, contiguous_signal=sig, top=2)
    assert out.logprobs.tolist() == [[[0.0]], [[0.0]]] and out.top_ids.tolist() == [[[[-1, -1]]]] * 2
    out.logprobs.sum().backward()
    assert all(p.grad is None or not p.grad.any() for p in m.parameters())


@pytest.mark.parametrize("name", ["default", "unified", "pred2d"])
def test_gradient_vs_oracle_autograd(name):
    """sum(w logprobs) + sum(u entropy), w and u random a position, against autograd through the fp32 oracle on the same bf16 weights.
    Tolerance: the loss's own backward, a sum over positions with weights of ONE sign, is within 4e-2 of its largest element (bf16
    activations and gradients, 2 layers).  The backward is linear in the gradients it starts from, so this objective's gradient is the
    sum of four such one-signed parts, G = G(w > 0) + G(w < 0) + G(u > 0) + G(u < 0), and its error is at most the sum of theirs:
    4e-2 (max|G(w > 0)| + max|G(w < 0)| + max|G(u > 0)| + max|G(u < 0)|) - the parts cancel in G, their errors do not."""
    from oracle import libra_oracle as LO
    m, w, t, c, over = _model(name)
    m.requires_grad_(True)
    ids, lab = t["in.input_ids"].cuda(), t["in.labels"].cuda()
    g = torch.Generator().manual_seed(1)
    Q, B, S = lab.shape
    wt, ut = torch.randn(Q, B, S, generator=g) / 20, torch.randn(Q, B, S, generator=g) / 20
    out = m.token_logprobs(ids, lab, **_inputs(t))
    fin = torch.isfinite(out.logprobs)
    (torch.where(fin, out.logprobs, torch.zeros_like(out.logprobs)) * wt.cuda() + out.entropy * ut.cuda()).sum().backward()
    sdf = {k: v.to(BF).float().requires_grad_(True) for k, v in w.items()}
    kw = dict(layers=c["num_hidden_layers"], heads=c["num_attention_heads"], vocab=c["vocab_size"],
              max_vision_token_length=c["max_vision_token_length"], eps=c["rms_norm_eps"], max_pos=c["max_position_embeddings"])
    hid, flag = LO.model_forward(sdf, t["in.input_ids"], t["in.attention_mask"], t["in.vision_indices"], t["in.signal"].to(BF).float(), **kw)
    z = _oracle_logits(LO, sdf, hid, flag, over, c)[:, :, :-1]
    lp = torch.log_softmax(z, -1)
    tg = t["in.labels"][:, :, 1:]
    given = torch.gather(lp, -1, tg.clamp_min(0)[..., None])[..., 0]
    on = (tg >= 0) & torch.isfinite(given)
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    given, ent, wt, ut = torch.where(on, given, torch.zeros_like(given)), ent * (tg >= 0), wt[:, :, 1:], ut[:, :, 1:]
    names = [n for n in sdf]
    parts = [torch.autograd.grad(f.sum(), [sdf[n] for n in names], retain_graph=True, allow_unused=True) for f in (
        given * wt.clamp_min(0), given * wt.clamp_max(0), ent * ut.clamp_min(0), ent * ut.clamp_max(0))]
    n = 0
    params = dict(m.named_parameters())
    for i, nm in enumerate(names):
        gs = [p[i] for p in parts if p[i] is not None]
        reach = sum(float(x.abs().max()) for x in gs)
        if nm not in params or reach < 1e-6:
            continue
        got = params[nm].grad
        assert got is not None, nm
        err = float((got.float().cpu() - sum(gs)).abs().max())
        assert err <= 4e-2 * reach, (nm, err / reach)
        n += 1
    assert n > 50


def test_mean_negative_logprob_is_the_loss():
    """-mean log p over the labels == the fused loss, value (fp32 sums of the same terms) and gradients: the logits' gradients differ by
    at most a bf16 step each (2^-8) and each of ~10 later stages rounds to bf16 on either side: 2^-8 + 20 * 2^-9 < 5e-2 in norm; the same
    bits with gradient checkpointing; into captured gradient buckets too."""
    from libra_amd import dp
    m, _, t, c, _ = _model("default")
    m.requires_grad_(True)
    m.train()
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    loss = m(input_ids=ids, labels=lab, **kw).loss
    loss.backward()
    want = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    def mean_nll():
        lp = m.token_logprobs(ids, lab, **kw).logprobs
        return -sum(lp[q].sum() / (lab[q][:, 1:] >= 0).sum() for q in range(2)) / 2
    m.zero_grad()
    mine = mean_nll()
    assert abs(float(mine.detach()) - float(loss.detach())) <= 2.0 ** -18 * float(loss.detach())
    mine.backward()
    got = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    assert set(got) == set(want)
    for n in want:
        assert float((got[n].float() - want[n].float()).norm()) <= 5e-2 * float(want[n].float().norm()) + 1e-6, n
    m.gradient_checkpointing_enable()
    m.zero_grad()
    mean_nll().backward()
    assert all(torch.equal(p.grad, got[n]) for n, p in m.named_parameters() if p.grad is not None)
    m.gradient_checkpointing_disable()
    m.zero_grad()
    named = [(n, p) for n, p in m.named_parameters() if n in got]
    gb = dp.GradBuckets(named)
    with gb.capture():
        mean_nll().backward()
    for n, v in gb.finish().items():
        assert torch.equal(v, got[n]), n
    with pytest.raises(RuntimeError):                   # a second backward through the same graph
        out = m.token_logprobs(ids, lab, **kw).logprobs.sum()
        out.backward(retain_graph=True)
        out.backward()


def test_two_scorings_in_flight():
    """Two scoring graphs alive at once (a preferred and a rejected answer): one backward over both == the sum of two, up to the rounding of
    the bf16 gradients' sum (half a step, 2^-9 relative to the larger of sum and parts); the tokens scored twice agree bit for bit."""
    import warnings
    m, _, t, c, _ = _model("default")
    m.requires_grad_(True)
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    other = lab.masked_fill(lab < c["vocab_size"], -100)
    parts = []
    for l in (lab, other):
        m.zero_grad()
        out = m.token_logprobs(ids, l, **kw)
        (out.logprobs.sum() / 30 + out.entropy.sum() / 50).backward()
        parts.append({n: p.grad.float() for n, p in m.named_parameters() if p.grad is not None})
    m.zero_grad()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                 # (the second forward says that it allocates fresh buffers)
        a, b = m.token_logprobs(ids, lab, **kw), m.token_logprobs(ids, other, **kw)
    both = other >= 0
    assert torch.equal(a.logprobs[both], b.logprobs[both])
    ((a.logprobs.sum() / 30 + a.entropy.sum() / 50) + (b.logprobs.sum() / 30 + b.entropy.sum() / 50)).backward()
    for n, p in m.named_parameters():
        if p.grad is not None:
            x, y = parts[0][n], parts[1][n]
            assert bool(((p.grad.float() - (x + y)).abs() <= 2.0 ** -8 * torch.maximum((x + y).abs(), torch.maximum(x.abs(), y.abs())) + 1e-30).all()), n


def test_scoring_refusals():
    m, _, t, c, _ = _model("default")
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    for bad in (dict(labels=lab[:1]), dict(labels=lab.int()), dict(top=65), dict(top=-1), dict(vision_indices=None)):
        with pytest.raises(ValueError):
            m.token_logprobs(ids, **dict(kw, **bad))
    with pytest.raises(ValueError):
        m.token_logprobs(ids[:1], **kw)
    with pytest.raises(RuntimeError):
        m.token_logprobs(ids.cpu(), **kw)


# ---- generation ---------------------------------------------------------------------------------------------------------------
def _gen():
    from libra_amd.libra import LibraConfig, LibraForCausalLM
    t, meta = load_golden("libra_tiny_generate.safetensors")
    m = LibraForCausalLM(LibraConfig(**meta["cfg"]))
    m.load_state_dict(sub(load_golden("libra_tiny.safetensors")[0], "w."), strict=True)
    return m.to(BF).cuda().eval(), t, meta


def _gen_kw(t, meta):
    from libra_amd.libra.generation import ValidImageLogitsProcessor
    c = meta["cfg"]
    proc = ValidImageLogitsProcessor(meta["valid_image_token_length"], meta["boi"], meta["eoi"], c["vocab_size"], c["vocab_size"] + c["vision_vocab_size"])
    return dict(logits_processor=[proc], max_length=meta["prompt_len"] + meta["steps"], pad_token_id=meta["pad_token_id"],
                eos_token_id=meta["eos_token_id"], attention_mask=t["in.attention_mask"].cuda(), vision_indices=t["in.vision_indices"].cuda(),
                contiguous_signal=t["in.signal"].to(BF).cuda())


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("sampled", [False, True])
def test_generated_tokens_logprobs(dtype, sampled):
    m, t, meta = _gen()
    kw = dict(_gen_kw(t, meta), output_scores=True, return_dict_in_generate=True, output_logprobs=True, top_logprobs=3, cache_dtype=dtype)
    run = (lambda **k: m.sample(t["in.input_ids"].cuda(), generator=torch.Generator(device="cuda").manual_seed(3), **k)) if sampled else \
        (lambda **k: m.greedy_search(t["in.input_ids"].cuda(), **k))
    out = run(**kw)
    T = len(out.scores)
    Q, B = out.sequences.shape[:2]
    assert out.logprobs.shape == (Q, B, T) and out.top_ids.shape == (Q, B, T, 3)
    new = out.sequences[:, :, meta["prompt_len"]:]
    ended = torch.zeros(B, dtype=torch.bool, device="cuda")
    for s in range(T):
        z = out.scores[s].cpu().double()
        for q in range(Q):
            lp, ent = R.logprobs(z[q])
            given = torch.where(ended, torch.full_like(new[q, :, s], -100), new[q, :, s]).cpu()[None]
            near(out.logprobs[q, :, s][None], R.pick(lp, given, 0), torch.gather(tol_lp(z[q], lp), 1, given.clamp_min(0).t()).t(), "logprobs")
            near(out.entropy[q, :, s], torch.where(given[0] >= 0, ent, torch.zeros_like(ent)), 8 * e_r(z.shape[-1]) * (ent + 1), "entropy")
            assert torch.equal(out.top_ids[q, :, s].cpu(), R.order(z[q], 3))
            ended = ended | (new[q, :, s] == meta["eos_token_id"])
    if not sampled:                                     # the most likely id IS the greedy choice
        live = out.logprobs.abs() + out.entropy.abs() > 0
        assert torch.equal(out.top_ids[..., 0][live], new[live])
    plain = run(**{k: v for k, v in kw.items() if k not in ("output_logprobs", "top_logprobs")})
    assert torch.equal(plain.sequences, out.sequences) and plain.logprobs is None
    with pytest.raises(ValueError):
        run(**dict(kw, output_logprobs=False))


def _steps(m, t, meta, graphs, n=6, **cache):
    """Prefill and n steps of fixed tokens (an image, then text in row 0, text in row 1) -> logits of every call, the cache."""
    c = meta["cfg"]
    V, L = c["vocab_size"], c["max_vision_token_length"]
    m.decode_graphs = graphs
    kw = dict(attention_mask=t["in.attention_mask"].cuda(), vision_indices=t["in.vision_indices"].cuda(), contiguous_signal=t["in.signal"].to(BF).cuda())
    out = m(input_ids=t["in.input_ids"].cuda(), use_cache=True, max_cache_len=40, **cache, **kw)
    past, logits = out.past_key_values, [out.logits]
    for s in range(n):
        img = s < L - 2                                 # codes 1 ... L - 2 of an image, then text
        ids = torch.tensor([[[V + 3 + s if img else 7], [5 + s]], [[V + 7 + s if img else 7], [5 + s]]], device="cuda")
        vi = torch.tensor([[1 + s if img else L], [L]], device="cuda")
        logits.append(m(input_ids=ids, vision_indices=vi, past_key_values=past, use_cache=True).logits)
    m.decode_graphs = True
    return torch.cat(logits, 2).float().cpu(), past


@pytest.mark.parametrize("block", [1, 16, 64])
def test_fp8_cache_steps(block, monkeypatch):
    """Steps over the 8-bit cache: captured == launched kernel by kernel, bit for bit; equal - up to the attention output's rounding - to the
    same steps with the cache read back and the bf16 attention kernel over it; what the prompt left in the cache is within half an e4m3
    step of the exact rows."""
    from libra_amd import kernels as K
    m, t, meta = _gen()
    a, past = _steps(m, t, meta, True, cache_dtype="fp8", cache_block=block)
    b, _ = _steps(m, t, meta, False, cache_dtype="fp8", cache_block=block)
    key = lambda x: torch.nan_to_num(x, posinf=1e30, neginf=-1e30)  # noqa: E731
    assert torch.equal(key(a), key(b))
    assert past.dtype == "fp8" and past.length == meta["prompt_len"] + 6 and past.capacity == 40 and past.layers[0][0].shape[3] % block == 0

    def read_back(q, codes, scales, key_flag, query_flag, kv_len, scale, *, kv_start=None):
        rows = K.kv8_read(codes, scales, 0, codes.shape[3])
        return K.bridge_attn_decode(q, *rows, key_flag, query_flag, kv_len, codes.shape[2], scale, kv_start=kv_start)

    def apart(qkv, tb, bk_l, bk_v, bv_l, bv_v, flag, cos, sin, positions, H, codes, scales, slot):
        kc, vc = K.rope_bridge_pos(qkv, tb, bk_l, bk_v, bv_l, bv_v, flag, cos, sin, positions, H)
        K.kv8_append((qkv[:, H * 128:2 * H * 128], kc, qkv[:, 2 * H * 128:], vc), codes, scales, slot)
    monkeypatch.setattr(K, "bridge_attn_decode8", read_back)
    monkeypatch.setattr(K, "rope_bridge_pos_append8", apart)
    ref, _ = _steps(m, t, meta, False, cache_dtype="fp8", cache_block=block)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(a), fin) and rel_err(a[fin], ref[fin]) < 1e-2
    exact, past16 = _steps(m, t, meta, False)
    S = meta["prompt_len"]
    start = past16.start.tolist()
    for i in range(len(past.layers)):
        for x, y in zip(past16.rows(i, 0, S), past.rows(i, 0, S)):
            x, y = x.cpu().double(), y.cpu().double()
            for row in range(x.shape[0]):
                u, v = x[row, start[row]:], y[row, start[row]:]
                # the largest value of a block is at least 224 scales, so 2^-10 scale <= 2^-10 / 224 of the largest cached value; appended tokens may
                # have grown the last block's scale: twice that
                assert bool(((u - v).abs() <= torch.maximum(2.0 ** -4 * u.abs(), 2.0 ** -9 / 224 * 2 * x.abs().max())).all())
                assert not y[row, :start[row]].any()    # padding: zeros
    fin = torch.isfinite(exact)
    assert rel_err(a[fin], exact[fin]) < 0.2            # (the model's own sensitivity to cache rounding: informative, e4m3 is 2^-4)


def test_fp8_cache_reorder_and_limits():
    from libra_amd.libra import LibraForCausalLM
    m, t, meta = _gen()
    a, past = _steps(m, t, meta, True, n=2, cache_dtype="fp8")
    beam = torch.tensor([1, 0, 1], device="cuda")
    before = [r.clone() for r in past.rows(1)]
    LibraForCausalLM._reorder_cache(past, beam)
    assert past.B == 3 and all(torch.equal(x[beam], y) for x, y in zip(before, past.rows(1)))
    L = meta["cfg"]["max_vision_token_length"]
    ids = torch.full((2, 3, 1), 9, dtype=torch.long, device="cuda")
    z = m(input_ids=ids, vision_indices=torch.full((3, 1), L, device="cuda"), past_key_values=past, use_cache=True).logits
    assert torch.equal(z[:, 0], z[:, 2])
    bf, past16 = _steps(m, t, meta, True, n=2)
    m2 = past16.nbytes()
    _, p8 = _steps(m, t, meta, True, n=0, cache_dtype="fp8", cache_block=8)
    assert p8.nbytes() * 2 < m2 * 1.01 + 4 * sum(s.numel() for _, s in p8.layers)
    with pytest.raises(ValueError):
        p8.rows(0, 0, 99)
    for bad in (dict(cache_dtype="int4"), dict(cache_dtype="fp8", cache_block=3)):
        with pytest.raises(ValueError):
            _steps(m, t, meta, True, n=0, **bad)


@pytest.mark.parametrize("name", ["rope2d", "pred2d", "nobridge"])
def test_fp8_cache_with_variants(name):
    """The configurations whose steps take other positions / heads: fp8-cache logits near the bf16-cache ones (e4m3 noise), finite pattern equal."""
    m, w, t, t0, meta, over = _build(name)
    m.eval()
    ids, vi, sig = t0["in.input_ids"].cuda()[:, :1], t0["in.vision_indices"].cuda()[:1], t0["in.signal"].to(BF).cuda()[:1]
    S, P = ids.shape[2], 10
    res = []
    for dt in ("bf16", "fp8"):
        out = m(input_ids=ids[:, :, :P], vision_indices=vi[:, :P], contiguous_signal=sig[:, :P], use_cache=True, cache_dtype=dt)
        past, z = out.past_key_values, []
        for s in range(P, P + 3):
            z.append(m(input_ids=ids[:, :, s:s + 1], vision_indices=vi[:, s:s + 1], past_key_values=past, use_cache=True).logits.float().cpu())
        res.append(torch.cat(z, 2))
    fin = torch.isfinite(res[0])
    assert torch.equal(fin, torch.isfinite(res[1])) and rel_err(res[1][fin], res[0][fin]) < 0.2


def test_default_scores_do_not_depend_on_left_padding():
    """Row 0 of the generation fixture is left-padded by 4: the same tokens are scored as with the prompt alone, with the same values.  The two
    runs' logits agree within 1e-2 of their largest (the bound that the padded prompt's own test holds them to: other key tiles, bf16);
    log p = z_t - lse, and the entropy, a mean of such differences, move by at most twice that each (entropy: by its probabilities as well,
    which move by twice the logits' error relative, times the spread of log p, log V + the range of the logits)."""
    m, t, meta = _gen()
    ids, vi, sig, am = (t[f"in.{k}"].cuda() for k in ("input_ids", "vision_indices", "signal", "attention_mask"))
    sig = sig.to(BF)
    assert am[0].tolist()[:5] == [0, 0, 0, 0, 1]
    with torch.no_grad():
        z = m(input_ids=ids[:, :1, 4:], vision_indices=vi[:1, 4:], contiguous_signal=sig[:1, 4:]).logits.float()
        wide = m.token_logprobs(ids, attention_mask=am, vision_indices=vi, contiguous_signal=sig)
        alone = m.token_logprobs(ids[:, :1, 4:], vision_indices=vi[:1, 4:], contiguous_signal=sig[:1, 4:])
    d = 1e-2 * float(z[torch.isfinite(z)].abs().max())
    spread = float(torch.log(torch.tensor(float(z.shape[-1])))) + 2 * float(z[torch.isfinite(z)].abs().max())
    assert not wide.logprobs[:, 0, :5].any() and not wide.entropy[:, 0, :5].any()
    assert torch.equal(wide.logprobs[:, 0, 4:] != 0, alone.logprobs[:, 0] != 0) and int((alone.logprobs != 0).sum()) > 0
    assert float((wide.logprobs[:, 0, 4:] - alone.logprobs[:, 0]).abs().max()) <= 2 * d
    assert float((wide.entropy[:, 0, 4:] - alone.entropy[:, 0]).abs().max()) <= 2 * d + 2 * d * spread


def test_scoring_leaves_nothing_behind():
    """Call after call - backward over both outputs, over one, or none - the memory in use stays where it was, and the row arena is free again."""
    import gc
    m, _, t, c, _ = _model("default")
    m.requires_grad_(True)
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    gc.collect()                                        # (what earlier tests left in cycles)
    gc.disable()
    try:
        used = []
        for i in range(7):
            out = m.token_logprobs(ids, lab, top=2, **kw)
            if i % 3 < 2:
                (out.logprobs.sum() + (out.entropy.sum() if i % 3 == 0 else 0)).backward()
            del out
            m.zero_grad()
            assert m._packed.arena is None or not m._packed.arena.busy, i
            used.append(torch.cuda.memory_allocated())
        assert len(set(used[3:])) == 1, used            # (the first three bring the operands and the arena's buffers)
    finally:
        gc.enable()


def test_gradients_at_positions_that_are_not_scored_are_dropped():
    """sqrt(entropy) has an infinite derivative at the 0 of an unscored position: it belongs to a constant.  Bit for bit the gradient of the
    same sum over the scored positions alone."""
    m, _, t, c, _ = _model("default")
    m.requires_grad_(True)
    ids, lab, kw = t["in.input_ids"].cuda(), t["in.labels"].cuda(), _inputs(t)
    on = lab >= 0
    on[:, :, 0] = False
    assert bool(on.any()) and not bool(on[:, :, 1:].all())
    grads = []
    for every in (False, True):
        m.zero_grad()
        out = m.token_logprobs(ids, lab, **kw)
        (out.entropy if every else out.entropy[on]).sqrt().sum().backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys() and len(grads[0]) > 50
    for n, g in grads[0].items():
        assert bool(torch.isfinite(g).all()) and torch.equal(g, grads[1][n]), n
