"""LibraForCausalLM.token_logprobs without a GPU: which positions its default labels score, with the autograd node replaced by a recorder
(host tensors that call themselves device tensors)."""
import gc
import types
import weakref

import pytest
import torch

from helpers import load_golden
from libra_amd.libra import LibraConfig, LibraForCausalLM
from libra_amd.libra import modeling_libra as M


class Device(torch.Tensor):
    """A host tensor that passes the entry point's device check."""
    is_cuda = True


def _default_labels(monkeypatch, unified, mask, vision_indices, ids):
    _, meta = load_golden("libra_tiny.safetensors")
    m = LibraForCausalLM(LibraConfig(**dict(meta["cfg"], unified_head=unified)))
    seen = {}

    def record(model, holder, names, input_ids, attention_mask, vision_indices, signal, labels, top, *params):
        seen["labels"] = labels
        holder.update(top_ids=None, top_logprobs=None)
        return None, None
    monkeypatch.setattr(M._LibraScoreFunction, "apply", staticmethod(record))
    m.token_logprobs(ids.as_subclass(Device), attention_mask=mask, vision_indices=vision_indices)
    return seen["labels"].as_subclass(torch.Tensor), m


@pytest.mark.parametrize("unified", [False, True])
@pytest.mark.parametrize("kind", [torch.bool, torch.int64])
def test_default_labels_leave_out_what_a_padding_row_would_predict(monkeypatch, unified, kind):
    """Row t - 1 predicts token t: the first token behind left padding is predicted by nothing, like the token at position 0."""
    _, meta = load_golden("libra_tiny.safetensors")
    L, S = meta["cfg"]["max_vision_token_length"], 6
    mask = torch.tensor([[0, 0, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1], [1, 1, 1, 0, 0, 0], [0, 0, 0, 0, 0, 1]]).to(kind)
    ids = torch.arange(5, 5 + 4 * S).view(1, 4, S).repeat(2, 1, 1)
    labels, _ = _default_labels(monkeypatch, unified, mask, torch.full((4, S), L), ids)
    scored = labels >= 0
    first = [2, 0, 0, 5]
    for b in range(4):
        for s in range(S):
            # (position 0 has a label with either head, and scoring answers 0 there: nothing predicts it)
            want = s == 0 if s == first[b] else bool(mask[b, s])
            assert scored[:, b, s].tolist() == [want] * 2, (b, s)
    assert torch.equal(labels[scored], ids[scored])


@pytest.mark.parametrize("pad", [1, 3])
def test_default_labels_do_not_depend_on_the_padding(monkeypatch, pad):
    """An image and text, alone and left-padded: the same tokens are scored."""
    _, meta = load_golden("libra_tiny.safetensors")
    L, V = meta["cfg"]["max_vision_token_length"], meta["cfg"]["vocab_size"]
    ids = torch.tensor([3, V + 1, V + 2, V + 4, 9, 8])[None, None].repeat(2, 1, 1)
    vi = torch.tensor([[L, 0, 1, L - 1, L, L]])
    alone, _ = _default_labels(monkeypatch, False, torch.ones(1, 6, dtype=torch.bool), vi, ids)
    wide = lambda x, v: torch.nn.functional.pad(x, (pad, 0), value=v)  # noqa: E731
    padded, _ = _default_labels(monkeypatch, False, wide(torch.ones(1, 6), 0) > 0, wide(vi, L), wide(ids, 0))
    assert torch.equal(padded[:, :, pad + 1:], alone[:, :, 1:]) and bool((padded[:, :, :pad + 1] < 0).all())


class _State:
    pass


class _Engine:
    """Stands in for the decoder engine: a forward whose saved state is one object that can be watched."""

    def __init__(self, monkeypatch):
        self.alive = []
        monkeypatch.setattr(M.DE, "forward", self.forward)
        monkeypatch.setattr(M.DE, "backward", lambda sd, packed, dims, out, want, g_scores: {
            n: g_scores[0].sum() + 2 * g_scores[1].sum() + torch.zeros(3) for n in want if out["saved"]["x"]})
        self.model = types.SimpleNamespace(_refresh_packed=lambda sd: None, _dims=None, _packed=None, training=True,
                                           model=types.SimpleNamespace(gradient_checkpointing=False))

    def forward(self, sd, packed, dims, ids, mask, vi, signal, labels, *, save, recompute, score):
        state = _State()
        self.alive.append(weakref.ref(state))
        scores = dict(logprobs=torch.zeros(2, 1, 4), entropy=torch.zeros(2, 1, 4), top_ids=torch.zeros(2, 1, 4, 0), top_logprobs=torch.zeros(2, 1, 4, 0),
                      parts=[state], scored=torch.ones(2, 4))
        return dict(scores=scores, z_lang=state, saved=dict(scores=scores, x=[state]) if save else None)

    def call(self, p, grad_on=True):
        return M._LibraScoreFunction.apply(self.model, dict(grad_on=grad_on), ["w"], None, None, None, None, None, 0, p)


@pytest.mark.parametrize("mode", ["both", "logprobs", "entropy", "dropped", "not saved"])
def test_a_scoring_call_is_freed_with_its_outputs(monkeypatch, mode):
    """Nothing of a call outlives its outputs, without the collector's help: activations (and with them the row arena's lease) go at once."""
    e = _Engine(monkeypatch)
    p = torch.nn.Parameter(torch.zeros(3))
    gc.disable()
    try:
        for _ in range(3):
            lp, ent = e.call(p, mode != "not saved")
            if mode == "both":
                (lp.sum() + ent.sum()).backward()
            elif mode in ("logprobs", "entropy"):
                (lp if mode == "logprobs" else ent).sum().backward()
            del lp, ent
            assert [r() for r in e.alive] == [None] * len(e.alive)
    finally:
        gc.enable()
    assert (p.grad is None) == (mode in ("dropped", "not saved"))


def test_a_backward_frees_the_call_and_is_the_only_one(monkeypatch):
    e = _Engine(monkeypatch)
    p = torch.nn.Parameter(torch.zeros(3))
    lp, ent = e.call(p)
    both = lp.sum() + ent.sum()
    both.backward(retain_graph=True)
    assert e.alive[0]() is None and p.grad.tolist() == [24.0] * 3          # (lp and ent are still held)
    with pytest.raises(RuntimeError, match="ran already"):
        both.backward()


def test_rows_that_are_not_scored_answer_zero_whatever_they_hold(monkeypatch):
    """A row whose logits are not finite and whose token is not scored: 0, not 0 * NaN."""
    from libra_amd import kernels as K
    monkeypatch.setattr(M.DE.K, "token_logprobs", lambda z, t, *, target_sub, top: K.TokenLogprobs(
        torch.zeros(t.shape), torch.stack([z.amax(-1), z.sum(-1), z.mean(-1)]), (torch.zeros(len(z), top, dtype=torch.int64), torch.zeros(len(z), top))))
    z = torch.tensor([[1.0, 3.0], [float("nan"), 0.0], [float("inf"), 0.0], [2.0, 4.0]])
    labels = torch.tensor([[[0, 1, -100, -1]], [[0, -100, -100, 1]]])                  # the rows of tokens 0 .. 2 predict 1 .. 3
    d = types.SimpleNamespace(vocab=2)
    out = M.DE.score_heads(d, labels, z, [None, None], None, torch.arange(4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), 1)
    assert out["entropy"].tolist() == [[[0.0, 2.0, 0.0, 0.0]], [[0.0, 0.0, 0.0, float("inf")]]]
