"""Engines whose gated feed-forwards are kept in 8 bits: what is loaded, every feed-forward of their steps against the definition in 64 bits, replayed
steps and generation."""
import pytest
import torch

import helpers as H
import plain_fp8 as plain
import tiny_configs
import tiny_fovosun
import tiny_kuvonex
import tiny_nosedra
import tiny_pagonex

pytestmark = pytest.mark.gpu
MODELS = {"llama4 B": (tiny_configs, "B"), "llama4 D": (tiny_configs, "D"), "kuvonex even": (tiny_kuvonex, "even"), "kuvonex odd": (tiny_kuvonex, "odd"),
          "fovosun odd": (tiny_fovosun, "odd"), "fovosun even": (tiny_fovosun, "even"), "pagonex even": (tiny_pagonex, "even"), "nosedra even": (tiny_nosedra, "even")}


def _folder(tmp_path, which):
    from sharpinference_amd import load_config
    from sharpinference_amd.weights.loader import write_random_model
    module, name = MODELS[which]
    path = str(tmp_path / "model")
    write_random_model(load_config(module.CONFIGS[name]), path, module.SEEDS[name], std=0.1)
    return path


def _engine(path, **kw):
    return H.make_engine(path, "bfloat16", feed_forward="fp8", **kw)


def _parts(engine):
    from sharpinference_amd.parts.feedforward import DenseSwiGLU, MoESwiGLU
    found, seen = [], set()

    def walk(o):
        if id(o) in seen or isinstance(o, (torch.Tensor, str, int, float)) or o is None:
            return
        seen.add(id(o))
        if isinstance(o, (DenseSwiGLU, MoESwiGLU)):
            found.append(o)
        for v in (o.values() if isinstance(o, dict) else o if isinstance(o, (list, tuple)) else vars(o).values() if hasattr(o, "__dict__") else ()):
            walk(v)
    walk(engine.model)
    return found


@pytest.mark.parametrize("which", list(MODELS))
def test_feed_forwards_are_loaded_in_8_bits(tmp_path, which):
    """Each gated feed-forward without biases holds the quantised values of the matrices that a bfloat16 engine holds; the others are left."""
    from sharpinference_amd import ops
    path = _folder(tmp_path, which)
    few, whole = _parts(_engine(path)), _parts(H.make_engine(path, "bfloat16"))
    assert len(few) == len(whole) > 0
    kinds = set()
    for a, b in zip(few, whole):
        eight = isinstance(a.w_gate_up, ops.Fp8Weight)
        assert eight == (not getattr(b, "bias", False) and getattr(b, "gated", True))
        kinds.add(eight)
        if not eight:
            continue
        for name in ("w_gate_up", "w_down"):
            w = getattr(b, name)
            w = ops.unpack_weight(w) if isinstance(w, ops.PackedWeight) else w
            K, got = w.shape[-1], getattr(a, name)
            n = got.shape[0] if w.dim() == 3 else None
            want = plain.rows(w.reshape(-1, K)).view(w.shape)
            assert torch.equal(got.values().double()[:n], want[:n]) and (n is None or n >= a.E)
            if w.dim() == 3 and n == a.E + 1:      # the always-on expert: its own matrices
                own = getattr(b.shared, name)
                own = ops.unpack_weight(own) if isinstance(own, ops.PackedWeight) else own
                assert torch.equal(got.select(a.E).values().double(), plain.rows(own))
    assert kinds == ({False} if which.startswith("nosedra") else {True})


def _bounds(x, w1, w2, act, score, few):
    """(result, bound) of a feed-forward of quantised rows x, in 64 bits."""
    a, b = x @ w1.T, x.abs() @ w1.abs().T
    # few tokens: float sums of K exact products; more: what the matrix instruction may cut
    d = b * (x.shape[1] * 2.0 ** -24 if few else 2.0 ** -10)
    if score is not None:
        a, d = a * score[:, None], d * score[:, None].abs()
    (g, u), (dg, du) = a.chunk(2, 1), d.chunk(2, 1)
    limit = act[1] if isinstance(act, tuple) else None
    kind = {1: "silu", 2: "gelu_tanh"}.get(act, None) if limit is None else ("swish_clamp", limit)
    h = plain.unit(kind, g, u)
    one = plain.unit(kind, g, torch.zeros_like(u)) if limit is not None else plain.unit(kind, g, torch.ones_like(u))
    # the activations' slopes are at most 1.2, their values |g|; u (or its clamped form plus one) multiplies
    wide = (u.abs() + du + (1 if limit is not None else 0))
    dh = 1.2 * dg * wide + one.abs() * du + 2.0 ** -19 * (1 + g.abs()) * h.abs() + 1e-30
    q, dq = plain.hidden_rows(h, dh)
    y = q @ w2.T
    return y, plain.cut(q, w2) + dq @ w2.abs().T


class _Checked:
    """ops.feed_forward_fp8 and ops.experts_fp8 with every call checked."""

    def __init__(self, monkeypatch):
        from sharpinference_amd import ops
        self.real, self.calls = (ops.feed_forward_fp8, ops.experts_fp8), {"dense few": 0, "dense many": 0, "experts few": 0, "experts many": 0}
        monkeypatch.setattr(ops, "feed_forward_fp8", self.dense)
        monkeypatch.setattr(ops, "experts_fp8", self.experts)

    def dense(self, x, w1, w2, act=1):
        y = self.real[0](x, w1, w2, act)
        few = x.shape[0] <= 64
        self.calls["dense few" if few else "dense many"] += 1
        want, bound = _bounds(plain.rows(x), w1.values().double(), w2.values().double(), act, None, few)
        assert ((y.double() - want).abs() <= bound + plain.stored(want)).all()
        return y

    def experts(self, x, ids, wts, w1, w2, act=1, score_on_input=False, shared=False):
        y = self.real[1](x, ids, wts, w1, w2, act, score_on_input, shared)
        few = x.shape[0] <= 16
        self.calls["experts few" if few else "experts many"] += 1
        E, q = w1.shape[0] - (1 if shared else 0), plain.rows(x)
        want, bound = torch.zeros_like(y, dtype=torch.float64), torch.zeros_like(y, dtype=torch.float64)
        for e in range(E + (1 if shared else 0)):
            a, b = w1.select(e).values().double(), w2.select(e).values().double()
            for j in range(ids.shape[1] if e < E else 1):
                at = torch.nonzero(ids[:, j] == e).flatten() if e < E else torch.arange(x.shape[0], device=x.device)
                if at.numel():
                    s = wts[at, j].double() if e < E else None
                    v, d = _bounds(q[at], a, b, act, s if score_on_input else None, few)
                    f = s[:, None] if s is not None and not score_on_input else 1.0
                    want[at] += v * f
                    bound[at] += d * f
        assert ((y.double() - want).abs() <= bound + 2.0 ** -20 * want.abs() + plain.stored(want)).all()
        return y


@pytest.mark.parametrize("which", [m for m in MODELS if not m.startswith("nosedra")])
def test_every_feed_forward_of_a_trace_is_the_definitions(tmp_path, monkeypatch, which):
    checked = _Checked(monkeypatch)
    eng = _engine(_folder(tmp_path, which), decode_graphs=False, max_tokens_per_step=128)
    tokens = H.random_tokens(110, int(eng.config.vocab_size), 7)
    logits = H.run_cut(eng, "a", tokens, [90, 12, 1, 1, 1, 5])
    assert logits.isfinite().all()
    kinds = {k.split()[0] for k, n in checked.calls.items() if n}
    assert kinds and all(checked.calls[f"{k} few"] and checked.calls[f"{k} many"] for k in kinds)


@pytest.mark.parametrize("which", ["llama4 B", "kuvonex even", "fovosun even", "pagonex even"])
def test_replayed_steps_generate_what_eager_ones_do(tmp_path, which):
    path = _folder(tmp_path, which)
    eager, graphs = _engine(path, decode_graphs=False), _engine(path)
    vocab = int(eager.config.vocab_size)
    prompts = [H.random_tokens(n, vocab, n) for n in (5, 40, 1, 17)]
    for _ in range(2):
        want = [r.token_ids for r in eager.generate(prompts, max_new_tokens=24, temperature=0.0, stop_token_ids=())]
        got = [r.token_ids for r in graphs.generate(prompts, max_new_tokens=24, temperature=0.0, stop_token_ids=())]
        assert got == want and all(len(t) == 24 for t in got)
