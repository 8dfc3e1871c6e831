"""GPU: beam search end to end (TextDecoder.generate_beam: the paged operators
run together, eagerly and as a captured step) against a 64-bit beam search
that recomputes every hypothesis from its ids, without any cache."""

from __future__ import annotations

import math

import pytest
import torch

import vlasr
from vlasr.decoder import TextDecoder

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HD, FFN, LAYERS, VOCAB = 512, 4, 2, 128, 512, 2, 640
AUDIO_ID, EOS = 639, (7, 8)
AUDIO_ROWS = 9
PROMPT = [1, 2] + [AUDIO_ID] * AUDIO_ROWS + [3, 4, 5]


def make_weights(seed):
    g = torch.Generator().manual_seed(seed)

    def w(*shape, std):
        return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)

    p = "language_model.model."
    out = {p + "embed_tokens.weight": w(VOCAB, HIDDEN, std=1.0),
           "language_model.lm_head.weight": w(VOCAB, HIDDEN, std=0.09),
           p + "norm.weight": (1 + w(HIDDEN, std=0.02)).to(torch.bfloat16)}
    for l in range(LAYERS):
        q = f"{p}layers.{l}."
        out[q + "input_layernorm.weight"] = (1 + w(HIDDEN, std=0.02)).to(torch.bfloat16)
        out[q + "post_attention_layernorm.weight"] = (1 + w(HIDDEN, std=0.02)).to(torch.bfloat16)
        for n, rows in (("q", HEADS * HD), ("k", KV * HD), ("v", KV * HD), ("o", HIDDEN)):
            cols = HEADS * HD if n == "o" else HIDDEN
            out[q + f"self_attn.{n}_proj.weight"] = w(rows, cols, std=0.05)
        out[q + "mlp.gate_proj.weight"] = w(FFN, HIDDEN, std=0.04)
        out[q + "mlp.up_proj.weight"] = w(FFN, HIDDEN, std=0.04)
        out[q + "mlp.down_proj.weight"] = w(HIDDEN, FFN, std=0.04)
    return out


class Plain:
    """The model in 64 bits: log-probabilities after a prompt and ids."""

    def __init__(self, weights, audio):
        self.w = {k: v.double() for k, v in weights.items()}
        self.audio = audio.double().cpu()

    def rms(self, x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w

    def rope(self, x):
        pos = torch.arange(x.shape[0], dtype=torch.float64)
        f = 10000.0 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)
        a = pos[:, None, None] * f
        lo, hi = x[..., :HD // 2], x[..., HD // 2:]
        return torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1)

    def log_probs(self, chunk, ids):
        w, p = self.w, "language_model.model."
        h = w[p + "embed_tokens.weight"][torch.tensor(PROMPT + list(ids))].clone()
        at = [i for i, t in enumerate(PROMPT) if t == AUDIO_ID]
        h[at] = self.audio[chunk]
        n = h.shape[0]
        mask = torch.full((n, n), -math.inf, dtype=torch.float64).triu(1)
        for l in range(LAYERS):
            q = f"{p}layers.{l}."
            y = self.rms(h, w[q + "input_layernorm.weight"])
            qh = self.rope((y @ w[q + "self_attn.q_proj.weight"].T).view(n, HEADS, HD))
            kh = self.rope((y @ w[q + "self_attn.k_proj.weight"].T).view(n, KV, HD))
            vh = (y @ w[q + "self_attn.v_proj.weight"].T).view(n, KV, HD)
            kh, vh = (t.repeat_interleave(HEADS // KV, 1) for t in (kh, vh))
            s = torch.einsum("ihd,jhd->hij", qh, kh) / math.sqrt(HD) + mask
            a = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vh).reshape(n, -1)
            h = h + a @ w[q + "self_attn.o_proj.weight"].T
            y = self.rms(h, w[q + "post_attention_layernorm.weight"])
            g = torch.nn.functional.silu(y @ w[q + "mlp.gate_proj.weight"].T)
            h = h + (g * (y @ w[q + "mlp.up_proj.weight"].T)) @ w[q + "mlp.down_proj.weight"].T
        x = self.rms(h[-1], w[p + "norm.weight"])
        return torch.log_softmax(w["language_model.lm_head.weight"] @ x, -1)

    def score(self, chunk, ids):
        return sum(float(self.log_probs(chunk, ids[:i])[t]) for i, t in enumerate(ids))

    def search(self, chunk, beams, steps):
        live = [(0.0, [])]
        for _ in range(steps):
            found = []
            for s, ids in live:
                if ids and ids[-1] in EOS:
                    found.append((s, ids))
                    continue
                lp = self.log_probs(chunk, ids)
                top = torch.topk(lp, beams)
                found += [(s + float(v), ids + [int(t)]) for v, t in zip(*top)]
            live = sorted(found, key=lambda x: -x[0])[:beams]
        return live


@pytest.fixture(scope="module")
def model(dev):
    weights = make_weights(3)
    g = torch.Generator().manual_seed(4)
    audio = torch.randn(3, AUDIO_ROWS, HIDDEN, generator=g).to(torch.bfloat16)
    dec = TextDecoder({k: v.to(dev) for k, v in weights.items()}, heads=HEADS, kv_heads=KV,
                      dtype=torch.bfloat16, max_seq_len=128, audio_token_id=AUDIO_ID, eos_ids=EOS)
    return dec, Plain(weights, audio), audio.to(dev)


# A step's log-probability in bf16: logits of magnitude up to 8 whose rounding
# alone is 2^-9 relative (0.016), after two layers of bf16 activations, each of
# whose dozen roundings (2^-9) moves a logit by a few hundredths: 0.1 a step
# covers them threefold.
STEP_TOL = 0.1


@pytest.mark.parametrize("chunks,beams,page,steps", [(1, 4, 16, 10), (3, 2, 16, 21), (3, 7, 32, 6),
                                                     (2, 1, 16, 8)])
def test_matches_the_plain_search(model, chunks, beams, page, steps):
    """Every returned hypothesis has the log-probability that the plain model
    gives its ids, and the best is as good as the plain search's best: wrong
    pages, positions, parents or copies would show in either."""
    dec, plain, audio = model
    res = dec.generate_beam(audio[:chunks], PROMPT, beams=beams, max_new_tokens=steps,
                            page_size=page, length_penalty=0.0)
    assert len(res.per_chunk_ids) == chunks
    for c in range(chunks):
        hyps = res.hypotheses[c]
        assert res.per_chunk_ids[c] == hyps[0][0]
        assert len({tuple(h[0]) for h in hyps}) == len(hyps) == beams
        assert all(a[2] >= b[2] for a, b in zip(hyps, hyps[1:]))
        for ids, logp, _ in hyps[:3]:
            assert abs(logp - plain.score(c, ids)) <= STEP_TOL * len(ids)
        best = plain.search(c, beams, steps)[0]
        assert hyps[0][1] >= best[0] - 2 * STEP_TOL * steps


def test_captured_and_eager_steps_agree(model):
    dec, _, audio = model
    kw = dict(beams=3, max_new_tokens=19, page_size=16)
    eager = dec.generate_beam(audio, PROMPT, graphs=False, **kw)
    first = dec.generate_beam(audio, PROMPT, **kw)
    again = dec.generate_beam(audio, PROMPT, **kw)       # replays the captured step
    torch.cuda.synchronize()
    assert eager.hypotheses == first.hypotheses == again.hypotheses
    assert eager.steps == first.steps == again.steps


def test_fused_and_library_layers_agree(model):
    """Up to 16 rows run vl_decode_linear, more cuBLAS: the scores agree to the
    steps' tolerance where both return a hypothesis."""
    dec, _, audio = model
    runs = []
    for fused in (True, False):
        dec.fused = fused
        try:
            dec._states.clear()
            runs.append(dec.generate_beam(audio, PROMPT, beams=4, max_new_tokens=5))
        finally:
            dec.fused = True
            dec._states.clear()
    for a, b in zip(*[r.hypotheses for r in runs]):
        scores = {tuple(h[0]): h[1] for h in a}
        both = [(scores[tuple(h[0])], h[1]) for h in b if tuple(h[0]) in scores]
        assert both and all(abs(x - y) <= 2 * 5 * STEP_TOL for x, y in both)


def test_one_beam_is_greedy(model):
    """One beam takes the likeliest token of every step, as generate() does,
    unless two are closer than the roundings of the two paths."""
    dec, plain, audio = model
    beam = dec.generate_beam(audio, PROMPT, beams=1, max_new_tokens=8)
    greedy = dec.generate(audio, PROMPT, max_new_tokens=8)
    for c in range(audio.shape[0]):
        for i, (x, y) in enumerate(zip(beam.per_chunk_ids[c], greedy.per_chunk_ids[c])):
            if x != y:
                lp = plain.log_probs(c, beam.per_chunk_ids[c][:i])
                assert abs(float(lp[x] - lp[y])) <= 2 * STEP_TOL
                break


def test_a_chunk_does_not_depend_on_its_neighbours(model):
    dec, _, audio = model
    three = dec.generate_beam(audio, PROMPT, beams=2, max_new_tokens=6)
    one = dec.generate_beam(audio[1:2], PROMPT, beams=2, max_new_tokens=6)
    a = {tuple(h[0]): h[1] for h in three.hypotheses[1]}
    both = [(a[tuple(h[0])], h[1]) for h in one.hypotheses[0] if tuple(h[0]) in a]
    assert both and all(abs(x - y) <= 2 * 6 * STEP_TOL for x, y in both)


def test_refusals(model):
    dec, _, audio = model
    with pytest.raises(vlasr.VlasrInputError, match="beams"):
        dec.generate_beam(audio, PROMPT, beams=33)
    with pytest.raises(vlasr.VlasrInputError, match="max_seq_len"):
        dec.generate_beam(audio, PROMPT, max_new_tokens=200)
    with pytest.raises(vlasr.VlasrInputError, match="page_size"):
        dec.generate_beam(audio, PROMPT, max_new_tokens=4, page_size=48)


@pytest.mark.parametrize("graphs", [False, True])
def test_a_failure_inside_a_step_is_raised(model, monkeypatch, graphs):
    """A page id out of range in the tables that a step's attention is given
    (read as zeros, and reported) ends the search with an error."""
    dec, _, audio = model
    attend = vlasr.decoder.paged.paged_attention

    def bad(q, kc, vc, start, length, table, **kw):
        return attend(q, kc, vc, start, length, torch.full_like(table, kc.shape[0]), **kw)

    dec._states.clear()
    monkeypatch.setattr(vlasr.decoder.paged, "paged_attention", bad)
    try:
        with pytest.raises(vlasr.VlasrExecutionError, match="status 8"):
            dec.generate_beam(audio, PROMPT, beams=2, max_new_tokens=4, graphs=graphs)
    finally:
        dec._states.clear()


def test_audio_that_is_not_finite_is_an_error(model):
    dec, _, audio = model
    bad = audio.clone()
    bad[1, 3] = float("nan")
    for graphs in (False, True):
        with pytest.raises(vlasr.VlasrExecutionError, match=r"chunks \[1\]"):
            dec.generate_beam(bad, PROMPT, beams=2, max_new_tokens=4, graphs=graphs)
    good = dec.generate_beam(audio, PROMPT, beams=2, max_new_tokens=4)
    assert all(math.isfinite(h[0][1]) for h in good.hypotheses)
