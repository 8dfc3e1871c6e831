"""GPU: beam_select and paged_beam_reorder against their plain 64-bit
statements (tests/paged_ref.py).  Tokens, parents, tables, lengths and caches
are compared bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref
import vlasr
from helpers import torch_dtype

pytestmark = pytest.mark.gpu

# The sum of a row is off by at most 64 fp32 additions per lane (64 * 2^-24),
# exp2's 2^-22 and its argument's rounding (40 * 2^-24): below 1e-5, and so
# its logarithm; the value is then rounded to fp32 once.
VALUE_TOL = 1e-5


def f64(t):
    return t.detach().double().cpu().numpy()


def run_select(dev, logits, scores, finished=None, eos=(), pad=0, min_gap=2 * VALUE_TOL):
    batch, beams = scores.shape
    fin = None if finished is None else finished.to(dev)
    tok, par, val, end = vlasr.beam_select(logits, scores.to(dev), finished=fin, eos_ids=eos,
                                           pad_id=pad)
    torch.cuda.synchronize()
    assert tok.dtype == torch.int64 and par.dtype == torch.int32 and end.dtype == torch.bool
    wt, wp, wv, we, gap = paged_ref.select(f64(logits), scores.numpy(),
                                           None if finished is None else finished.numpy(), eos,
                                           pad, beams)
    assert gap > min_gap            # the inputs tell the candidates apart
    assert np.array_equal(tok.cpu().numpy(), wt)
    assert np.array_equal(par.cpu().numpy(), wp)
    assert np.array_equal(end.cpu().numpy(), we)
    got = f64(val)
    assert np.array_equal(np.isinf(got), np.isinf(wv))
    ok = np.isfinite(wv)
    assert (np.abs(got[ok] - wv[ok]) <= VALUE_TOL + 2.0 ** -24 * np.abs(wv[ok])).all()
    return tok, par, val, end


def make(dev, name, batch, beams, vocab, seed, std=3.0, stride=None, offset=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    x = (torch.randn(batch * beams, vocab, generator=g) * std).to(torch_dtype(name))
    scores = -torch.rand(batch, beams, generator=g) * 5
    if stride:
        wide = torch.full((batch * beams, stride), 50.0, dtype=x.dtype, device=dev)
        wide[:, offset:offset + vocab] = x.to(dev)
        return wide[:, offset:offset + vocab], scores
    return x.to(dev), scores


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,beams,vocab", [(1, 4, 59264), (3, 5, 1001), (2, 1, 333),
                                               (2, 8, 4097), (1, 32, 700), (1, 2, 1), (2, 3, 2),
                                               (1, 16, 20011)])
def test_select(dev, name, batch, beams, vocab):
    logits, scores = make(dev, name, batch, beams, vocab, seed=vocab + beams)
    run_select(dev, logits, scores)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_select_strided_and_unaligned_rows(dev, name, offset):
    """What lies between the rows (larger than any logit) is not read as one."""
    logits, scores = make(dev, name, 2, 3, 2051, seed=5 + offset, stride=2063, offset=offset)
    run_select(dev, logits, scores)


def test_select_first_step_and_few_candidates(dev):
    """Only beam 0 counts at the start; a vocabulary smaller than the beams
    leaves places empty."""
    logits, scores = make(dev, "f32", 2, 4, 500, seed=7)
    scores[:] = -float("inf")
    scores[:, 0] = 0.0
    _, par, _, _ = run_select(dev, logits, scores)
    assert (par == 0).all()
    logits, scores = make(dev, "f32", 2, 4, 3, seed=8)
    scores[:] = -float("inf")
    scores[:, 0] = 0.0
    tok, par, val, end = run_select(dev, logits, scores, pad=2)
    assert tok[:, 3].tolist() == [2, 2] and par[:, 3].tolist() == [3, 3]
    assert end[:, 3].all() and torch.isinf(val[:, 3]).all()


def test_select_finished_beams_and_eos(dev):
    logits, scores = make(dev, "bf16", 6, 4, 900, seed=9)
    finished = torch.rand(6, 4, generator=torch.Generator().manual_seed(10)) < 0.5
    finished[0] = True
    finished[1] = False
    logits[finished.view(-1).to(dev)] = 1e4      # a finished beam's logits are not looked at
    logits[4:8, 17] = 20.0
    run_select(dev, logits, scores, finished=finished, eos=(17, 30), pad=30)


def test_select_masked_logits(dev):
    """-inf is never taken; a row of nothing, of NaN or with +inf offers nothing."""
    logits, scores = make(dev, "f32", 3, 4, 1200, seed=11)
    logits[:, ::2] = -float("inf")
    logits[1] = -float("inf")
    logits[2, 40] = float("nan")
    logits[3, 41] = float("inf")
    logits[4, 2:] = -float("inf")
    logits[5] = -float("inf")
    logits[5, 7] = 3.0
    logits[8:12] = -float("inf")
    tok, par, val, end = run_select(dev, logits, scores, pad=5)
    assert (par[0] == 0).all() and torch.isinf(val[2]).all() and end[2].all()


def test_select_minus_inf_score_and_finished_without_score(dev):
    logits, scores = make(dev, "f16", 2, 3, 640, seed=12)
    scores[0, 1] = -float("inf")
    scores[1, 2] = -float("inf")
    finished = torch.tensor([[False, False, True], [False, True, True]])
    run_select(dev, logits, scores, finished=finished, pad=1)


def test_select_ties_go_to_the_lower_index(dev):
    """Equal logits within a row, and equal rows of equal score across beams."""
    g = torch.Generator(device="cpu").manual_seed(13)
    row = torch.randn(9000, generator=g)
    row[[8000, 17, 4096, 4097, 2500]] = 9.0
    logits = row.repeat(4, 1).to(dev)
    scores = torch.zeros(1, 4)
    tok, par, _, _ = run_select(dev, logits, scores)
    assert tok.tolist() == [[17, 2500, 4096, 4097]] and par.tolist() == [[0, 0, 0, 0]]
    flat = torch.zeros(4, 9000, device=dev)
    tok, par, _, _ = run_select(dev, flat, scores)
    assert tok.tolist() == [[0, 1, 2, 3]] and par.tolist() == [[0, 0, 0, 0]]
    one = torch.full((4, 9000), -float("inf"), device=dev)
    one[:, 77] = 1.0
    tok, par, _, _ = run_select(dev, one, scores)
    assert tok.tolist() == [[77] * 4] and par.tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("beams", [1, 4, 32])
def test_select_more_candidates_than_the_heap_holds(dev, name, beams):
    """Rows in ascending order (every value beats the ones before it) and rows
    of few values (nearly all candidates are ties)."""
    vocab = 20000
    up = torch.linspace(-8.0, 8.0, vocab).to(torch_dtype(name)).repeat(2 * beams, 1)
    up[1:] -= 0.25 * torch.arange(1, 2 * beams).view(-1, 1).to(torch_dtype(name))
    scores = -torch.linspace(0, 3, 2 * beams).view(2, beams) * 1.7
    run_select(dev, up.to(dev), scores)
    g = torch.Generator(device="cpu").manual_seed(16)
    few = torch.randint(0, 3, (2 * beams, vocab), generator=g).to(torch_dtype(name))
    run_select(dev, few.to(dev), scores)


@pytest.mark.parametrize("name,vocab", [("f32", 59264), ("f32", 40001), ("bf16", 120000)])
def test_select_rows_in_one_piece(dev, name, vocab):
    """So many rows that each is one piece and goes round its ring of copies
    more than once."""
    batch, beams = 75, 4
    logits, scores = make(dev, name, batch, beams, vocab, seed=17)
    # one f32-exact place a row with a value of its own per entry and beam, so
    # that 16-bit logits tie nowhere among the best
    best = torch.arange(batch * beams, device=dev)
    logits[best, (best * 131) % vocab] = 24.0
    tok, par, val, _ = vlasr.beam_select(logits, scores.to(dev))
    torch.cuda.synchronize()
    x = logits.double()
    values = scores.to(dev).double().view(-1, 1) + x - torch.logsumexp(x, 1, keepdim=True)
    top, at = values.view(batch, beams * vocab).topk(beams + 1)
    clear = (top[:, :-1] - top[:, 1:]).amin(1) > 2 * VALUE_TOL
    assert int(clear.sum()) >= batch // 2
    assert torch.equal(tok[clear], (at % vocab)[clear, :beams])
    assert torch.equal(par[clear].long(), (at // vocab)[clear, :beams])
    assert ((val.double() - top[:, :beams]).abs() <=
            VALUE_TOL + 2.0 ** -24 * top[:, :beams].abs()).all()


def test_select_in_place_repeated_and_captured(dev):
    """scores_out = scores and finished_out = finished, captured and replayed."""
    batch, beams, vocab = 2, 4, 5000
    logits, scores = make(dev, "bf16", batch, beams, vocab, seed=14)
    want = run_select(dev, logits, scores, finished=torch.zeros(batch, beams, dtype=torch.bool),
                      eos=(3,))
    s, f = scores.to(dev), torch.zeros(batch, beams, dtype=torch.bool, device=dev)
    tok = torch.empty(batch, beams, dtype=torch.int64, device=dev)
    par = torch.empty(batch, beams, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        vlasr.beam_select(logits, s.clone(), finished=f.clone(), eos_ids=(3,))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            vlasr.beam_select(logits, s, finished=f, eos_ids=(3,), tokens=tok, parents=par,
                              scores_out=s, finished_out=f)
    torch.cuda.synchronize()
    for _ in range(3):
        s.copy_(scores)
        f.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((tok, par, s, f), want):
            assert torch.equal(a, b)


def test_select_refusals(dev):
    logits, scores = make(dev, "f32", 2, 3, 64, seed=15)
    scores = scores.to(dev)
    with pytest.raises(vlasr.VlasrInputError, match="batch \\* beams rows"):
        vlasr.beam_select(logits[:5], scores)
    with pytest.raises(vlasr.VlasrInputError, match="pad_id"):
        vlasr.beam_select(logits, scores, pad_id=64)
    with pytest.raises(vlasr.VlasrInputError, match="scores must be"):
        vlasr.beam_select(logits, scores.double())
    with pytest.raises(vlasr.VlasrInputError, match="tokens must be"):
        vlasr.beam_select(logits, scores, tokens=torch.zeros(2, 3, device=dev))
    with pytest.raises(vlasr.VlasrInputError, match="beams"):
        vlasr.beam_select(torch.zeros(40, 64, device=dev), torch.zeros(1, 40, device=dev))
    with pytest.raises(vlasr.VlasrInputError, match="finished must be"):
        vlasr.beam_select(logits, scores, finished=torch.zeros(2, 3, device=dev))


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------

def run_reorder(dev, table, parents, kv_len, first, pool, kc, vc, expect_bad=None, **kw):
    t = torch.tensor(np.asarray(table), dtype=torch.int32, device=dev)
    p = torch.tensor(np.asarray(parents), dtype=torch.int32, device=dev)
    n = torch.tensor(np.asarray(kv_len), dtype=torch.int32, device=dev)
    f = torch.tensor(np.asarray(first), dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    want = paged_ref.reorder(t.cpu().numpy(), p.cpu().numpy(), n.cpu().numpy(), f.cpu().numpy(),
                             pool, f64(kc), f64(vc))
    old = t.clone()
    out, lens = vlasr.paged_beam_reorder(t, p, n, f, pool, kc, vc, status=status, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want[0])
    assert np.array_equal(lens.cpu().numpy(), want[1])
    assert np.array_equal(f64(kc), want[2]) and np.array_equal(f64(vc), want[3])
    assert torch.equal(t, old)
    if expect_bad is not None:
        assert want[4] == expect_bad
    assert int(status) == (vlasr.VL_STATUS_BAD_PAGE if want[4] else 0)
    return out, lens


def caches(dev, name, layers, pages, ps, kvh=2, hd=32, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    shape = (layers, pages, ps, kvh, hd)
    return [torch.randn(shape, generator=g).to(torch_dtype(name)).to(dev) for _ in range(2)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("beams,ps", [(1, 16), (3, 16), (4, 32), (8, 16), (32, 16)])
def test_reorder_random_walk(dev, name, beams, ps):
    """Forty steps of random parents, the lengths growing by one: tables,
    copies and reuse of freed pages as in the plain statement."""
    rng = np.random.default_rng(beams)
    batch, prompt, steps = 3, 21, 40
    full = prompt // ps
    width = (prompt + steps) // ps + 2
    pool = beams * (width - full)
    total = batch * (full + pool)
    kc, vc = caches(dev, name, 3, total, ps, seed=beams)
    first = [batch * full + e * pool for e in range(batch)]
    table = np.full((batch * beams, width), -1, np.int32)
    for e in range(batch):
        table[e * beams:(e + 1) * beams, :full] = range(e * full, (e + 1) * full)
        if prompt % ps:      # the prompt's last page, shared at first
            table[e * beams:(e + 1) * beams, full] = first[e]
    lens = np.full(batch * beams, prompt, np.int32)
    for _ in range(steps):
        parents = rng.integers(0, beams, (batch, beams))
        out, got = run_reorder(dev, table, parents, lens, first, pool, kc, vc, expect_bad=False)
        table, lens = out.cpu().numpy(), got.cpu().numpy() + 1
        wp = (lens - 1) // ps
        mine = table[np.arange(len(lens)), wp].reshape(batch, beams)
        assert all(len(set(r)) == beams for r in mine.tolist())     # nobody shares a written page


def test_reorder_prompt_page_outside_the_range(dev):
    """A part-filled prompt page that several entries share is copied by all."""
    kc, vc = caches(dev, "bf16", 2, 12, 16)
    table = [[0, 1, -1]] * 4
    out, _ = run_reorder(dev, table, [[0, 1], [1, 1]], [20] * 4, [2, 6], 4, kc, vc,
                         expect_bad=False)
    assert out[:, 1].tolist() == [2, 3, 6, 7]


def test_reorder_lengths_that_differ(dev):
    """A page that one row reads whole is not written by another that holds
    part of it."""
    kc, vc = caches(dev, "f16", 2, 16, 16)
    table = [[4, 5, -1], [4, -1, -1], [6, 7, 8]]
    run_reorder(dev, table, [[0, 1, 2]], [18, 7, 40], [4], 12, kc, vc, expect_bad=False)
    run_reorder(dev, table, [[1, 1, 0]], [18, 7, 40], [4], 12, kc, vc, expect_bad=False)
    run_reorder(dev, table, [[2, 2, 2]], [16, 0, 32], [4], 12, kc, vc, expect_bad=False)


def test_reorder_full_tables_and_zero_lengths(dev):
    kc, vc = caches(dev, "f16", 1, 16, 16)
    table = [[4, 5], [6, 7]]
    out, _ = run_reorder(dev, table, [[1, 1]], [32, 32], [4], 12, kc, vc, expect_bad=False)
    assert out.tolist() == [[6, 7], [6, 7]]
    out, _ = run_reorder(dev, [[-1, -1]] * 2, [[0, 0]], [0, 0], [4], 12, kc, vc, expect_bad=False)
    assert out.tolist() == [[4, -1], [5, -1]]


def test_reorder_what_is_out_of_range(dev):
    kc, vc = caches(dev, "bf16", 2, 16, 16)
    table = [[4, 5, -1], [4, 6, -1]]
    run_reorder(dev, table, [[0, 2]], [20, 20], [4], 8, kc, vc, expect_bad=True)      # parent
    run_reorder(dev, table, [[-1, 1]], [20, 20], [4], 8, kc, vc, expect_bad=True)
    run_reorder(dev, table, [[0, 1]], [49, -1], [4], 8, kc, vc, expect_bad=True)      # lengths
    run_reorder(dev, [[99, 5, -1], [4, 16, -1]], [[0, 1]], [20, 20], [4], 8, kc, vc,
                expect_bad=True)                                                      # page ids
    run_reorder(dev, table, [[0, 0]], [20, 20], [4], 2, kc, vc, expect_bad=True)      # exhausted
    run_reorder(dev, table, [[0, 0]], [20, 20], [12], 8, kc, vc, expect_bad=True)     # range
    run_reorder(dev, table, [[0, 0]], [20, 20], [4], 0, kc, vc, expect_bad=True)


def test_reorder_strided_caches_and_tables(dev):
    """Layers inside pages, tables as slices, a single 4-D layer, odd row bytes."""
    g = torch.Generator(device="cpu").manual_seed(3)
    both = torch.randn(16, 5, 16, 1, 32, generator=g).to(torch.bfloat16).to(dev)
    kc = both.transpose(0, 1)
    vc = both.clone().transpose(0, 1)
    wide = torch.full((2, 9), -7, dtype=torch.int32, device=dev)
    run_reorder(dev, [[4, 5, -1], [4, 6, -1]], [[0, 0]], [20, 20], [4], 8, kc, vc,
                expect_bad=False, out=wide[:, 2:5])
    assert (wide[:, :2] == -7).all() and (wide[:, 5:] == -7).all()
    k5, v5 = caches(dev, "f16", 1, 12, 16, kvh=1, hd=3, seed=4)       # rows of six bytes
    run_reorder(dev, [[4, 5], [4, 6]], [[1, 1]], [29, 29], [4], 8, k5, v5, expect_bad=False)
    k5, v5 = caches(dev, "f32", 1, 12, 16, kvh=1, hd=3, seed=5)
    t = torch.tensor([[4, 5], [4, 6]], dtype=torch.int32, device=dev)
    par = torch.tensor([[1, 1]], dtype=torch.int32, device=dev)
    n = torch.tensor([29, 29], dtype=torch.int32, device=dev)
    f = torch.tensor([4], dtype=torch.int32, device=dev)
    want = paged_ref.reorder(t.cpu().numpy(), par.cpu().numpy(), n.cpu().numpy(), [4], 8, f64(k5),
                             f64(v5))
    out, _ = vlasr.paged_beam_reorder(t, par, n, f, 8, k5[0], v5[0])
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(f64(k5), want[2])


def test_reorder_refusals(dev):
    kc, vc = caches(dev, "bf16", 1, 8, 16)
    t = torch.zeros(4, 3, dtype=torch.int32, device=dev)
    par = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    n = torch.zeros(4, dtype=torch.int32, device=dev)
    f = torch.zeros(2, dtype=torch.int32, device=dev)
    with pytest.raises(vlasr.VlasrInputError, match="overlap"):
        vlasr.paged_beam_reorder(t, par, n, f, 4, kc, vc, out=t)
    with pytest.raises(vlasr.VlasrInputError, match="overlap"):
        vlasr.paged_beam_reorder(t, par, n, f, 4, kc, vc, kv_len_out=n)
    with pytest.raises(vlasr.VlasrInputError, match="page_table must be"):
        vlasr.paged_beam_reorder(t[:3], par, n, f, 4, kc, vc)
    with pytest.raises(vlasr.VlasrInputError, match="parents must be"):
        vlasr.paged_beam_reorder(t, par.long(), n, f, 4, kc, vc)
    with pytest.raises(vlasr.VlasrInputError, match="same shape"):
        vlasr.paged_beam_reorder(t, par, n, f, 4, kc, vc[:, :4])
    with pytest.raises(vlasr.VlasrInputError, match="pool_start"):
        vlasr.paged_beam_reorder(t, par, n, f[:1].contiguous(), 4, kc, vc)


def test_select_status_stays_clear(dev):
    """A masked row is no failure: the word is set only by a wait that ran out."""
    logits, scores = make(dev, "bf16", 2, 3, 5000, seed=18)
    logits[1] = -float("inf")
    logits[4, 7] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    want = vlasr.beam_select(logits, scores.to(dev))
    got = vlasr.beam_select(logits, scores.to(dev), status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    with pytest.raises(vlasr.VlasrInputError, match="status"):
        vlasr.beam_select(logits, scores.to(dev), status=status.long())


def test_select_values_over_the_longest_rows(dev):
    """2^24 tokens a row, so many rows that each is one piece: the value keeps
    VALUE_TOL where every round adds the same to a lane's sum (roundings all
    one way), and where the lanes' maxima grow from round to round."""
    batch, vocab = 296, 1 << 24
    logits = torch.empty(batch, vocab, device=dev)
    scores = torch.zeros(batch, 1, device=dev)
    best = torch.arange(batch, device=dev) * 50021 % vocab
    row = torch.arange(batch, device=dev)

    def check(first):
        tok, par, val, _ = vlasr.beam_select(logits, scores)
        torch.cuda.synchronize()
        assert torch.equal(tok[:, 0], first) and int(par.count_nonzero()) == 0
        want = torch.stack([logits[i, first[i]].double() - torch.logsumexp(logits[i].double(), 0)
                            for i in range(batch)])
        off = (val[:, 0].double() - want).abs()
        assert (off <= VALUE_TOL + 2.0 ** -24 * want.abs()).all(), float(off.max())

    rounds = vocab // 8192
    logits[:] = -torch.linspace(0.1, 8.0, batch, device=dev).view(-1, 1)
    logits[:, :1024:4] = 0.0                 # a maximum for every lane, in the first round
    check(torch.zeros_like(best))
    # one value a lane and round climbs, by 0.00005 to 0.005 a round
    logits.view(batch, rounds, 8192)[:, :, :1024:4] = \
        (torch.linspace(0.1, 10.0, batch, device=dev).view(-1, 1)
         * torch.linspace(0.0, 1.0, rounds, device=dev)).unsqueeze(2)
    logits[row, best] = 11.0
    check(best)
