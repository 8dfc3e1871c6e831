"""GPU: the paged-cache operators (vl_paged_rope_append, vl_paged_attention)
against their plain 64-bit statements (tests/paged_ref.py).

Tolerances are bounds, not measurements: half a step of the output's type,
plus what the fp32 arithmetic in between may add (stated at each use)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref
import vlasr
from helpers import torch_dtype

pytestmark = pytest.mark.gpu

NAMES = ["f32", "f16", "bf16"]


def f64(t):
    return t.detach().double().cpu().numpy()


class Paged:
    """A ragged batch over shuffled pages.  Every cache row that no sequence
    holds is NaN, and so are the packed rows behind the last sequence."""

    def __init__(self, dev, name, new, past, nq, nkv, hd, ps, seed, pad=0, packed=False, std=1.0,
                 extra_cols=0, layers_view=False, fill_new=True):
        g = torch.Generator(device="cpu").manual_seed(seed)
        dt = torch_dtype(name)
        self.name, self.nq, self.nkv, self.hd, self.ps = name, nq, nkv, hd, ps
        self.new, self.past = new, past
        lens = [n + p for n, p in zip(new, past)]
        per = [-(-max(n, 0) // ps) for n in lens]
        width = max(max(per), 1) + 1
        total = sum(per) + 3
        order = torch.randperm(total, generator=g).int()
        table = torch.full((len(new), width + extra_cols), 0x7ffffff0, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        starts = np.concatenate([[0], np.cumsum(new)])
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=dev)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.table = table.to(dev)[:, :width]
        tokens = int(starts[-1]) + pad

        def rand(*shape):
            return (torch.randn(shape, generator=g) * std).to(dt)

        qkv = rand(tokens, (nq + 2 * nkv) * hd)
        if pad:
            qkv[tokens - pad:] = float("nan")
        qkv = qkv.to(dev)
        cols = [qkv[:, :nq * hd], qkv[:, nq * hd:(nq + nkv) * hd], qkv[:, (nq + nkv) * hd:]]
        self.q, self.k, self.v = cols if packed else [c.contiguous() for c in cols]
        kc = torch.full((total, ps, nkv, hd), float("nan"), dtype=dt)
        vc = kc.clone()
        for b in range(len(new)):
            for p in range(lens[b] if fill_new else past[b]):
                page, r = int(table[b, p // ps]), p % ps
                kc[page, r] = rand(nkv, hd)
                vc[page, r] = rand(nkv, hd)
        if layers_view:      # pages of two layers interleaved: a page stride
            self.kc = torch.stack([kc, kc], 1).to(dev)[:, 1]
            self.vc = torch.stack([vc, vc], 1).to(dev)[:, 1]
        else:
            self.kc, self.vc = kc.to(dev), vc.to(dev)
        self.tokens, self.pad = tokens, pad

    def ints(self):
        return (self.q_start.cpu().numpy(), self.kv_len.cpu().numpy(), self.table.cpu().numpy())


def check_rows(got, want, tol, name):
    """|got - want| <= half a step of want + tol, elementwise."""
    got = f64(got).reshape(want.shape)
    bound = paged_ref.HALF_STEP[name] * (np.abs(want) + tol) + tol
    bound += 2.0 ** -25 if name == "f16" else 1e-38          # a subnormal's half step
    off = np.abs(got - want)
    assert np.isfinite(got[np.isfinite(want)]).all()
    worst = np.nanmax(off / bound) if off.size else 0.0
    assert worst <= 1.0, worst


# ---------------------------------------------------------------------------
# rotation and append
# ---------------------------------------------------------------------------

def run_append(p, rotary, interleaved, scale, base=10000.0, with_q=True, in_place=False):
    dev = p.kc.device
    q0 = f64(p.q).reshape(p.tokens, p.nq, p.hd)
    k0 = f64(p.k).reshape(p.tokens, p.nkv, p.hd)
    v0 = f64(p.v).reshape(p.tokens, p.nkv, p.hd)
    kc0, vc0 = f64(p.kc), f64(p.vc)
    before_k, before_v = p.k.clone(), p.v.clone()
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = p.q if in_place else torch.full((p.tokens, p.nq * p.hd), 3.0, dtype=p.q.dtype, device=dev)
    vlasr.paged_rope_append(p.q if with_q else None, p.k, p.v, p.kc, p.vc, p.q_start, p.kv_len,
                            p.table, head_dim=p.hd, rotary_dim=rotary, base=base,
                            interleaved=interleaved, position_scale=scale,
                            q_out=out if with_q else None, status=status)
    torch.cuda.synchronize()
    qs, kl, tab = p.ints()
    qo, kc, vc = paged_ref.append(q0, k0, v0, kc0, vc0, qs, kl, tab, rotary, base, interleaved,
                                  scale)
    # cos and sin are within 3e-7 of the exact ones, the two products and
    # their sum within 2^-24 each: 5e-7 of |x1| + |x2|
    rot = 5e-7
    real = p.tokens - p.pad
    if with_q:
        check_rows(out[:real], qo[:real].reshape(real, -1),
                   rot * paged_ref.rotation_bound(q0, rotary, interleaved)[:real].reshape(real, -1),
                   p.name)
        if p.pad and not in_place:
            assert (out[real:] == 3.0).all()
    got_k, got_v = f64(p.kc), f64(p.vc)
    assert np.array_equal(got_v, vc, equal_nan=True)
    # rotated rows within the bound; all other rows bit for bit
    same = np.array_equal(np.isnan(got_k), np.isnan(kc))
    assert same
    big = np.nan_to_num(np.abs(k0)).max() * 2
    bound = paged_ref.HALF_STEP[p.name] * np.abs(kc) + rot * big + 2.0 ** -25
    assert (np.nan_to_num(np.abs(got_k - kc)) <= np.nan_to_num(bound, nan=1.0)).all()
    written = np.zeros(kc.shape[:2], bool)
    for b in range(len(p.new)):
        for i in range(p.new[b]):
            pos = kl[b] - p.new[b] + i
            written[tab[b, pos // p.ps], pos % p.ps] = True
    assert np.array_equal(got_k[~written], kc0[~written], equal_nan=True)
    assert torch.equal(p.k[:real], before_k[:real]) and torch.equal(p.v[:real], before_v[:real])
    assert int(status) == 0


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("hd,rotary", [(64, 64), (128, 128), (128, 64), (64, 16), (96, 48),
                                       (32, 6), (256, 256), (64, 0)])
def test_append_layouts(dev, name, interleaved, hd, rotary):
    p = Paged(dev, name, [1, 5, 0, 19], [0, 30, 4, 15], 6, 2, hd, 16, seed=1, pad=3, packed=True)
    run_append(p, rotary, interleaved, 1.0)


@pytest.mark.parametrize("seqs", [1, 31, 32, 33, 70, 1100])
def test_append_single_tokens(dev, seqs):
    """A decode step of many sequences: the sequence lookup at and around its
    32-wide rounds."""
    rng = np.random.default_rng(seqs)
    p = Paged(dev, "bf16", [1] * seqs, rng.integers(0, 40, seqs).tolist(), 2, 1, 64, 16, seed=2)
    run_append(p, 64, False, 1.0)


def test_append_empty_sequences_between(dev):
    new = [0, 0, 3, 0, 1, 0, 0, 7, 0]
    p = Paged(dev, "f16", new, [5, 0, 2, 9, 16, 0, 3, 31, 8], 4, 4, 128, 32, seed=3)
    run_append(p, 128, False, 1.0)


def test_append_in_place_and_far_positions(dev):
    """q rotated in place; positions of 2^20 whose angle needs fp64."""
    p = Paged(dev, "f32", [2], [0], 4, 2, 64, 16, seed=4)
    run_append(p, 64, True, 0.125, in_place=True)
    p = Paged(dev, "f32", [2], [0], 4, 2, 64, 256, seed=5)
    far = 1 << 20
    p.kv_len += far
    width = far // 256 + 2
    table = torch.full((1, width), -1, dtype=torch.int32, device=dev)
    table[0, far // 256] = 1
    p.table = table
    run_append(p, 64, False, 1.0, base=500000.0)


def test_append_strided_pages_and_no_q(dev):
    p = Paged(dev, "bf16", [4, 9], [14, 3], 8, 2, 128, 16, seed=6, layers_view=True, extra_cols=5)
    run_append(p, 128, False, 1.0)
    p = Paged(dev, "bf16", [4, 9], [14, 3], 8, 2, 128, 16, seed=7)
    run_append(p, 128, True, 1.0, with_q=False)


def test_append_unaligned_rows(dev):
    """k rows at an odd stride take the element-by-element kernel."""
    p = Paged(dev, "f16", [3, 2], [1, 17], 2, 1, 64, 16, seed=8)
    wide = torch.zeros(p.tokens, 67, dtype=torch.float16, device=dev)
    wide[:, 1:65] = p.k
    p.k = wide[:, 1:65]
    run_append(p, 32, False, 1.0)


def test_append_skips_what_is_out_of_range(dev):
    p = Paged(dev, "bf16", [2, 2, 2], [16, 16, 16], 2, 1, 64, 16, seed=9, fill_new=False)
    kc0, vc0 = p.kc.clone(), p.vc.clone()
    p.table = p.table.clone()
    p.table[0, 1] = p.kc.shape[0]       # a page id past the end
    p.table[1, 1] = -5
    p.kv_len[2] = 1                     # first token at position -1, second at 0
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = vlasr.paged_rope_append(p.q, p.k, p.v, p.kc, p.vc, p.q_start, p.kv_len, p.table,
                                  status=status)
    torch.cuda.synchronize()
    assert int(status) & vlasr.VL_STATUS_BAD_PAGE
    page = int(p.table[2, 0])
    assert torch.equal(p.vc[page, 0].view(-1), p.v[5])
    p.vc[page, 0] = vc0[page, 0]
    p.kc[page, 0] = kc0[page, 0]
    assert np.array_equal(f64(p.kc), f64(kc0), equal_nan=True)
    assert np.array_equal(f64(p.vc), f64(vc0), equal_nan=True)
    assert torch.isfinite(out).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def run_attention(p, max_q, scale=0.0, out=None, **kw):
    qs, kl, tab = p.ints()
    q0 = f64(p.q).reshape(p.tokens, p.nq, p.hd)
    fill = torch.full((p.tokens, p.nq * p.hd), 5.0, dtype=p.q.dtype, device=p.q.device)
    got = fill.clone() if out is None else out
    before = f64(got).reshape(p.tokens, p.nq, p.hd)
    status = torch.zeros(1, dtype=torch.int32, device=p.q.device)
    vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q,
                          scale=scale, out=got, status=status, **kw)
    torch.cuda.synchronize()
    rounds_p = 0.0 if p.name == "f32" or p.hd not in (64, 128) else paged_ref.HALF_STEP[p.name]
    want, tol = paged_ref.attention(q0, f64(p.kc), f64(p.vc), qs, kl, tab,
                                    scale or p.hd ** -0.5, before, rounds_p)
    check_rows(got, want.reshape(p.tokens, -1), tol.reshape(p.tokens, -1), p.name)
    assert int(status) == 0
    return got


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("nq,nkv,hd", [(16, 4, 128), (5, 1, 64), (8, 8, 128), (6, 2, 64),
                                       (16, 1, 128), (3, 3, 96), (4, 2, 32), (2, 1, 256)])
def test_attention_single_tokens(dev, name, nq, nkv, hd):
    past = [0, 1, 14, 15, 16, 62, 63, 64, 65, 200]
    p = Paged(dev, name, [1] * len(past), past, nq, nkv, hd, 16, seed=20, pad=2, packed=True)
    run_attention(p, 1)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_attention_page_sizes(dev, ps):
    """Pages that end inside a 64- or 128-position tile and pages larger than one."""
    past = [0, 30, 63, 64, 127, 128, 300]
    p = Paged(dev, "bf16", [1] * len(past), past, 8, 2, 128, ps, seed=21)
    run_attention(p, 1)
    new = [1, 33, 2, 130]
    p = Paged(dev, "bf16", new, [100, 0, 257, 31], 8, 2, 128, ps, seed=22)
    run_attention(p, max(new))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd,new", [
    (4, 2, 128, [2, 1, 3, 8, 0, 5]), (16, 4, 128, [4, 1, 0, 2]), (5, 1, 64, [3, 1, 2]),
    (2, 2, 64, [16, 1, 9])])
def test_attention_few_tokens(dev, name, nq, nkv, hd, new):
    """A few tokens per sequence (up to 16 query rows per kv head), causal
    among themselves."""
    past = [(37 * i) % 90 for i in range(len(new))]
    p = Paged(dev, name, new, past, nq, nkv, hd, 16, seed=23)
    run_attention(p, max(new))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", [(16, 4, 128), (4, 4, 64), (10, 2, 64), (7, 1, 128),
                                       (3, 1, 64), (32, 1, 64), (12, 2, 128)])
def test_attention_chunks(dev, name, nq, nkv, hd):
    """Ragged chunks beside single tokens and empty sequences."""
    new = [40, 1, 0, 129, 17]
    past = [0, 70, 9, 0, 140]
    p = Paged(dev, name, new, past, nq, nkv, hd, 16, seed=24, pad=5, packed=True)
    run_attention(p, max(new))


@pytest.mark.parametrize("new,past", [(31, 0), (32, 0), (33, 0), (63, 65), (64, 64), (65, 63),
                                      (127, 1), (128, 128), (129, 127), (256, 0), (300, 90)])
def test_attention_chunk_edges(dev, new, past):
    """Chunk lengths and cache lengths around the tiles' edges."""
    p = Paged(dev, "bf16", [new], [past], 4, 1, 64, 32, seed=25 + new)
    run_attention(p, new)


def test_attention_f32_chunk(dev):
    p = Paged(dev, "f32", [20, 3], [10, 0], 4, 2, 64, 16, seed=26)
    run_attention(p, 20)


def test_attention_rows_that_see_nothing(dev):
    """kv_len below the number of new tokens: the first of them see no position."""
    for max_q, new in ((3, [3, 2]), (40, [40, 2])):
        p = Paged(dev, "bf16", new, [0, 0], 4, 1, 128, 16, seed=27)
        p.kv_len -= torch.tensor([2, 2], dtype=torch.int32, device=dev)
        got = run_attention(p, max_q)
        assert int(got[:2].count_nonzero()) == 0
        assert int(got[new[0]:].count_nonzero()) == 0


def test_attention_large_scores(dev):
    """Scores of hundreds: the running maximum moves, weights underflow."""
    p = Paged(dev, "bf16", [1, 1], [300, 77], 4, 1, 64, 16, seed=28, std=6.0)
    run_attention(p, 1)
    p = Paged(dev, "f16", [50], [200], 4, 1, 64, 16, seed=29, std=6.0)
    run_attention(p, 50)


def test_attention_out_is_q_and_strided_tables(dev):
    for max_q, new in ((1, [1, 1, 1]), (30, [30, 1, 12])):
        p = Paged(dev, "bf16", new, [20, 100, 3], 4, 2, 128, 16, seed=30, packed=True,
                  extra_cols=7, layers_view=True)
        q = p.q.clone()
        want = run_attention(p, max_q).clone()
        p2 = p.q
        vlasr.paged_attention(p2, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q,
                              out=p2)
        torch.cuda.synchronize()
        assert torch.equal(p2, want)
        p2.copy_(q)


def test_attention_scale(dev):
    p = Paged(dev, "f16", [1, 1], [40, 200], 4, 1, 64, 16, seed=31)
    run_attention(p, 1, scale=0.3)
    p = Paged(dev, "f16", [35], [40], 4, 1, 64, 16, seed=32)
    run_attention(p, 35, scale=0.3)


@pytest.mark.parametrize("max_q", [1, 64])
def test_attention_bad_lengths_and_pages(dev, max_q):
    """Out-of-range lengths give zero rows, a bad page id rows of zeros; the
    other sequences are as without them."""
    new = [1, 1, 1, 1] if max_q == 1 else [40, 3, 64, 20]
    past = [50, 20, 90, 33]
    p = Paged(dev, "bf16", new, past, 4, 1, 128, 16, seed=33)
    run_attention(p, max_q)
    starts = p.q_start.tolist()
    p.kv_len[1] = -3
    p.kv_len[2] = p.table.shape[1] * 16 + 1
    p.table = p.table.clone()
    p.table[3, 1] = p.kc.shape[0] + 7
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full_like(p.q, 9.0)
    vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q, out=out,
                          status=status)
    torch.cuda.synchronize()
    assert int(status) == vlasr.VL_STATUS_BAD_PAGE
    assert int(out[starts[1]:starts[3]].count_nonzero()) == 0
    qs, kl, tab = p.ints()
    want, tol = paged_ref.attention(f64(p.q).reshape(p.tokens, 4, 128), f64(p.kc), f64(p.vc), qs,
                                    np.array([kl[0], 0, 0, kl[3]]), tab, 128 ** -0.5,
                                    np.zeros((p.tokens, 4, 128)), paged_ref.HALF_STEP["bf16"])
    check_rows(out, want.reshape(p.tokens, -1), tol.reshape(p.tokens, -1), "bf16")


def test_attention_more_tokens_than_promised(dev):
    """A sequence longer than max_q_len gives zero rows and the status bit."""
    p = Paged(dev, "bf16", [1, 9, 1], [30, 30, 30], 4, 1, 64, 16, seed=34)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=1,
                                status=status)
    torch.cuda.synchronize()
    assert int(status) == vlasr.VL_STATUS_BAD_PAGE
    assert int(out[1:10].count_nonzero()) == 0 and int(out[0].count_nonzero()) > 0


def test_attention_q_start_out_of_range(dev):
    """Row ranges that are not the batch's are skipped, nothing is written there."""
    for max_q in (1, 64):
        p = Paged(dev, "bf16", [1, 1, 1], [30, 30, 30], 4, 1, 64, 16, seed=35)
        p.q_start.copy_(torch.tensor([0, 1, 7, 6], dtype=torch.int32))
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        out = torch.full_like(p.q, 4.0)
        vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q,
                              out=out, status=status)
        torch.cuda.synchronize()
        assert int(status) == vlasr.VL_STATUS_BAD_PAGE
        assert (out[1:] == 4.0).all() and (out[0] != 4.0).any()


@pytest.mark.parametrize("max_q,new", [(1, [1] * 6), (90, [90, 1, 33, 64, 0, 12])])
def test_attention_repeats_bit_for_bit(dev, max_q, new):
    """Twice the same call, with a workspace full of NaN and on another
    stream: the same bits."""
    p = Paged(dev, "bf16", new, [500, 3, 800, 64, 10, 129], 8, 2, 128, 32, seed=36)
    a = run_attention(p, max_q)
    need = vlasr.paged_attention_workspace_bytes(p.tokens, len(new), max_q, 8, 2, 128)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        b = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q,
                                  workspace=ws)
        c = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=max_q,
                                  workspace=ws)
    side.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_attention_calls_at_once_and_captured(dev):
    """Two streams at once, and two graphs replayed at once, each with a
    workspace of its own; a captured call follows lengths that change."""
    ps = [Paged(dev, "bf16", [1] * 9, [100 * i % 701 for i in range(9)], 8, 2, 128, 16, seed=40 + s)
          for s in range(2)]
    want = [run_attention(p, 1).clone() for p in ps]
    streams = [torch.cuda.Stream(dev) for _ in ps]
    graphs, outs = [], []
    for p, st in zip(ps, streams):
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            out = torch.zeros_like(p.q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=1,
                                      out=out)
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)
    p = ps[0]
    p.kv_len -= torch.arange(9, dtype=torch.int32, device=dev).clamp(max=1)
    graphs[0].replay()
    torch.cuda.synchronize()
    eager = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=1)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager)


def test_append_then_attention_captured_with_pdl(dev):
    """The two operators as a decode layer runs them, captured once and
    replayed over growing lengths, the attention as a programmatic dependent."""
    seqs, nq, nkv, hd, ps = 5, 8, 2, 128, 16
    past = [0, 15, 16, 40, 100]
    p = Paged(dev, "bf16", [1] * seqs, [x + 8 for x in past], nq, nkv, hd, ps, seed=50, packed=True)
    p.kv_len.copy_(torch.tensor([x + 1 for x in past], dtype=torch.int32))
    qkv = torch.empty(seqs, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device=dev)
    q, k, v = qkv[:, :nq * hd], qkv[:, nq * hd:(nq + nkv) * hd], qkv[:, (nq + nkv) * hd:]
    rot, out = torch.empty_like(p.q), torch.empty(seqs, nq * hd, dtype=torch.bfloat16, device=dev)

    def step():
        vlasr.paged_rope_append(q, k, v, p.kc, p.vc, p.q_start, p.kv_len, p.table, q_out=rot)
        vlasr.paged_attention(rot, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=1, out=out,
                              pdl=True)

    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    qkv.copy_(torch.randn(qkv.shape))
    kc, vc = p.kc.clone(), p.vc.clone()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(g, stream=side):
            step()
    torch.cuda.synchronize()
    p.kc.copy_(kc)
    p.vc.copy_(vc)
    gen = torch.Generator(device="cpu").manual_seed(51)
    for i in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=gen))
        g.replay()
        torch.cuda.synchronize()
        qs, kl, tab = p.ints()
        qo, kc64, vc64 = paged_ref.append(
            f64(q).reshape(seqs, nq, hd), f64(k).reshape(seqs, nkv, hd),
            f64(v).reshape(seqs, nkv, hd), f64(p.kc), f64(p.vc), qs, kl, tab, hd, 10000.0, False,
            1.0)
        check_rows(rot, qo.reshape(seqs, -1),
                   5e-7 * paged_ref.rotation_bound(f64(q).reshape(seqs, nq, hd), hd, False)
                   .reshape(seqs, -1), "bf16")
        want, tol = paged_ref.attention(f64(rot).reshape(seqs, nq, hd), f64(p.kc), f64(p.vc), qs,
                                        kl, tab, hd ** -0.5, np.zeros((seqs, nq, hd)),
                                        paged_ref.HALF_STEP["bf16"])
        check_rows(out, want.reshape(seqs, -1), tol.reshape(seqs, -1), "bf16")
        p.kv_len += 1


def test_attention_offsets_past_32_bits(dev):
    """A cache whose pages lie more than 2^31 elements apart."""
    nkv, hd, ps = 4, 128, 256
    pages = (1 << 31) // (ps * nkv * hd) + 600
    kc = torch.empty(pages, ps, nkv, hd, dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    ids = [pages - 1, 3, pages - 599, 0]
    g = torch.Generator(device="cpu").manual_seed(60)
    for i in ids:
        kc[i] = torch.randn(ps, nkv, hd, generator=g)
        vc[i] = torch.randn(ps, nkv, hd, generator=g)
    small_k, small_v = kc[ids].contiguous(), vc[ids].contiguous()
    far = torch.tensor([ids], dtype=torch.int32, device=dev)
    near = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    for n in (1, 70):
        q = torch.randn(n, 16 * hd, generator=g).to(torch.bfloat16).to(dev)
        qs = torch.tensor([0, n], dtype=torch.int32, device=dev)
        kl = torch.tensor([1000], dtype=torch.int32, device=dev)
        a = vlasr.paged_attention(q, kc, vc, qs, kl, far, max_q_len=n)
        b = vlasr.paged_attention(q, small_k, small_v, qs, kl, near, max_q_len=n)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    k = torch.randn(5, nkv * hd, generator=g).to(torch.bfloat16).to(dev)
    qs = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    kl = torch.tensor([5], dtype=torch.int32, device=dev)
    vlasr.paged_rope_append(None, k, k, kc, vc, qs, kl, far, rotary_dim=0)
    torch.cuda.synchronize()
    assert torch.equal(vc[pages - 1, :5].view(5, -1), k)
    assert torch.equal(kc[pages - 1, :5].view(5, -1), k)


def test_wrapper_refusals(dev):
    p = Paged(dev, "bf16", [1, 1], [3, 4], 4, 2, 64, 16, seed=70)
    args = (p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table)
    with pytest.raises(vlasr.VlasrInputError, match="shape and strides"):
        vlasr.paged_attention(p.q, p.kc, p.vc[:2], *args[3:], max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="match dtype"):
        vlasr.paged_attention(p.q.float(), *args[1:], max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="q_start must be"):
        vlasr.paged_attention(*args[:3], p.q_start[:2].contiguous(), *args[4:], max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="kv_len must be torch.int32"):
        vlasr.paged_attention(*args[:4], p.kv_len.long(), p.table, max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="page_table"):
        vlasr.paged_attention(*args[:5], p.table[0], max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="max_q_len"):
        vlasr.paged_attention(*args, max_q_len=0)
    with pytest.raises(vlasr.VlasrInputError, match="q's rows"):
        vlasr.paged_attention(*args, max_q_len=1, out=torch.empty_like(p.q[:1]))
    with pytest.raises(vlasr.VlasrInputError, match="workspace"):
        vlasr.paged_attention(*args, max_q_len=1,
                              workspace=torch.empty(8, dtype=torch.uint8, device=dev))
    with pytest.raises(vlasr.VlasrInputError, match="cache's heads"):
        vlasr.paged_rope_append(p.q, p.k[:, :64], p.v, *args[1:])
    with pytest.raises(vlasr.VlasrInputError, match="rotary_dim"):
        vlasr.paged_rope_append(p.q, p.k, p.v, *args[1:], rotary_dim=66)
    with pytest.raises(vlasr.VlasrInputError, match="q_out needs q"):
        vlasr.paged_rope_append(None, p.k, p.v, *args[1:], q_out=p.q)


@pytest.mark.parametrize("name,nq,nkv,hd,ps", [("bf16", 4, 2, 128, 32), ("f16", 5, 1, 64, 16),
                                               ("bf16", 8, 1, 64, 256)])
def test_attention_chunks_over_long_caches(dev, name, nq, nkv, hd, ps):
    """Few cells and many tiles: each is cut into pieces that are joined; one
    ends right where the cache does, one is too short to be cut."""
    new, past = [33, 1, 70, 0, 20], [2999, 767, 1466, 40, 100]
    p = Paged(dev, name, new, past, nq, nkv, hd, ps, seed=60, pad=3)
    run_attention(p, max(new))


def test_attention_long_single_tokens(dev):
    """One and two sequences whose units spread over many blocks."""
    for new, past in (([1], [5000]), ([1, 2], [1, 3001])):
        p = Paged(dev, "bf16", new, past, 8, 2, 128, 64, seed=61)
        run_attention(p, max(new))


@pytest.mark.parametrize("seqs,max_q", [(33, 1), (1100, 1), (40, 24), (1100, 24)])
def test_attention_many_sequences(dev, seqs, max_q):
    """The lookup of sequences beyond one and beyond 32 lanes' worth, empty
    ones and runs of short ones among them."""
    rng = np.random.default_rng(seqs + max_q)
    new = rng.integers(0, 2, seqs) if max_q == 1 else \
        np.where(rng.random(seqs) < 0.1, rng.integers(1, max_q + 1, seqs), rng.integers(0, 2, seqs))
    past = rng.integers(0, 40, seqs)
    new[seqs // 2] = max_q
    p = Paged(dev, "f16", new.tolist(), past.tolist(), 2, 1, 64, 16, seed=62, pad=2)
    run_attention(p, max_q)


def test_attention_chunk_longer_than_promised(dev):
    """As for single tokens: zero rows and the status bit, the others as they are."""
    p = Paged(dev, "bf16", [20, 60, 33], [30, 200, 0], 4, 1, 64, 16, seed=63)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=40,
                                status=status)
    torch.cuda.synchronize()
    assert int(status) == vlasr.VL_STATUS_BAD_PAGE
    assert int(out[20:80].count_nonzero()) == 0
    qs, kl, tab = p.ints()
    want, tol = paged_ref.attention(f64(p.q).reshape(p.tokens, 4, 64), f64(p.kc), f64(p.vc), qs,
                                    kl * np.array([1, 0, 1]), tab, 64 ** -0.5,
                                    np.zeros((p.tokens, 4, 64)), paged_ref.HALF_STEP["bf16"])
    check_rows(out, want.reshape(p.tokens, -1), tol.reshape(p.tokens, -1), "bf16")


def test_attention_chunks_captured_at_once(dev):
    """Two graphs of chunks that are cut and joined, replayed side by side with
    a workspace each; lengths that change between replays are followed."""
    ps = [Paged(dev, "bf16", [40, 25], [1500, 3], 4, 1, 128, 32, seed=64 + s) for s in range(2)]
    want = [run_attention(p, 40).clone() for p in ps]
    graphs, outs = [], []
    streams = [torch.cuda.Stream(dev) for _ in ps]
    for p, st in zip(ps, streams):
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            out = torch.zeros_like(p.q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=40,
                                      out=out)
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)
    ps[0].kv_len[0] -= 700
    short = run_attention(ps[0], 40).clone()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], short) and not torch.equal(short, want[0])


def test_empty_batches(dev):
    """No tokens, and no sequences: empty results, nothing else touched."""
    kc = torch.full((4, 16, 2, 64), 7.0, dtype=torch.bfloat16, device=dev)
    vc = kc.clone()
    i32 = dict(dtype=torch.int32, device=dev)
    status = torch.zeros(1, **i32)
    for batch in (0, 3):
        q = torch.empty(0, 4 * 64, dtype=torch.bfloat16, device=dev)
        k = torch.empty(0, 2 * 64, dtype=torch.bfloat16, device=dev)
        start, length = torch.zeros(batch + 1, **i32), torch.full((batch,), 5, **i32)
        table = torch.zeros(batch, 2, **i32)
        got = vlasr.paged_rope_append(q, k, k, kc, vc, start, length, table, status=status)
        assert got.shape == (0, 256)
        for max_q in (1, 50):
            got = vlasr.paged_attention(q, kc, vc, start, length, table, max_q_len=max_q,
                                        status=status)
            assert got.shape == (0, 256)
    torch.cuda.synchronize()
    assert int(status) == 0 and (kc == 7).all() and (vc == 7).all()
    tok, par, val, end = vlasr.beam_select(torch.empty(0, 100, device=dev),
                                           torch.empty(0, 4, device=dev))
    assert tok.shape == par.shape == val.shape == end.shape == (0, 4)
    out, held = vlasr.paged_beam_reorder(torch.empty(0, 2, **i32), torch.empty(0, 4, **i32),
                                         torch.empty(0, **i32), torch.empty(0, **i32), 2, kc, vc)
    assert out.shape == (0, 2) and held.shape == (0,)


@pytest.mark.parametrize("hd,new,past", [(128, 40, 300), (64, 40, 300), (128, 33, 2000),
                                         (128, 3, 300)])
def test_attention_keys_that_are_not_finite(dev, hd, new, past):
    """A NaN in a key makes the rows that see it non-finite and leaves the
    others alone; an infinite key is a weight of 0 where its score is -inf and
    non-finite where it is +inf.  Positions at every place of a group of eight."""
    p = Paged(dev, "bf16", [new], [past], 4, 1, hd, 16, seed=80)
    late = past + new // 2
    kc0 = p.kc.clone()
    for at in (late, *range(16, 24)):
        p.kc.copy_(kc0)
        p.kc[int(p.table[0, at // 16]), at % 16, 0, 5] = float("nan")
        got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new)
        torch.cuda.synchronize()
        sees = max(0, at - past)                     # the first token that does
        assert not torch.isfinite(got[sees:]).any()
        if sees:
            qs, kl, tab = p.ints()
            want, tol = paged_ref.attention(
                f64(p.q).reshape(new, 4, hd)[:sees], f64(kc0), f64(p.vc), [0, sees],
                [past + sees], tab, hd ** -0.5, np.zeros((sees, 4, hd)),
                paged_ref.HALF_STEP["bf16"])
            check_rows(got[:sees], want.reshape(sees, -1), tol.reshape(sees, -1), "bf16")
    q = f64(p.q).reshape(new, 4, hd)
    rows = (f64(kc0)[p.table[0].cpu().numpy()[:-(-(past + new) // 16)]].reshape(-1, hd)[:past + new],
            f64(p.vc)[p.table[0].cpu().numpy()[:-(-(past + new) // 16)]].reshape(-1, hd)[:past + new])
    for at in range(16, 24):
        p.kc.copy_(kc0)
        p.kc[int(p.table[0, at // 16]), at % 16, 0, 5] = float("inf")
        got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new)
        torch.cuda.synchronize()
        got = got.view(new, 4, hd)
        for t in range(new):
            for h in range(4):
                if q[t, h, 5] >= 0:
                    assert not torch.isfinite(got[t, h]).any()
                    continue
                use = np.delete(np.arange(past + t + 1), at)
                s = rows[0][use] @ q[t, h] * hd ** -0.5
                w = np.exp(s - s.max())
                w /= w.sum()
                mags = (np.abs(rows[0][use]) @ np.abs(q[t, h])).max() * hd ** -0.5
                rel = 2 * hd * 2.0 ** -23 * mags + (len(use) + hd) * 2.0 ** -23 + 2.0 ** -20
                tol = (rel + paged_ref.HALF_STEP["bf16"]) * (w @ np.abs(rows[1][use]))
                check_rows(got[t, h], w @ rows[1][use], tol, "bf16")


def test_attention_rows_of_minus_infinity(dev):
    """Every score -inf: a row of zeros, as when nothing is seen."""
    for new, past in ((40, 300), (2, 300), (33, 2000)):
        p = Paged(dev, "bf16", [new], [past], 2, 1, 128, 16, seed=81)
        seen = torch.isfinite(p.kc[..., 5])
        p.kc[..., 5][seen] = float("inf")
        p.q.view(new, 2, 128)[:, :, 5] = -1.0
        got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new)
        torch.cuda.synchronize()
        assert int(got.count_nonzero()) == 0


@pytest.mark.parametrize("name,nq,nkv,hd,new", [
    ("bf16", 16, 4, 128, [1, 1, 1, 1]), ("f16", 5, 1, 64, [1, 3, 0, 2, 1]),
    ("bf16", 4, 2, 128, [8, 1, 5, 0, 2]), ("f16", 16, 1, 128, [1, 1]), ("bf16", 3, 3, 64, [2, 16])])
def test_few_tokens_by_cluster_and_along_the_line(dev, name, nq, nkv, hd, new):
    """Short caches through narrow page tables (a cluster per pair) and through
    wide ones (equal runs, joined by a second launch): lengths that leave some
    of a cluster's blocks without tiles, none at all, rows that see nothing."""
    for past in ([0, 1, 60, 500, 940], [700, 63, 0, 64, 2], [128, 1000, 900, 3, 190]):
        p = Paged(dev, name, new, past[:len(new)], nq, nkv, hd, 16, seed=90)
        narrow = p.table
        a = run_attention(p, max(new))
        p.table = torch.nn.functional.pad(narrow, (0, 100), value=-3)
        b = run_attention(p, max(new))
        tol = 4 * paged_ref.HALF_STEP[name]          # a rounding of P and of the output each
        assert (a.float() - b.float()).abs().max() <= tol * a.float().abs().max() * 2
        p.kv_len[0] = new[0] - 1                     # the first token sees nothing
        for table in (narrow, p.table):
            p.table = table
            got = run_attention(p, max(new))
            assert int(got[0].count_nonzero()) == 0


@pytest.mark.parametrize("wide", [0, 100])
def test_few_tokens_out_of_range(dev, wide):
    """Bad lengths, pages and row ranges give the same in both forms."""
    new = [1, 2, 3, 2, 1]
    p = Paged(dev, "bf16", new, [50, 20, 90, 33, 7], 4, 2, 128, 16, seed=91)
    if wide:
        p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
    run_attention(p, 3)
    starts = p.q_start.tolist()
    p.kv_len[0] = -1
    p.kv_len[1] = p.table.shape[1] * 16 + 1
    p.table = p.table.clone()
    p.table[3, 0] = p.kc.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full_like(p.q, 9.0)
    vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=2, out=out,
                          status=status)
    torch.cuda.synchronize()
    assert int(status) == vlasr.VL_STATUS_BAD_PAGE
    assert int(out[:starts[3]].count_nonzero()) == 0          # 2: more tokens than promised
    qs, kl, tab = p.ints()
    want, tol = paged_ref.attention(f64(p.q).reshape(p.tokens, 4, 128), f64(p.kc), f64(p.vc), qs,
                                    np.array([0, 0, 0, kl[3], kl[4]]), tab, 128 ** -0.5,
                                    np.zeros((p.tokens, 4, 128)), paged_ref.HALF_STEP["bf16"])
    check_rows(out, want.reshape(p.tokens, -1), tol.reshape(p.tokens, -1), "bf16")


@pytest.mark.parametrize("wide", [0, 100])
def test_few_tokens_captured_at_once(dev, wide):
    """Two graphs of the same form side by side, each with a workspace."""
    ps = [Paged(dev, "f16", [1, 2, 1], [200, 700, 3], 8, 2, 64, 16, seed=92 + s) for s in range(2)]
    graphs, outs, want = [], [], []
    streams = [torch.cuda.Stream(dev) for _ in ps]
    for p, st in zip(ps, streams):
        if wide:
            p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
        want.append(run_attention(p, 2).clone())
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            out = torch.zeros_like(p.q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=2,
                                      out=out)
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)


@pytest.mark.parametrize("wide", [0, 100])
@pytest.mark.parametrize("new", [1, 3])
def test_few_tokens_that_are_not_a_number(dev, new, wide):
    """A NaN query row, and NaN keys that fill what a warp, a tile or a whole
    share of the tiles sees: the rows that see one are not finite, whichever
    form the table's width chooses, and the other rows are right."""
    past = [0, 64, 300, 255, 130, 700]
    # first and last NaN position of each sequence (none: its query is NaN)
    spans = [(0, 0), (64, 64), None, (64, 127), (0, 130), (650, 650)]
    p = Paged(dev, "bf16", [new] * len(past), past, 4, 1, 128, 16, seed=95)
    if wide:
        p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
    sees = torch.zeros(p.tokens, dtype=torch.bool)
    for b, span in enumerate(spans):
        rows = torch.arange(b * new, (b + 1) * new)
        if span is None:
            p.q[rows[0]] = float("nan")
            sees[rows[0]] = True
            continue
        for at in range(span[0], span[1] + 1):
            p.kc[int(p.table[b, at // 16]), at % 16] = float("nan")
        sees[rows] = past[b] + torch.arange(new) >= span[0]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new,
                                status=status)
    torch.cuda.synchronize()
    assert int(status) == 0 and not torch.isfinite(got[sees.to(dev)]).any()
    fine = (~sees).numpy()
    if fine.any():
        with np.errstate(invalid="ignore"):
            want, tol = paged_ref.attention(
                f64(p.q).reshape(p.tokens, 4, 128), f64(p.kc), f64(p.vc), *p.ints(), 128 ** -0.5,
                np.zeros((p.tokens, 4, 128)), paged_ref.HALF_STEP["bf16"])
        check_rows(got[(~sees).to(dev)], want[fine].reshape(fine.sum(), -1),
                   tol[fine].reshape(fine.sum(), -1), "bf16")


@pytest.mark.parametrize("new", [40, 1])
def test_attention_at_the_longest_length(dev, new):
    """kv_len 2^31 - 256, the longest that the calls take, through a table that
    repeats one page; the keys of that page weigh nothing (score -512 below
    the others), so the rows are those of the last two pages alone."""
    ps, hd = 256, 64
    pages = ((1 << 31) - 256) // ps
    g = torch.Generator(device="cpu").manual_seed(96)
    kc = torch.randn(3, ps, 1, hd, generator=g)
    kc[..., 0] = 0.0
    kc[0, :, 0, 0] = -512.0
    kc = kc.to(torch.bfloat16).to(dev)
    vc = torch.randn(3, ps, 1, hd, generator=g).to(torch.bfloat16).to(dev)
    q = torch.randn(new, 4, hd, generator=g)
    q[..., 0] = 8.0
    q = q.to(torch.bfloat16).to(dev).view(new, 4 * hd)
    table = torch.zeros(1, pages, dtype=torch.int32, device=dev)
    table[0, -2:] = torch.tensor([2, 1], dtype=torch.int32, device=dev)
    start = torch.tensor([0, new], dtype=torch.int32, device=dev)
    length = torch.tensor([pages * ps], dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = vlasr.paged_attention(q, kc, vc, start, length, table, max_q_len=new, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    want, tol = paged_ref.attention(f64(q).reshape(new, 4, hd), f64(kc), f64(vc), [0, new],
                                    [2 * ps], np.array([[2, 1]]), hd ** -0.5,
                                    np.zeros((new, 4, hd)), paged_ref.HALF_STEP["bf16"])
    check_rows(got, want.reshape(new, -1), tol.reshape(new, -1), "bf16")


@pytest.mark.parametrize("name,nq,nkv,hd,new,wide", [
    ("bf16", 8, 2, 128, [1, 1, 1], 0), ("bf16", 8, 2, 128, [1, 1, 1], 100),
    ("f16", 5, 1, 64, [40, 3, 17], 0), ("f32", 4, 2, 96, [5, 1, 2], 0)])
def test_what_padding_rows_hold_does_not_matter(dev, name, nq, nkv, hd, new, wide):
    """Rows behind the last sequence: the same bits whatever they hold, and
    they are left as they were."""
    p = Paged(dev, name, new, [30, 700, 3], nq, nkv, hd, 16, seed=97, pad=9, packed=True)
    if wide:
        p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
    real, got = p.tokens - p.pad, []
    for value in (0.0, float("inf"), float("nan"), 3.0):
        for x in (p.q, p.k, p.v):
            x[real:] = value
        kc, vc = p.kc.clone(), p.vc.clone()
        out = torch.full((p.tokens, nq * hd), 7.0, dtype=p.q.dtype, device=dev)
        rot = vlasr.paged_rope_append(p.q, p.k, p.v, kc, vc, p.q_start, p.kv_len, p.table,
                                      q_out=out.clone())
        vlasr.paged_attention(rot, kc, vc, p.q_start, p.kv_len, p.table, max_q_len=max(new), out=out)
        torch.cuda.synchronize()
        assert (rot[real:] == 7.0).all() and (out[real:] == 7.0).all()
        got.append([t.nan_to_num(99.0) for t in (rot[:real], out[:real], kc, vc)])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("at", [129, 130, 131, 133])
@pytest.mark.parametrize("name,hd", [("bf16", 128), ("f16", 64)])
def test_attention_nan_among_minus_infinity(dev, name, hd, at):
    """A NaN key in a long stretch whose other scores are -inf: a cut cell's
    piece has no finite maximum, and its rows are not finite all the same."""
    new, past = 33, 2000
    p = Paged(dev, name, [new], [past], 4, 1, hd, 16, seed=98)
    ids = p.table[0].cpu().long()
    for page in range(94):                       # positions 0 .. 1503
        p.kc[ids[page], :, 0, 5] = -float("inf")
    p.q.view(new, 4, hd)[:, :, 5] = 1.0
    status = torch.zeros(1, dtype=torch.int32, device=dev)

    def run():
        got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new,
                                    status=status)
        torch.cuda.synchronize()
        return got

    assert torch.isfinite(run()).all()
    p.kc[ids[at // 16], at % 16, 0] = float("nan")
    assert not torch.isfinite(run()).any() and int(status) == 0


@pytest.mark.parametrize("new,past,wide", [(1, 1000, 0), (1, 1000, 100), (3, 900, 0),
                                           (40, 1400, 0), (300, 0, 0)])
@pytest.mark.parametrize("name,hd", [("f16", 64), ("f16", 128), ("bf16", 128)])
def test_attention_of_many_small_weights(dev, name, hd, new, past, wide):
    """One key takes nearly all of a row's weight and its value is 0; what is
    left are weights of 2^-26 each, which sum to the result."""
    p = Paged(dev, name, [new], [past], 4, 1, hd, 16, seed=99)
    if wide:
        p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
    ids = p.table[0, :-(-(new + past) // 16)].cpu().long()
    p.kc[ids], p.q[:] = 0.0, 0.0
    p.kc[ids[0], 0, 0, 5], p.vc[ids[0], 0] = 8.0, 0.0
    p.q.view(new, 4, hd)[:, :, 5] = 2.25         # a score of 18 against 0
    run_attention(p, new, scale=1.0)


@pytest.mark.parametrize("new,past,wide", [(3, 500, 0), (3, 500, 100), (70, 500, 0), (70, 3000, 0)])
@pytest.mark.parametrize("name,hd", [("f16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("peak", [2000, 4000])
def test_attention_of_enormous_scores(dev, name, hd, new, past, wide, peak):
    """Scores of 10^7 and more, where fp32 no longer holds their fractions: a
    row is its best key's value (the next is 10^6 below), and finite."""
    p = Paged(dev, name, [new], [past], 4, 1, hd, 16, seed=101)
    if wide:
        p.table = torch.nn.functional.pad(p.table, (0, wide), value=-3)
    ids = p.table[0, :-(-(new + past) // 16)].cpu().long()
    p.kc[ids], p.q[:] = 0.0, 0.0
    g = torch.Generator(device="cpu").manual_seed(102)
    rising = torch.arange(past + new) % 400 * 8.0 + 128.0       # 128 .. 3320, in many tiles
    best = past - 77
    rising[best] = 16000.0
    flat = torch.zeros(len(ids) * 16)
    flat[:past + new] = rising
    p.kc[ids, :, 0, 5] = flat.view(-1, 16).to(p.kc.dtype).to(dev)
    # many queries, so that the products' roundings fall both ways
    p.q.view(new, 4, hd)[:, :, 5] = (
        peak * (1 + torch.rand(new, 4, generator=g)) / 2).to(p.q.dtype).to(dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = vlasr.paged_attention(p.q, p.kc, p.vc, p.q_start, p.kv_len, p.table, max_q_len=new,
                                scale=1.0, status=status)
    torch.cuda.synchronize()
    want = p.vc[ids[best // 16], best % 16, 0].expand(new, 4, hd).reshape(new, -1)
    assert int(status) == 0 and torch.isfinite(got).all()
    # the weight's rounding and the output's
    assert ((got - want).float().abs() <=
            2 * paged_ref.HALF_STEP[name] * want.float().abs() * 1.01 + 2.0 ** -24).all()


@pytest.mark.parametrize("seqs,share", [(12, 0.5), (300, 0.1), (1500, 0.05), (1500, 0.5)])
@pytest.mark.parametrize("name,hd", [("bf16", 128), ("f16", 64)])
def test_attention_chunks_among_sequences_that_see_nothing(dev, name, hd, seqs, share):
    """Rows of sequences without positions, many in a row, between chunks that
    end inside a tile: every block's run has pieces without tiles behind one
    that has some."""
    rng = np.random.default_rng(seqs)
    new = rng.integers(1, 4, seqs)
    past = rng.integers(0, 60, seqs)
    new[seqs // 3] = 20
    p = Paged(dev, name, new.tolist(), past.tolist(), 2, 2, hd, 16, seed=103)
    lens = p.kv_len.cpu().numpy()
    gone = rng.random(seqs) > share
    gone[seqs // 3] = False
    lens[gone] = 0
    p.kv_len.copy_(torch.from_numpy(lens))
    got = run_attention(p, 20)
    starts = p.q_start.cpu().numpy()
    for b in np.nonzero(gone)[0][:50]:
        assert int(got[starts[b]:starts[b + 1]].count_nonzero()) == 0
