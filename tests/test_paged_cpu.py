"""CPU: what the paged-cache and beam-search entry points refuse, before any
CUDA call, and the plain statements the GPU tests compare with, against
independent small cases."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import paged_ref
import vlasr
from vlasr import _lib

FAKE = 0x10000
FAR = 0x100000000     # bases far enough apart not to overlap


@pytest.fixture(scope="module")
def lib():
    return vlasr.load()


def _err(lib) -> str:
    return lib.vl_last_error().decode()


def test_append_rejects(lib):
    def call(q=FAR, k=2 * FAR, v=3 * FAR, qo=4 * FAR, kc=5 * FAR, vc=6 * FAR, qst=FAKE, kvl=FAKE,
             tab=FAKE, tokens=4, batch=2, max_pages=8, ts=8, nq=16, nkv=4, hd=128, rot=128,
             inter=0, base=1e4, scale=1.0, qs=2048, ks=512, vs=512, os_=2048, pages=64, ps=16,
             stride=16 * 512, dtype=2):
        return lib.vl_paged_rope_append(q, k, v, qo, kc, vc, qst, kvl, tab, tokens, batch,
                                        max_pages, ts, nq, nkv, hd, rot, inter, base, scale, qs,
                                        ks, vs, os_, pages, ps, stride, dtype, None, None)

    assert call(k=None) == 2 and "null" in _err(lib)
    assert call(kc=None) == 2 and "null" in _err(lib)
    assert call(tab=None) == 2 and "null" in _err(lib)
    assert call(q=None) == 2 and "n_q_heads" in _err(lib)
    assert call(dtype=5) == 2 and "dtype" in _err(lib)
    assert call(tokens=-1) == 2 and "shape" in _err(lib)
    assert call(nkv=0) == 2 and "shape" in _err(lib)
    for ps in (0, 8, 24, 512):
        assert call(ps=ps, stride=1 << 20) == 2 and "page_size" in _err(lib)
    assert call(pages=0) == 2 and "num_pages" in _err(lib)
    assert call(ts=7) == 2 and "table_stride" in _err(lib)
    assert call(stride=100) == 2 and "page_stride" in _err(lib)
    assert call(rot=130) == 2 and "rotary_dim" in _err(lib)
    assert call(rot=63) == 2 and "rotary_dim" in _err(lib)
    assert call(inter=2) == 2 and "interleaved" in _err(lib)
    assert call(base=0.0) == 2 and "base" in _err(lib)
    assert call(scale=math.inf) == 2 and "position_scale" in _err(lib)
    assert call(qs=100) == 2 and "strides" in _err(lib)
    assert call(qo=FAR + 64) == 2 and "overlaps" in _err(lib)
    # disjoint columns of one buffer are not an overlap; nothing to do is not an error
    assert call(tokens=0, qo=FAR + 4096, qs=6144, os_=6144) == 0
    assert call(batch=0) == 0


def test_attention_rejects(lib):
    def call(q=FAR, kc=2 * FAR, vc=3 * FAR, qst=FAKE, kvl=FAKE, tab=FAKE, tokens=4, batch=4,
             mq=1, max_pages=8, ts=8, nq=16, nkv=4, hd=128, scale=0.0, qs=2048, os_=2048,
             pages=64, ps=16, stride=16 * 512, out=4 * FAR, dtype=2, ws=5 * FAR, wsb=1 << 30,
             flags=0):
        return lib.vl_paged_attention(q, kc, vc, qst, kvl, tab, tokens, batch, mq, max_pages, ts,
                                      nq, nkv, hd, scale, qs, os_, pages, ps, stride, out, dtype,
                                      ws, wsb, None, flags, None)

    assert call(q=None) == 2 and "null" in _err(lib)
    assert call(kvl=None) == 2 and "null" in _err(lib)
    assert call(dtype=9) == 2 and "dtype" in _err(lib)
    assert call(flags=4) == 2 and "flags" in _err(lib)
    assert call(nq=14) == 2 and "heads" in _err(lib)
    assert call(nq=1024, nkv=4, qs=1 << 17, os_=1 << 17) == 2 and "heads" in _err(lib)
    assert call(hd=72, nkv=4) == 2 and "head_dim" in _err(lib)
    assert call(hd=288, stride=1 << 20) == 2 and "head_dim" in _err(lib)
    assert call(mq=0) == 2 and "max_q_len" in _err(lib)
    assert call(scale=math.nan) == 2 and "scale" in _err(lib)
    assert call(scale=-1.0) == 2 and "scale" in _err(lib)
    assert call(os_=100) == 2 and "strides" in _err(lib)
    assert call(qs=2052) == 2 and "multiples" in _err(lib)
    assert call(stride=16 * 512 + 4) == 2 and "multiples" in _err(lib)
    assert call(out=4 * FAR + 2) == 2 and "aligned" in _err(lib)
    assert call(ps=48) == 2 and "page_size" in _err(lib)
    assert call(wsb=8) == 2 and "workspace" in _err(lib)
    assert call(ws=None) == 2 and "workspace" in _err(lib)
    assert call(out=2 * FAR) == 2 and "overlaps" in _err(lib)
    assert call(out=FAR + 2048) == 2 and "overlaps" in _err(lib)
    assert call(tokens=0) == 0 and call(batch=0) == 0
    ws = lib.vl_paged_attention_workspace_bytes
    assert ws(4, 4, 1, 16, 4, 128, 2) > 0
    assert ws(4, 4, 1, 15, 4, 128, 2) == 0 and ws(4, 4, 0, 16, 4, 128, 2) == 0
    assert ws(4, 4, 1, 16, 4, 100, 2) == 0 and ws(-1, 4, 1, 16, 4, 128, 2) == 0


def test_select_rejects(lib):
    eos = (ctypes.c_int64 * 2)(1, 2)

    def call(lg=FAR, batch=2, beams=4, vocab=1000, rs=1000, sc=FAKE, fin=None, n_eos=2, pad=0,
             tok=2 * FAR, par=3 * FAR, so=4 * FAR, fo=5 * FAR, dtype=2, ws=6 * FAR, wsb=1 << 30):
        return lib.vl_beam_select(lg, batch, beams, vocab, rs, sc, fin, eos, n_eos, pad, tok, par,
                                  so, fo, dtype, ws, wsb, None)

    assert call(lg=None) == 2 and "null" in _err(lib)
    assert call(so=None) == 2 and "null" in _err(lib)
    assert call(dtype=3) == 2 and "dtype" in _err(lib)
    for beams in (0, 33):
        assert call(beams=beams) == 2 and "beams" in _err(lib)
    assert call(batch=20000) == 2 and "batch" in _err(lib)
    assert call(vocab=0) == 2 and "vocab" in _err(lib)
    assert call(vocab=(1 << 24) + 1, rs=1 << 25) == 2 and "vocab" in _err(lib)
    assert call(rs=999) == 2 and "stride" in _err(lib)
    assert call(lg=FAR + 1) == 2 and "aligned" in _err(lib)
    assert call(n_eos=9) == 2 and "n_eos" in _err(lib)
    assert call(pad=1000) == 2 and "pad_id" in _err(lib)
    assert call(so=FAKE + 4) == 2 and "overlaps" in _err(lib)
    assert call(fin=5 * FAR + 1) == 2 and "overlaps" in _err(lib)
    assert call(wsb=16) == 2 and "workspace" in _err(lib)
    assert call(batch=0) == 0
    ws = lib.vl_beam_select_workspace_bytes
    assert ws(2, 4, 1000) > 0 and ws(0, 4, 1000) == 0 and ws(2, 33, 1000) == 0


def test_reorder_rejects(lib):
    def call(tab=FAR, par=FAKE, kvl=2 * FAR, first=FAKE, pool=32, batch=2, beams=4, mp=8, ts=8,
             out=3 * FAR, os_=8, ko=4 * FAR, kc=5 * FAR, vc=6 * FAR, layers=2, pages=64, ps=16,
             row=1024, pstride=16 * 1024, lstride=64 * 16 * 1024):
        return lib.vl_paged_beam_reorder(tab, par, kvl, first, pool, batch, beams, mp, ts, out,
                                         os_, ko, kc, vc, layers, pages, ps, row, pstride,
                                         lstride, None, None)

    assert call(par=None) == 2 and "null" in _err(lib)
    assert call(kc=None) == 2 and "null" in _err(lib)
    assert call(beams=33) == 2 and "beams" in _err(lib)
    assert call(mp=4097, ts=5000, os_=5000) == 2 and "max_pages" in _err(lib)
    assert call(os_=7) == 2 and "strides" in _err(lib)
    assert call(pool=16385) == 2 and "pool_pages" in _err(lib)
    assert call(ps=17) == 2 and "page_size" in _err(lib)
    assert call(layers=-1) == 2 and "layers" in _err(lib)
    assert call(row=1023) == 2 and "row_bytes" in _err(lib)
    assert call(pstride=1024) == 2 and "page_stride_bytes" in _err(lib)
    assert call(out=FAR) == 2 and "overlap" in _err(lib)
    assert call(ko=2 * FAR + 4) == 2 and "overlap" in _err(lib)
    assert call(batch=0) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 8)
    with pytest.raises(vlasr.VlasrInputError, match="CUDA"):
        vlasr.beam_select(x, torch.zeros(2, 2))
    with pytest.raises(vlasr.VlasrInputError, match="CUDA"):
        vlasr.paged_attention(x, x, x, x, x, x, max_q_len=1)
    with pytest.raises(vlasr.VlasrInputError, match="CUDA"):
        vlasr.paged_rope_append(None, x, x, x, x, x, x, x)
    with pytest.raises(vlasr.VlasrInputError, match="CUDA"):
        vlasr.paged_beam_reorder(x, x, x, x, 1, x, x)


# ---------------------------------------------------------------------------
# the plain statements themselves
# ---------------------------------------------------------------------------

def test_plain_rotation_turns_pairs():
    x = np.array([[1.0, 0.0, 0.0, 0.0, 7.0]])
    half = paged_ref.rotate(x, 3, 4, 100.0, False, 0.5)
    assert np.allclose(half, [[math.cos(1.5), 0, math.sin(1.5), 0, 7.0]])
    inter = paged_ref.rotate(x, 3, 4, 100.0, True, 0.5)
    assert np.allclose(inter, [[math.cos(1.5), math.sin(1.5), 0, 0, 7.0]])
    second = paged_ref.rotate(np.array([[0, 1.0, 0, 0]]), 3, 4, 100.0, False, 1.0)
    assert np.allclose(second, [[0, math.cos(0.3), 0, math.sin(0.3)]])


def test_plain_attention_matches_softmax():
    rng = np.random.default_rng(0)
    kc, vc = rng.normal(size=(3, 16, 1, 4)), rng.normal(size=(3, 16, 1, 4))
    q = rng.normal(size=(2, 2, 4))
    table = np.array([[2, 0]])
    out, _ = paged_ref.attention(q, kc, vc, [0, 2], [18], table, 0.5, np.zeros((2, 2, 4)), 0.0)
    K = np.concatenate([kc[2], kc[0]])[:18, 0]
    V = np.concatenate([vc[2], vc[0]])[:18, 0]
    s = torch.softmax(torch.from_numpy(q[1] @ K.T * 0.5), -1).numpy()
    assert np.allclose(out[1], s @ V)
    s = torch.softmax(torch.from_numpy(q[0] @ K[:17].T * 0.5), -1).numpy()
    assert np.allclose(out[0], s @ V[:17])


def test_plain_select_matches_topk():
    rng = np.random.default_rng(1)
    lg = rng.normal(size=(6, 50))
    sc = -rng.random((2, 3))
    tok, par, val, _, _ = paged_ref.select(lg, sc, None, (), 0, 3)
    x = torch.log_softmax(torch.from_numpy(lg), -1).view(2, 3, 50) + torch.from_numpy(sc)[..., None]
    top = x.view(2, -1).topk(3, -1)
    assert np.allclose(val, top.values.numpy())
    assert np.array_equal(par * 50 + tok, top.indices.numpy())


def test_plain_reorder_keeps_copies_and_frees():
    # one entry, three beams, pages of 16; page 0 is the shared prompt
    kc = np.arange(8 * 16, dtype=np.float64).reshape(1, 8, 16, 1, 1)
    table = np.array([[0, 3, -1], [0, 4, -1], [0, 5, -1]], np.int32)
    out, lens, kc2, _, bad = paged_ref.reorder(table, np.array([[1, 1, 0]], np.int32),
                                               np.array([20, 20, 20], np.int32),
                                               np.array([3], np.int32), 4, kc, kc)
    assert out.tolist() == [[0, 4, -1], [0, 5, -1], [0, 3, -1]] and not bad
    assert lens.tolist() == [20, 20, 20]
    assert np.array_equal(kc2[0, 5, :4], kc[0, 4, :4])       # the copy
    assert np.array_equal(kc2[0, 5, 4:], kc[0, 5, 4:])
    out, _, kc3, _, _ = paged_ref.reorder(table, np.array([[0, 0, 0]], np.int32),
                                          np.array([16, 16, 16], np.int32),
                                          np.array([3], np.int32), 4, kc, kc)
    assert out[:, 1].tolist() == [3, 4, 5] and np.array_equal(kc3, kc)   # fresh pages, no copies


def test_trace_beams_follows_parents_and_stops_at_eos():
    from vlasr.decoder import trace_beams
    tokens = [[[10, 11]], [[12, 13]], [[9, 14]], [[9, 15]]]
    parents = [[[0, 0]], [[1, 0]], [[0, 1]], [[0, 1]]]
    hyps = trace_beams(tokens, parents, [[-3.0, -4.0]], eos_ids=(9,), length_penalty=1.0)
    assert hyps == [[([11, 12, 9], -3.0, -1.0), ([10, 13, 14, 15], -4.0, -1.0)]]
    ranked = trace_beams(tokens, parents, [[-3.0, -3.2]], eos_ids=(9,), length_penalty=1.0)
    assert ranked[0][0][0] == [10, 13, 14, 15]              # the longer one wins per id
    raw = trace_beams(tokens, parents, [[-3.0, -3.2]], eos_ids=(9,), length_penalty=0.0)
    assert raw[0][0][0] == [11, 12, 9]
    lost = trace_beams(tokens, parents, [[-3.0, float("-inf")]], eos_ids=(9,))
    assert [len(h) for h in lost] == [1]


def test_backend_passes_beams_on():
    from vlasr.backend import VlasrAsrBackend

    class Engine:
        def __init__(self):
            self.calls = []

        def transcribe_ids(self, pcm, prompt_ids, max_new_tokens=256, **more):
            self.calls.append(more)
            return [[1]] * len(pcm)

    class Processor:
        class tokenizer:
            @staticmethod
            def decode(ids, skip_special_tokens=True):
                return "word"

        def apply_transcription_request(self, arrays):
            return type("R", (), {"input_ids": [[1, 2]]})

    for beams, want in ((1, {}), (4, {"beams": 4})):
        engine = Engine()
        VlasrAsrBackend(engine=engine, processor=Processor(), beams=beams,
                        audio_loader=lambda path: np.ones(16000, np.float32)).transcribe("x", "en")
        assert engine.calls == [want]


def test_empty_calls_and_what_is_not_aligned(lib):
    """No tokens or no sequences: nothing to do, whatever the empty buffers'
    pointers; a buffer that is not aligned to its type is refused."""
    def append(tokens, batch, q=FAR, k=2 * FAR, kvl=FAKE, max_pages=8):
        return lib.vl_paged_rope_append(
            q, k, k and 3 * FAR, q and 4 * FAR, 5 * FAR, 6 * FAR, FAKE, kvl, kvl, tokens, batch,
            max_pages, max_pages, 16, 4, 128, 128, 0, 1e4, 1.0, 2048, 512, 512, 2048, 64, 16,
            16 * 512, 2, None, None)

    assert append(0, 2, q=None, k=None) == 0
    assert append(0, 0, q=None, k=None, kvl=None) == 0
    assert append(4, 0, kvl=None) == 0
    assert append(4, 2, kvl=None) == 2 and "null" in _err(lib)
    assert append(4, 2, k=2 * FAR + 1) == 2 and "aligned" in _err(lib)
    assert append(0, 2, max_pages=(1 << 27) - 15) == 2 and "num_pages" in _err(lib)
    assert append(0, 2, max_pages=(1 << 27) - 16) == 0

    def attend(tokens, batch, q=FAR, kvl=FAKE):
        return lib.vl_paged_attention(
            q, 5 * FAR, 6 * FAR, FAKE, kvl, kvl, tokens, batch, 1, 8, 8, 16, 4, 128, 0.0, 2048,
            2048, 64, 16, 16 * 512, q and 2 * FAR, 2, None, 0, None, 0, None)

    assert attend(0, 2, q=None) == 0 and attend(4, 0, kvl=None) == 0
    assert attend(4, 2, kvl=None) == 2 and "null" in _err(lib)
    eos = (ctypes.c_int64 * 1)(0)
    assert lib.vl_beam_select(None, 0, 4, 100, 100, None, None, eos, 0, 0, None, None, None, None,
                              2, None, 0, None) == 0
    assert lib.vl_paged_beam_reorder(None, None, None, None, 4, 0, 4, 8, 8, None, 8, None,
                                     5 * FAR, 6 * FAR, 2, 64, 16, 1024, 16384, 1 << 20, None,
                                     None) == 0


def test_attention_rejects_more_tiles_than_are_counted(lib):
    """64-position tiles times kv heads of a sequence are counted in 31 bits."""
    def call(nkv, max_pages):
        return lib.vl_paged_attention(
            FAR, 5 << 40, 6 << 40, FAKE, FAKE, FAKE, 1, 1, 1, max_pages, max_pages, nkv, nkv, 64,
            0.0, nkv * 64, nkv * 64, 4, 256, 256 * nkv * 64, 2 * FAR, 2, None, 0, None, 0, None)

    most = ((1 << 31) - 1) // (4 * 128)            # pages of four tiles, 128 kv heads
    assert call(128, most + 1) == 2 and "tiles" in _err(lib)
    assert call(128, most) == 2 and "workspace" in _err(lib)
    assert call(63, (1 << 23) - 1) == 2 and "workspace" in _err(lib)


def test_append_rejects_rows_past_31_bits(lib):
    """A token's elements, q, k and v together, are counted in an int."""
    def call(nq, nkv=4, hd=128):
        return lib.vl_paged_rope_append(
            1 << 56, 1 << 57, 1 << 58, 1 << 59, 1 << 60, 1 << 61, FAKE, FAKE, FAKE, 1, 0, 8, 8, nq,
            nkv, hd, 0, 0, 1e4, 1.0, 1 << 40, 1 << 40, 1 << 40, 1 << 40, 64, 16, 1 << 40, 2, None,
            None)

    assert call((1 << 24) - 8) == 2 and "elements" in _err(lib)
    assert call(1, 65535, 1 << 15) == 2 and "elements" in _err(lib)
    assert call((1 << 24) - 9) == 2 and "elements" in _err(lib)
    assert call((1 << 24) - 10) == 0


def test_append_rejects_outputs_over_inputs(lib):
    """q_out may be q; over k, v or a cache it would be read back or appended
    over, and so would a cache that lies over q, k or v."""
    def call(q=FAR, k=2 * FAR, v=3 * FAR, qo=4 * FAR, kc=5 * FAR, vc=6 * FAR, tokens=4, batch=0,
             qs=2048, ks=512, os_=2048):
        return lib.vl_paged_rope_append(
            q, k, v, qo, kc, vc, FAKE, FAKE, FAKE, tokens, batch, 8, 8, 16 if q else 0, 4, 128, 128,
            0, 1e4, 1.0, qs, ks, ks, os_, 64, 16, 16 * 512, 2, None, None)

    assert call() == 0 and call(qo=FAR) == 0
    for over in (2, 3, 5, 6):
        assert call(qo=over * FAR) == 2 and "overlap" in _err(lib)
        assert call(qo=over * FAR + 1024) == 2 and "overlap" in _err(lib)
    for name in ("q", "k", "v"):
        for cache in (5, 6):
            assert call(**{name: cache * FAR + 4096}) == 2 and "overlap" in _err(lib)
    # the columns of one projection, rotated in place
    packed = dict(q=FAR, k=FAR + 4096, v=FAR + 5120, qo=FAR, qs=3080, ks=3080, os_=3080)
    assert call(**packed) == 0
    assert call(**{**packed, "qo": FAR + 4096, "tokens": 1}) == 2 and "overlap" in _err(lib)
    # k and v may be the same rows; a last row of q_out that ends where k begins is apart
    assert call(k=3 * FAR) == 0
    assert call(k=4 * FAR + 4 * 4096) == 0 and call(k=4 * FAR + 4 * 4096 - 16) == 2
    assert call(q=None, qo=None) == 0


def test_select_status_word(lib, monkeypatch):
    """vl_beam_select_status refuses what vl_beam_select does, and the wrapper
    hands its status word over."""
    eos = (ctypes.c_int64 * 1)(1)

    def call(pad=0, batch=2, ws=6 * FAR):
        return lib.vl_beam_select_status(FAR, batch, 4, 1000, 1000, FAKE, None, eos, 1, pad,
                                         2 * FAR, 3 * FAR, 4 * FAR, None, 2, ws, 1 << 30,
                                         7 * FAR, None)

    assert call(pad=1000) == 2 and "pad_id" in _err(lib)
    assert call(ws=None) == 2 and "workspace" in _err(lib)
    assert call(batch=0) == 0

    seen = []

    class Fake:
        vl_beam_select_workspace_bytes = staticmethod(lambda *a: 16)
        vl_beam_select_status = staticmethod(lambda *a: seen.append(a) or 0)

    from vlasr import paged
    monkeypatch.setattr(paged, "_lead", lambda t, name: (0, t.dtype, t.get_device()))
    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged._lib, "load", lambda: Fake)
    status = torch.zeros(1, dtype=torch.int32)
    paged.beam_select(torch.zeros(2, 9), torch.zeros(1, 2), status=status)
    paged.beam_select(torch.zeros(2, 9), torch.zeros(1, 2))
    assert seen[0][-2] == status.data_ptr() and seen[1][-2] is None
    with pytest.raises(vlasr.VlasrInputError, match="status"):
        paged.beam_select(torch.zeros(2, 9), torch.zeros(1, 2), status=status.long())


def _stub_decoder(monkeypatch, layers=2):
    """A TextDecoder of CPU tensors whose operators are stand-ins."""
    from types import SimpleNamespace

    from vlasr import decoder
    dec = object.__new__(decoder.TextDecoder)
    dec.shape = SimpleNamespace(heads=2, kv_heads=1, head_dim=64, hidden=64, eps=1e-5, layers=layers,
                                rope_base=1e4)
    dec.fused, dec.device, dec.eos_ids, dec.embed = False, torch.device("cpu"), (3,), None
    dec.dtype, dec._states = torch.float32, {}
    dec.layer_w = [{"ln1": None, "qkv_t": torch.zeros(64, 256), "o_t": torch.zeros(128, 64)}
                   for _ in range(layers)]
    dec._mlp = lambda lw, h, a: a
    monkeypatch.setattr(decoder.ops, "add_rmsnorm", lambda h, d, w, eps: h)
    return dec, decoder


def test_beam_search_hands_its_status_to_every_call(monkeypatch):
    """What the operators of a step report reaches the word that
    generate_beam looks at."""
    dec, decoder = _stub_decoder(monkeypatch)
    seen = []

    def op(name, result):
        def call(*args, **kw):
            seen.append((name, kw.get("status")))
            return result(*args)
        return call

    monkeypatch.setattr(decoder.paged, "paged_rope_append", op("append", lambda q, *a: q))
    monkeypatch.setattr(decoder.paged, "paged_attention", op("attend", lambda q, *a: q))
    monkeypatch.setattr(decoder.paged, "beam_select", op("select", lambda *a: None))
    monkeypatch.setattr(decoder.paged, "paged_beam_reorder", op("reorder", lambda *a: None))
    i32 = torch.zeros(1, 2, dtype=torch.int32)
    st = {k: i32 for k in ("table", "next_table", "held", "next_held", "parents", "scores",
                           "finished", "tokens", "pool_start")}
    st.update(k_cache=[None] * 2, v_cache=[None] * 2, pool_pages=1, status=torch.zeros(1),
              step=torch.zeros(1, dtype=torch.int64), all_tokens=torch.zeros(3, 1, 2),
              all_parents=torch.zeros(3, 1, 2))
    st["all_tokens"], st["all_parents"] = (t.to(torch.int32) for t in (st["all_tokens"],
                                                                       st["all_parents"]))
    dec._paged_layers(torch.zeros(2, 64), st, i32, i32, i32, 1)
    dec._beam_select(st, torch.zeros(2, 9))
    assert [n for n, _ in seen] == ["append", "attend"] * 2 + ["select", "reorder"]
    assert all(s is st["status"] for _, s in seen)


def test_a_chunk_without_a_hypothesis_is_an_error(monkeypatch):
    """Beams that all ended at -inf (logits that are not finite) are no
    transcription."""
    dec, _ = _stub_decoder(monkeypatch)
    st = {"all_tokens": torch.tensor([[[5, 6], [7, 3]]]), "all_parents": torch.zeros(1, 2, 2).int(),
          "scores": torch.tensor([[-1.0, -2.0], [-0.5, -math.inf]])}
    ids, steps, hyps = dec._beam_collect(st, 1, 1.0)
    assert ids == [[5], [7]] and steps == 1 and [len(h) for h in hyps] == [2, 1]
    st["scores"][1, 0] = -math.inf
    with pytest.raises(vlasr.VlasrExecutionError, match=r"chunks \[1\]"):
        dec._beam_collect(st, 1, 1.0)


def test_wrappers_tell_their_own_errors_from_wrong_arguments(monkeypatch):
    """An argument that is no tensor is an input error; an AttributeError with
    tensors in every place is not called one."""
    from vlasr import paged
    x = torch.zeros(4, 8)
    for bad in (None, 3, [1.0]):
        with pytest.raises(vlasr.VlasrInputError, match="k is not a torch.Tensor"):
            vlasr.paged_rope_append(None, bad, x, x, x, x, x, x)
    with pytest.raises(vlasr.VlasrInputError, match="scores is not a torch.Tensor"):
        monkeypatch.setattr(paged, "_lead", lambda t, name: (0, t.dtype, t.get_device()))
        vlasr.beam_select(x, scores=[[0.0, 0.0]] * 2)

    def broken(t, name):
        raise AttributeError("no such helper")

    monkeypatch.setattr(paged, "_lead", broken)
    with pytest.raises(AttributeError, match="no such helper"):
        vlasr.beam_select(x, torch.zeros(2, 2))
    with pytest.raises(AttributeError, match="no such helper"):
        vlasr.paged_rope_append(None, x, x, x, x, x, x, x)


def test_beams_below_one_are_refused():
    """Not taken for greedy decoding."""
    from vlasr.engine import AsrEngine, transcribe_ids_sharded
    engine = object.__new__(AsrEngine)
    for beams in (0, -2):
        with pytest.raises(vlasr.VlasrInputError, match="beams"):
            engine.transcribe_ids(np.zeros(16, np.float32), [1], beams=beams)
        with pytest.raises(vlasr.VlasrInputError, match="beams"):
            transcribe_ids_sharded(engine, np.zeros((1, 16), np.float32), [1], beams=beams)


def test_backend_does_not_take_no_beams_for_greedy():
    from vlasr.backend import VlasrAsrBackend

    class Engine:
        def transcribe_ids(self, pcm, prompt_ids, max_new_tokens=256, beams=1):
            if beams < 1:
                raise vlasr.VlasrInputError("beams")
            return [[1]] * len(pcm)

    class Processor:
        class tokenizer:
            @staticmethod
            def decode(ids, skip_special_tokens=True):
                return "word"

        def apply_transcription_request(self, arrays):
            return type("R", (), {"input_ids": [[1, 2]]})

    backend = VlasrAsrBackend(engine=Engine(), processor=Processor(), beams=0,
                              audio_loader=lambda path: np.ones(16000, np.float32))
    with pytest.raises(Exception, match="beams"):
        backend.transcribe("x", "en")


def test_sizes_of_zero_are_input_errors(monkeypatch):
    from vlasr import paged
    empty = torch.zeros(2, 16, 1, 0)
    with pytest.raises(vlasr.VlasrInputError, match="head_dim"):
        paged._cache_pages(empty, empty)
    dec, _ = _stub_decoder(monkeypatch)
    dec.max_seq_len = 64
    for page_size in (0, -16, 8, 48, 512):
        with pytest.raises(vlasr.VlasrInputError, match="page_size"):
            dec.generate_beam(torch.zeros(1, 375, 64), [1, 2], beams=2, max_new_tokens=4,
                              page_size=page_size)


def test_exponential_polynomial():
    """2^f on [-1/2, 1/2] by the coefficients that the kernel holds, in fp32 with
    fused steps as there: within the 2.2e-7 that its comment states."""
    import re

    from conftest import PKG
    text = (PKG / "csrc" / "vl_paged_attn_tc.cu").read_text()
    body = text[text.index("float2 ex2_pair"):text.index("halves_of(p)")]
    cf = [np.float32(x) for x in re.findall(r"pair_of\((0\.\d+|1\.\d+)f, \1f\)", body)]
    assert len(cf) == 6
    f = np.linspace(-0.5, 0.5, 400001).astype(np.float32)
    p = np.full_like(f, cf[0])
    for c in cf[1:]:
        p = (p.astype(np.float64) * f + np.float64(c)).astype(np.float32)
    off = np.abs(p.astype(np.float64) / np.exp2(f.astype(np.float64)) - 1)
    assert off.max() <= 2.2e-7


def test_wrong_arguments_on_another_device_are_input_errors(monkeypatch):
    """The call is made again under the tensors' device; its checks are the same."""
    import contextlib

    from vlasr import paged
    under = []

    @contextlib.contextmanager
    def device(index):
        under.append(index)
        yield
        under.pop()

    def lead(t, name):
        if not under:
            raise paged._OtherDevice(3)
        return 0, t.dtype, t.get_device()

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(paged, "_lead", lead)
    with pytest.raises(vlasr.VlasrInputError, match="scores is not a torch.Tensor"):
        vlasr.beam_select(torch.zeros(2, 8), [[0.0, 0.0]])
