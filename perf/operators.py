"""Cases of the paged-cache decoding operators, with their plain forms.

Four operators that a beam-search decode over a paged KV cache is made of:

  append    vlasr.paged_rope_append    rotate q and k, store k and v through a page table
  attend    vlasr.paged_attention      causal attention of each sequence's new tokens over its pages
  select    vlasr.beam_select          best `beams` continuations of each entry's beams
  reorder   vlasr.paged_beam_reorder   page tables of the chosen parents, shared pages split by copying

With `own` false, `run` computes each of them from elementary torch
operations; with `own` true it makes the calls a user of the package makes.
`exact` computes them in 64 bits.
"""

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _vlasr():
    """The package, which lives beside this folder."""
    pkg = str(Path(__file__).resolve().parent.parent / "videolingo-user_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import vlasr
    return vlasr


def _device():
    return torch.device("cuda:0")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The rotation and append of one decode step of 16 chunks: 16 query
        # and 4 kv heads of 128, the smallest call, where latency counts.
        {"name": "append_step_16", "op": "append", "dtype": "bf16", "seqs": 16, "q_min": 1,
         "q_max": 1, "past_min": 384, "past_max": 640, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "position_scale": 1.0, "page": 32, "pad": 0,
         "mix": 1},
        # Prefill of 16 chunks: 375 audio tokens and a short prompt each.
        {"name": "append_prefill_16x383", "op": "append", "dtype": "bf16", "seqs": 16,
         "q_min": 383, "q_max": 383, "past_min": 0, "past_max": 0, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "rotary_dim": 128, "interleaved": False, "position_scale": 1.0,
         "page": 32, "pad": 0, "mix": 2},
        # Ragged chunks of long recordings, interleaved pairs over half of
        # each 64-wide head, positions compressed by four, with padding rows
        # behind the last sequence.
        {"name": "append_ragged_interleaved", "op": "append", "dtype": "f16", "seqs": 37,
         "q_min": 1, "q_max": 1501, "past_min": 0, "past_max": 2050, "heads": 20, "kv_heads": 5,
         "head_dim": 64, "rotary_dim": 32, "interleaved": True, "position_scale": 0.25, "page": 16,
         "pad": 13, "mix": 3},
        # One decode step of a single chunk with four beams.
        {"name": "attend_step_4", "op": "attend", "dtype": "bf16", "seqs": 4, "q_min": 1,
         "q_max": 1, "past_min": 400, "past_max": 600, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "page": 32, "pad": 0, "mix": 4},
        # One decode step of 64 sequences of up to 4096 positions.
        {"name": "attend_step_64x4096", "op": "attend", "dtype": "bf16", "seqs": 64, "q_min": 1,
         "q_max": 1, "past_min": 0, "past_max": 4095, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "page": 64, "pad": 0, "mix": 5},
        # Prefill attention of 16 chunks.
        {"name": "attend_prefill_16x383", "op": "attend", "dtype": "bf16", "seqs": 16,
         "q_min": 383, "q_max": 383, "past_min": 0, "past_max": 0, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "page": 32, "pad": 0, "mix": 6},
        # A chunk of a long transcript's prompt against what is cached of it.
        {"name": "attend_chunk_2048_of_16k", "op": "attend", "dtype": "bf16", "seqs": 1,
         "q_min": 2048, "q_max": 2048, "past_min": 14336, "past_max": 14336, "heads": 16,
         "kv_heads": 4, "head_dim": 128, "page": 128, "pad": 0, "mix": 7},
        # Ragged chunks beside single tokens, 64-wide heads in groups of
        # five, with padding rows behind the last sequence.
        {"name": "attend_ragged_f16", "op": "attend", "dtype": "f16", "seqs": 23, "q_min": 1,
         "q_max": 701, "past_min": 0, "past_max": 1301, "heads": 20, "kv_heads": 4, "head_dim": 64,
         "page": 16, "pad": 7, "mix": 8},
        # The selection of one chunk with four beams over the model's vocabulary.
        {"name": "select_1x4", "op": "select", "dtype": "bf16", "batch": 1, "beams": 4,
         "vocab": 59264, "done": 0.0, "masked": 0.0, "mix": 9},
        # The selection of 64 chunks with five beams, some of them finished,
        # an odd vocabulary and suppressed tokens.
        {"name": "select_64x5", "op": "select", "dtype": "f32", "batch": 64, "beams": 5,
         "vocab": 51865, "done": 0.2, "masked": 0.02, "mix": 10},
        # Beams of four chunks after a step: 28 layers of 16-token pages.
        {"name": "reorder_4x4", "op": "reorder", "dtype": "bf16", "batch": 4, "beams": 4,
         "layers": 28, "kv_heads": 4, "head_dim": 128, "page": 16, "prompt": 383, "made_min": 3,
         "made_max": 90, "max_pages": 40, "mix": 11},
        # Beams of 32 chunks after a step, the caches of 28 layers.
        {"name": "reorder_32x5", "op": "reorder", "dtype": "f16", "batch": 32, "beams": 5,
         "layers": 28, "kv_heads": 4, "head_dim": 128, "page": 32, "prompt": 383, "made_min": 1,
         "made_max": 40, "max_pages": 16, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "select", "reorder"])
    mix = rng.randrange(1 << 30)
    if op in ("append", "attend"):
        head_dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        q_max = rng.choice([1, _log_int(rng, 2, 2048)])
        q_min = rng.choice([1, q_max])
        past_max = rng.choice([0, _log_int(rng, 1, 14336 if q_max > 1 else 16384)])
        # bounded by the listed sizes: about 4 M cached (token, head) rows and
        # as many products as the long chunk's
        seqs = _log_int(rng, 1, 64)
        while seqs > 1 and (seqs * (q_max + past_max) * kv_heads > 1 << 20 or
                            seqs * q_max * (past_max + q_max) * heads > 1 << 28 or
                            seqs * q_max * heads > 1 << 17):
            seqs = seqs // 2
        while q_max * (past_max + q_max) * heads > 1 << 29:
            past_max //= 2
            q_max = max(1, q_max // 2)
            q_min = min(q_min, q_max)
        case = {"op": op, "dtype": rng.choice(["bf16", "f16"] + (["f32"] if op == "append" else [])),
                "seqs": seqs, "q_min": q_min, "q_max": q_max,
                "past_min": rng.choice([0, past_max]), "past_max": past_max, "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128]),
                "pad": rng.choice([0, 0, rng.randrange(1, 33)]), "mix": mix}
        if op == "append":
            case["rotary_dim"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 48])
            case["interleaved"] = rng.random() < 0.5
            case["position_scale"] = rng.choice([1.0, 1.0, 0.5, 0.125])
        return case
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = rng.choice([59264, 51865, _log_int(rng, 500, 130000)])
        batch = _log_int(rng, 1, 64)
        while batch > 1 and batch * beams * vocab > 320 * 51865:
            batch //= 2
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch,
                "beams": beams, "vocab": vocab, "done": rng.choice([0.0, 0.3]),
                "masked": rng.choice([0.0, 0.05]), "mix": mix}
    page = rng.choice([16, 32, 64])
    beams = rng.choice([2, 3, 4, 5, 8])
    layers = rng.choice([1, 4, 12, 28])
    prompt = _log_int(rng, 1, 1000)
    made_max = _log_int(rng, 1, 100)
    batch = _log_int(rng, 1, 32)
    while batch > 1 and batch * beams * layers > 32 * 5 * 28:
        batch //= 2
    return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch, "beams": beams,
            "layers": layers, "kv_heads": rng.choice([1, 2, 4]), "head_dim": rng.choice([64, 128]),
            "page": page, "prompt": prompt, "made_min": rng.choice([0, made_max // 2, made_max]),
            "made_max": made_max, "max_pages": -(-(prompt + made_max + 2) // page) + rng.randrange(3),
            "mix": mix}


def _lengths(case):
    """New tokens and cached positions of each sequence, from the case alone."""
    r = random.Random(case["mix"])
    new, past = [], []
    for _ in range(case["seqs"]):
        new.append(r.randint(case["q_min"], case["q_max"]))
        past.append(r.randint(case["past_min"], case["past_max"]))
    return new, past


def _reorder_shape(case):
    """Per entry: positions held before the call (the same for its beams)."""
    r = random.Random(case["mix"])
    return [case["prompt"] + r.randint(case["made_min"], case["made_max"])
            for _ in range(case["batch"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=_device(), dtype=torch.float32) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=_device())
    gen.manual_seed(int(seed) * 1000003 + case["mix"])
    if case["op"] in ("append", "attend"):
        return _prepare_cache(case, gen, seed)
    if case["op"] == "select":
        return _prepare_select(case, gen, seed)
    return _prepare_reorder(case, gen, seed)


def _prepare_cache(case, gen, seed):
    dev, dt = _device(), DTYPES[case["dtype"]]
    new, past = _lengths(case)
    page, hd = case["page"], case["head_dim"]
    qw, kw = case["heads"] * hd, case["kv_heads"] * hd
    lens = [n + p for n, p in zip(new, past)]
    per = [-(-n // page) for n in lens]
    max_pages = max(per) + 1
    total = sum(per) + 2
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    table = torch.full((case["seqs"], max_pages), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    tokens = sum(new) + case["pad"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    # q, k and v are the columns of one packed projection, as a decoder layer has them
    qkv = _normal(gen, (tokens, qw + 2 * kw), dt)
    s = {"case": case, "new": new, "past": past,
         "q_start": torch.tensor(starts, dtype=torch.int32, device=dev),
         "kv_len": torch.tensor(lens, dtype=torch.int32, device=dev), "table": table,
         "q": qkv[:, :qw], "k": qkv[:, qw:qw + kw], "v": qkv[:, qw + kw:],
         "k_cache": _normal(gen, (total, page, case["kv_heads"], hd), dt),
         "v_cache": _normal(gen, (total, page, case["kv_heads"], hd), dt),
         "out": torch.zeros((tokens, qw), dtype=dt, device=dev),
         "max_q_len": case["q_max"], "vl": _vlasr() if own else None}
    return s


def _prepare_select(case, gen, seed):
    dev, dt = _device(), DTYPES[case["dtype"]]
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    rows = batch * beams
    logits = torch.randn((rows, vocab), generator=gen, device=dev) * 2.0 - 4.0
    # a speech model's step: a handful of tokens carry most of the mass
    top = torch.randint(0, vocab, (rows, 12), generator=gen, device=dev)
    lift = 6.0 + 8.0 * torch.rand((rows, 12), generator=gen, device=dev)
    logits.scatter_(1, top, lift)
    if case["masked"] > 0:
        logits[torch.rand((rows, vocab), generator=gen, device=dev) < case["masked"]] = -math.inf
    scores = -torch.rand((batch, beams), generator=gen, device=dev) * 12.0
    finished = torch.rand((batch, beams), generator=gen, device=dev) < case["done"]
    eos = [vocab - 18, vocab - 11, vocab - 9]
    for i, e in enumerate(eos):  # ends come up as candidates now and then
        logits[i::7, e] = 9.5 + i
    return {"case": case, "logits": logits.to(dt), "scores": scores, "finished": finished,
            "eos": eos, "pad_id": eos[1], "vl": _vlasr() if own else None}


def _prepare_reorder(case, gen, seed):
    dev, dt = _device(), DTYPES[case["dtype"]]
    batch, beams, page = case["batch"], case["beams"], case["page"]
    held = _reorder_shape(case)
    full = case["prompt"] // page            # whole prompt pages, shared by the beams
    pool = beams * (case["max_pages"] - full)
    total = batch * (full + pool)
    table = torch.full((batch, beams, case["max_pages"]), -1, dtype=torch.int32, device=dev)
    r = random.Random(int(seed) * 7919 + case["mix"])
    parents = []
    for b in range(batch):
        base = batch * full + b * pool
        table[b, :, :full] = torch.arange(b * full, (b + 1) * full, dtype=torch.int32, device=dev)
        pages = list(range(base, base + pool))
        r.shuffle(pages)
        wp = held[b] // page
        rows = [[] for _ in range(beams)]
        for j in range(full, wp + 1):
            # a page that is full is often shared by several beams; the last is each beam's own
            ids = [pages.pop() for _ in range(beams)] if j == wp else None
            if ids is None:
                one = [pages.pop() for _ in range(r.randint(1, beams))]
                ids = [r.choice(one) for _ in range(beams)]
            for i in range(beams):
                rows[i].append(ids[i])
        last = wp + 1 if held[b] % page else wp
        if last > full:
            table[b, :, full:last] = torch.tensor([x[:last - full] for x in rows],
                                                  dtype=torch.int32, device=dev)
        alive = [r.randrange(beams) for _ in range(max(1, beams - 1))]
        parents.append([r.choice(alive) for _ in range(beams)])
    shape = (case["layers"], total, page, case["kv_heads"], case["head_dim"])
    return {"case": case,
            "table": table.view(batch * beams, -1),
            "parents": torch.tensor(parents, dtype=torch.int32, device=dev),
            "kv_len": torch.tensor(held, dtype=torch.int32, device=dev).repeat_interleave(beams),
            "pool_start": torch.arange(batch, dtype=torch.int32, device=dev) * pool + batch * full,
            "pool_pages": pool, "k_cache": _normal(gen, shape, dt),
            "v_cache": _normal(gen, shape, dt), "vl": _vlasr() if own else None}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return {"append": _append, "attend": _attend, "select": _select,
            "reorder": _reorder}[state["case"]["op"]](state)


def _append(s):
    c = s["case"]
    if own:
        s["vl"].paged_rope_append(
            s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["q_start"], s["kv_len"],
            s["table"], head_dim=c["head_dim"], rotary_dim=c["rotary_dim"], base=10000.0,
            interleaved=c["interleaved"], position_scale=c["position_scale"], q_out=s["out"])
        return {"q": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    dev, page = s["q"].device, c["page"]
    n = s["q_start"][-1:].long()
    tokens = s["q"].shape[0]
    t = torch.arange(tokens, device=dev)
    starts = s["q_start"].long()
    b = (t[:, None] >= starts[None, 1:]).sum(1).clamp(max=c["seqs"] - 1)
    live = t < n
    pos = s["kv_len"].long()[b] - (starts[b + 1] - t)
    pos = torch.where(live, pos, torch.zeros_like(pos))
    half = c["rotary_dim"] // 2
    freq = 10000.0 ** (-2.0 * torch.arange(half, device=dev, dtype=torch.float64) / c["rotary_dim"])
    angle = pos.double()[:, None] * c["position_scale"] * freq[None]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        y = x.reshape(tokens, -1, c["head_dim"]).float()
        r, rest = y[..., :2 * half], y[..., 2 * half:]
        if c["interleaved"]:
            a, e = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - e * sin, e * cos + a * sin), -1).flatten(-2)
        else:
            a, e = r[..., :half], r[..., half:]
            r = torch.cat((a * cos - e * sin, e * cos + a * sin), -1)
        return torch.cat((r, rest), -1).to(x.dtype)

    q, k = rotate(s["q"]), rotate(s["k"])
    v = s["v"].reshape(k.shape)
    real = tokens - c["pad"]
    s["out"][:real] = q.reshape(tokens, -1)[:real]
    slot_page = s["table"].long()[b, pos // page]
    at = slot_page[:real], (pos % page)[:real]
    s["k_cache"][at] = k[:real]
    s["v_cache"][at] = v[:real]
    return {"q": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s):
    c = s["case"]
    if own:
        return s["vl"].paged_attention(
            s["q"], s["k_cache"], s["v_cache"], s["q_start"], s["kv_len"], s["table"],
            max_q_len=s["max_q_len"], out=s["out"])
    hd, kvh, page = c["head_dim"], c["kv_heads"], c["page"]
    group = c["heads"] // kvh
    at = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        m = n + past
        ids = s["table"][b, :-(-m // page)].long()
        keys = s["k_cache"][ids].reshape(-1, kvh, hd)[:m].float().permute(1, 2, 0)
        vals = s["v_cache"][ids].reshape(-1, kvh, hd)[:m].float().permute(1, 0, 2)
        q = s["q"][at:at + n].reshape(n, kvh, group, hd).float()
        q = q.permute(1, 0, 2, 3).reshape(kvh, n * group, hd)
        w = torch.matmul(q, keys) * hd ** -0.5
        i = torch.arange(n, device=w.device).repeat_interleave(group)
        j = torch.arange(m, device=w.device)
        w = torch.where((j[None] > i[:, None] + past)[None], -math.inf, w)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        o = torch.matmul(w, vals) / w.sum(-1, keepdim=True)
        o = o.reshape(kvh, n, group, hd).permute(1, 0, 2, 3).reshape(n, -1)
        s["out"][at:at + n] = o.to(s["q"].dtype)
        at += n
    return s["out"]


def _select(s):
    c = s["case"]
    batch, beams, vocab = c["batch"], c["beams"], c["vocab"]
    if own:
        return s["vl"].beam_select(s["logits"], s["scores"], finished=s["finished"],
                                   eos_ids=s["eos"], pad_id=s["pad_id"])
    # in 64 bits: near ties between beams decide which one is taken
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    x = x - (m + torch.log(torch.exp(x - m).sum(1, keepdim=True)))
    x = x.reshape(batch, beams, vocab) + s["scores"].double()[..., None]
    done = s["finished"][..., None]
    x = torch.where(done | torch.isnan(x), -math.inf, x)
    held = torch.where(s["finished"], s["scores"].double(), -math.inf)
    x[:, :, s["pad_id"]] = torch.where(s["finished"], held, x[:, :, s["pad_id"]])
    x = x.reshape(batch, beams * vocab)
    tokens, parents, scores = [], [], []
    for i in range(beams):
        at = torch.argmax(x, 1, keepdim=True)  # the first of equal values
        best = torch.gather(x, 1, at)[:, 0]
        none = best == -math.inf
        tokens.append(torch.where(none, s["pad_id"], at[:, 0] % vocab))
        parents.append(torch.where(none, i, at[:, 0] // vocab))
        scores.append(best)
        x.scatter_(1, at, -math.inf)
    tokens, parents = torch.stack(tokens, 1), torch.stack(parents, 1)
    scores = torch.stack(scores, 1)
    ended = torch.gather(s["finished"], 1, parents) | (scores == -math.inf)
    for e in s["eos"]:
        ended = ended | (tokens == e)
    return tokens, parents.to(torch.int32), scores.float(), ended


def _reorder(s):
    c = s["case"]
    batch, beams, page = c["batch"], c["beams"], c["page"]
    if own:
        table, kv_len = s["vl"].paged_beam_reorder(
            s["table"], s["parents"], s["kv_len"], s["pool_start"], s["pool_pages"], s["k_cache"],
            s["v_cache"])
        return table, kv_len, s["k_cache"], s["v_cache"]
    dev, pages, pool = s["table"].device, c["max_pages"], s["pool_pages"]
    parents = s["parents"].long()
    src = torch.gather(s["table"].view(batch, beams, pages).long(), 1,
                       parents[..., None].expand(-1, -1, pages))
    held = torch.gather(s["kv_len"].view(batch, beams).long(), 1, parents)
    wp, fill = held // page, held % page
    j = torch.arange(pages, device=dev)
    whole = j < wp[..., None]
    out = torch.where(whole, src, -1)
    base = s["pool_start"].long()[:, None]
    part = torch.gather(src, 2, wp.clamp(max=pages - 1)[..., None])[..., 0]

    def mine(p):
        return (p >= base.view(-1, *[1] * (p.dim() - 1))) & (p < base.view(-1, *[1] * (p.dim() - 1)) + pool)

    used = torch.zeros((batch, pool + 1), dtype=torch.long, device=dev)
    spot = torch.where(whole & mine(src), src - base[..., None], pool).reshape(batch, -1)
    used.scatter_(1, spot, 1)
    read = torch.gather(used, 1, torch.where(mine(part), part - base, pool)) > 0
    i = torch.arange(beams, device=dev)
    earlier = ((part[:, :, None] == part[:, None, :]) & (i[None, None] < i[None, :, None])
               & (fill > 0)[:, None, :]).any(2)
    keep = (fill > 0) & mine(part) & ~read & ~earlier
    used.scatter_(1, torch.where(keep, part - base, pool), 1)
    free = torch.sort(used[:, :pool], dim=1, stable=True)[1]
    need = (wp < pages) & ~keep
    order = (torch.cumsum(need.long(), 1) - 1).clamp(min=0, max=pool - 1)
    fresh = torch.gather(free, 1, order) + base
    write = torch.where(keep, part, torch.where(need, fresh, -1))
    out.scatter_(2, wp.clamp(max=pages - 1)[..., None],
                 torch.where(wp < pages, write, out[..., -1])[..., None])
    # rows below `fill` of a shared page into the fresh one; a kept page onto itself
    from_page = torch.where(need & (fill > 0), part, write).reshape(-1)
    to_page = write.reshape(-1)
    moved = torch.arange(page, device=dev) < torch.where(need, fill, 0).reshape(-1, 1)
    for cache in (s["k_cache"], s["v_cache"]):
        cache[:, to_page] = torch.where(moved[None, ..., None, None], cache[:, from_page],
                                        cache[:, to_page])
    return (out.to(torch.int32).view(batch * beams, pages), held.to(torch.int32).view(-1),
            s["k_cache"], s["v_cache"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    es = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "append":
        new, _ = _lengths(case)
        n, hd = sum(new), case["head_dim"]
        # q, k and v read once; q, the cached k and v written once
        return {"bytes": 2 * n * (case["heads"] + 2 * case["kv_heads"]) * hd * es,
                "flops": 3 * n * (case["heads"] + case["kv_heads"]) * case["rotary_dim"]}
    if case["op"] == "attend":
        new, past = _lengths(case)
        hd = case["head_dim"]
        rows = sum(new) * case["heads"] * hd * es * 2
        cached = sum(n + p for n, p in zip(new, past)) * case["kv_heads"] * hd * es * 2
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        return {"bytes": rows + cached, "flops": 4 * pairs * case["heads"] * hd}
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        live = rows - int(rows * case["done"])
        return {"bytes": live * case["vocab"] * es + rows * 24, "flops": 3 * live * case["vocab"]}
    row = case["kv_heads"] * case["head_dim"] * es
    r = random.Random(case["mix"])
    filled = sum(h % case["page"] for h in _reorder_shape(case))
    # about half of an entry's beams share a parent: their part-filled pages
    # are read and written in every layer
    copied = filled * case["beams"] / 2 * case["layers"] * 2 * row * 2
    tables = case["batch"] * case["beams"] * case["max_pages"] * 8
    return {"bytes": copied + tables, "flops": 0}


# ---------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](s)


def _exact_append(s):
    c = s["case"]
    page, hd, half = c["page"], c["head_dim"], c["rotary_dim"] // 2
    out = s["out"].double()
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    table = s["table"].cpu().numpy()
    pair = torch.arange(half, device=out.device, dtype=torch.float64)
    first = (2 * pair if c["interleaved"] else pair).long()
    second = first + 1 if c["interleaved"] else first + half
    inverse = torch.exp(pair * (-2.0 / c["rotary_dim"]) * math.log(10000.0))
    t = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        where = np.arange(past, past + n)
        angle = torch.as_tensor(where, device=out.device).double()[:, None] * inverse
        turn = torch.polar(torch.ones_like(angle), angle * c["position_scale"])[:, None]

        def spin(x):
            y = x.reshape(n, -1, hd).double().clone()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out[t:t + n] = spin(s["q"][t:t + n]).reshape(n, -1)
        ids = torch.as_tensor(table[b][where // page].astype(np.int64), device=out.device)
        rows = torch.as_tensor(where % page, device=out.device)
        kc[ids, rows] = spin(s["k"][t:t + n])
        vc[ids, rows] = s["v"][t:t + n].reshape(n, -1, hd).double()
        t += n
    return {"q": out, "k_cache": kc, "v_cache": vc}


def _exact_attend(s):
    c = s["case"]
    hd, page = c["head_dim"], c["page"]
    group = c["heads"] // c["kv_heads"]
    out = s["out"].double()
    t = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        m = n + past
        slots = torch.arange(m, device=out.device)
        ids = s["table"][b].long()[slots // page]
        keys = s["k_cache"][ids, slots % page].double()
        vals = s["v_cache"][ids, slots % page].double()
        seen = torch.tril(torch.ones((n, m), dtype=torch.bool, device=out.device), diagonal=past)
        for h in range(c["heads"]):
            q = s["q"][t:t + n, h * hd:(h + 1) * hd].double()
            z = (q @ keys[:, h // group].T) / math.sqrt(hd)
            z = z.masked_fill(~seen, -math.inf)
            out[t:t + n, h * hd:(h + 1) * hd] = torch.softmax(z, -1) @ vals[:, h // group]
        t += n
    return out


def _exact_select(s):
    c = s["case"]
    batch, beams, vocab, pad = c["batch"], c["beams"], c["vocab"], s["pad_id"]
    logp = torch.log_softmax(s["logits"].double(), -1).view(batch, beams, vocab).cpu().numpy()
    score, done = s["scores"].double().cpu().numpy(), s["finished"].cpu().numpy()
    tokens = np.full((batch, beams), pad, np.int64)
    parents = np.tile(np.arange(beams, dtype=np.int64), (batch, 1))
    value = np.full((batch, beams), -np.inf)
    ended = np.ones((batch, beams), bool)
    for b in range(batch):
        found = []
        for i in range(beams):
            if done[b, i]:
                found.append((-score[b, i], i * vocab + pad))
                continue
            row = logp[b, i] + score[b, i]
            best = np.argpartition(-row, min(2 * beams, vocab - 1))[:2 * beams]
            cut = row[best].min()
            found += [(-row[v], i * vocab + int(v)) for v in np.nonzero(row >= cut)[0]
                      if row[v] > -np.inf]
        for k, (v, at) in enumerate(sorted(found)[:beams]):
            tokens[b, k], parents[b, k], value[b, k] = at % vocab, at // vocab, -v
            ended[b, k] = done[b, at // vocab] or at % vocab in s["eos"]
    return [torch.from_numpy(x) for x in (tokens, parents, value, ended)]


def _exact_reorder(s):
    c = s["case"]
    beams, page = c["beams"], c["page"]
    old, parents = s["table"].cpu().tolist(), s["parents"].cpu().tolist()
    lens, first = s["kv_len"].cpu().tolist(), s["pool_start"].cpu().tolist()
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    table, held = [], []
    for b in range(c["batch"]):
        rows = [b * beams + p for p in parents[b]]
        inside = range(first[b], first[b] + s["pool_pages"])
        readers = {p for r in rows for p in old[r][:lens[r] // page]}
        taken, kept = set(readers), {}
        for i, r in enumerate(rows):
            if lens[r] % page:
                p = old[r][lens[r] // page]
                if p in inside and p not in readers and p not in kept.values():
                    kept[i] = p
        taken |= set(kept.values())
        spare = iter([p for p in inside if p not in taken])
        for i, r in enumerate(rows):
            wp, fill = divmod(lens[r], page)
            new = old[r][:wp] + [-1] * (c["max_pages"] - wp)
            if wp < c["max_pages"]:
                new[wp] = kept[i] if i in kept else next(spare, -1)
                if i not in kept and fill and new[wp] >= 0:
                    kc[:, new[wp], :fill] = kc[:, old[r][wp], :fill]
                    vc[:, new[wp], :fill] = vc[:, old[r][wp], :fill]
            table.append(new)
            held.append(lens[r])
    return [torch.tensor(table), torch.tensor(held), kc, vc]
