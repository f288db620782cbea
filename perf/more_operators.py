"""Operators around the cache of a serving step, as a serving program calls them: rotary
positions, K/V written into pages (in 8 bits too) and read back, and the end of a beam
search's step.

With ``own`` false, ``run`` computes each operator in its plain form: elementary torch
operations in 32 bits (64 for angles and for scores that decide an order), rounded once at
the end.  With ``own`` true it makes the calls of the package's entry points.  Kinds:

  rotary   ``ia.apply_rotary``: queries and keys of packed tokens rotated to their positions
  write    ``ia.rotary_append_kv``: queries rotated, keys rotated into the pages, values into
           the pages; fp8 pages are scaled by what they hold, and what the touched pages
           then hold is read back (``ia.read_kv``), as a program does whose prompt attends
           the rounded rows
  read     ``ia.read_kv``: cached rows of sequences as packed tensors again
  select   ``ia.beam_select``: the best continuations over beams and vocabulary
  reorder  ``ia.reorder_sequences``: every beam's pages follow its parent's, in all layers

Values are those the path meets: unit-variance queries and values, keys with a scale per
(kv head, channel); pages in random order; logits with a spread of a few units.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f32": 4, "fp8": 1}
DEV = "cuda"
LARGEST_CODE = 448.0  # of e4m3
LOWEST_SCALE = 2.0 ** -126


# ------------------------------------------------------------------ the cases

def listed():
    gqa = {"hkv": 8, "g": 4, "d": 128}
    rotary = {"rot": 128, "layout": "half", "base": 500000.0, "scaling": "none", "factor": 1.0}
    return [
        # one decode step's queries and keys: latency
        dict(gqa, **rotary, name="rotary 32", kind="rotary", n=32, far=130000, dt="bf16", fused=True, len_seed=0),
        # packed prompts of a model with stretched positions, far out; a quarter of a head is not rotated
        dict(name="rotary 24001 far", kind="rotary", hkv=4, g=8, d=128, rot=96, layout="interleaved", base=10000.0,
             scaling="yarn", factor=16.0, n=24001, far=1000000, dt="bf16", fused=True, len_seed=1),
        # one decode step into an 8-bit cache: latency
        dict(gqa, **rotary, name="write fp8 32x1", kind="write", n=32, lo=1, hi=1, past_lo=500, past_hi=8000, kv="fp8",
             page=16, pool="split", fused=True, single=True, len_seed=2),
        # a batch of prompts into an 8-bit cache
        dict(gqa, name="write fp8 16x500-4000", kind="write", rot=128, layout="half", base=500000.0, scaling="llama3",
             factor=8.0, n=16, lo=500, hi=4000, past_lo=0, past_hi=300, kv="fp8", page=16, pool="split", fused=True,
             single=False, len_seed=3),
        # short ragged prompts, small heads, pages of 32 with keys and values side by side
        dict(name="write 12x1-900", kind="write", hkv=4, g=8, d=64, rot=32, layout="interleaved", base=10000.0,
             scaling="none", factor=1.0, n=12, lo=1, hi=900, past_lo=0, past_hi=2000, kv="bf16", page=32, pool="paired",
             fused=False, single=False, len_seed=4),
        # the last tokens of four sequences of an 8-bit cache
        dict(gqa, name="read fp8 4x1-600", kind="read", n=4, lo=1, hi=600, past_lo=0, past_hi=3000, kv="fp8", page=16,
             pool="paired", len_seed=5),
        # whole sequences moved out of the cache
        dict(gqa, name="read 8x4k-16k", kind="read", n=8, lo=4000, hi=16000, past_lo=0, past_hi=0, kv="bf16", page=16,
             pool="split", len_seed=6),
        # one request's four beams, twice as many candidates as beams
        dict(name="select 1x4 of 32000", kind="select", batch=1, beams=4, n=8, vocab=32000, dt="f32", done=False,
             len_seed=7),
        # sixteen requests, an odd vocabulary, some beams have ended
        dict(name="select 16x5 of 50021", kind="select", batch=16, beams=5, n=5, vocab=50021, dt="bf16", done=True,
             len_seed=8),
        # a large batch over a large vocabulary
        dict(name="select 64x8 of 128000", kind="select", batch=64, beams=8, n=16, vocab=128000, dt="bf16", done=False,
             len_seed=9),
        # one request of four beams, 24 layers: latency
        dict(name="reorder 1x4 at 900", kind="reorder", hkv=8, d=128, page=16, kv="bf16", layers=24, groups=1, ways=4,
             lo=900, hi=900, tail=37, spare=20, len_seed=10),
        # sixteen requests of eight beams each, eight layers of an 8-bit cache
        dict(name="reorder 16x8 at 2k-9k", kind="reorder", hkv=8, d=128, page=16, kv="fp8", layers=8, groups=16, ways=8,
             lo=2000, hi=9000, tail=150, spare=100, len_seed=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rotary(rng, d):
    scaling = rng.choice(["none", "none", "yarn", "llama3"])
    rot = rng.choice([d, d, d // 2, 3 * d // 4, d // 2 + 2 * rng.randint(1, d // 4 - 1)])
    return dict(rot=rot, layout=rng.choice(["half", "half", "interleaved"]), base=rng.choice([10000.0, 500000.0]),
                scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 40.0]))


def draw(rng):
    kind = rng.choice(["rotary", "write", "write", "read", "select", "reorder"])
    base = dict(kind=kind, len_seed=rng.randrange(1 << 20))
    if kind == "select":
        batch, beams = _log(rng, 1, 64), _log(rng, 1, 12)
        vocab = _log(rng, 500, min(200000, 60000000 // (batch * beams)))
        return dict(base, batch=batch, beams=beams, n=rng.choice([1, beams, beams, 2 * beams, 24]), vocab=vocab,
                    dt=rng.choice(["bf16", "bf16", "f32"]), done=rng.random() < 0.4)
    hkv, d = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128])
    page, pool = rng.choice([16, 16, 32, 64]), rng.choice(["split", "paired"])
    g = rng.choice([1, 2, 4, 4, 8, 6])
    if kind == "reorder":
        groups, ways = _log(rng, 1, 16), _log(rng, 2, 8)
        hi = _log(rng, 20, 9000)
        return dict(base, hkv=hkv, d=d, page=page, kv=rng.choice(["bf16", "fp8"]), layers=_log(rng, 1, 8), groups=groups,
                    ways=ways, lo=max(1, hi // 3), hi=hi, tail=_log(rng, 1, 200), spare=rng.randint(1, 100))
    kv = rng.choice(["bf16", "fp8", "fp8", "f32"])
    if kind == "rotary":
        return dict(base, **_draw_rotary(rng, d), hkv=hkv, g=g, d=d, n=_log(rng, 1, 24000),
                    far=_log(rng, 100, 2000000), dt=rng.choice(["bf16", "bf16", "f32"]), fused=rng.random() < 0.5)
    n, hi = _log(rng, 1, 16), _log(rng, 1, 2500)
    past = _log(rng, 1, 3000)
    base = dict(base, hkv=hkv, g=g, d=d, n=n, lo=rng.choice([1, hi]), hi=hi, past_lo=rng.choice([0, past]), past_hi=past,
                kv=kv, page=page, pool=pool)
    if kind == "read":
        return base
    single = rng.random() < 0.3
    if single:
        base = dict(base, n=_log(rng, 1, 64), lo=1, hi=1)
    return dict(base, **_draw_rotary(rng, d), fused=rng.random() < 0.5, single=single)


# ------------------------------------------------------------------ inputs

def _lens(c, lo, hi, count, salt):
    r = random.Random(c["len_seed"] * 8 + salt)
    return [r.randint(c[lo], c[hi]) for _ in range(count)]


def _new_past(c):
    return _lens(c, "lo", "hi", c["n"], 0), _lens(c, "past_lo", "past_hi", c["n"], 1)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(gen, shape, dtype):
    return torch.empty(shape, device=DEV, dtype=dtype).normal_(generator=gen)


def _channel_scale(gen, hkv, d):
    return (0.5 * _normal(gen, (hkv, 1, d), torch.float32)).exp()


def _i32(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _i32(out)


def _row_dtype(c):
    return torch.float32 if c.get("kv", c.get("dt")) == "f32" else torch.bfloat16


def _original(c):
    """The context that a stretched model was first trained on."""
    return 8192


def _frequencies(c):
    """Radians per position of each pair (64 bits, on the host) and the factor of the rotation."""
    r, base, s = c["rot"], c["base"], c["factor"]
    w = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if c["scaling"] == "yarn":  # short waves as they are, long ones stretched, a ramp over the pairs between
        def pair(turns):
            return r * math.log(_original(c) / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), r - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(r // 2)]
        return [a * (1 - t) + a / s * t for a, t in zip(w, ramp)], 0.1 * math.log(s) + 1.0
    if c["scaling"] == "llama3":  # the same by wave length: between a quarter of the context and all of it
        turns = [_original(c) * a / (2 * math.pi) for a in w]
        keep = [min(max((t - 1.0) / 3.0, 0.0), 1.0) for t in turns]
        return [a * k + a / s * (1 - k) for a, k in zip(w, keep)], 1.0
    return w, 1.0


def _rotary_state(c, s):
    """The frequencies, and where the package is asked, its plan of them, both kept by the program."""
    w, s["amplitude"] = _frequencies(c)
    s["w"] = torch.tensor(w, device=DEV, dtype=torch.float64)
    if own:
        import interattn_amd as ia

        scaling = None if c["scaling"] == "none" else {"rope_type": c["scaling"], "factor": c["factor"],
                                                       "original_max_position_embeddings": _original(c)}
        if c["scaling"] == "llama3":
            scaling.update(low_freq_factor=1.0, high_freq_factor=4.0)
        s["plan"] = ia.rotary_plan(c["rot"], base=c["base"], scaling=scaling, layout=c["layout"], device=DEV)


def _pool(c, gen, n_pages, key_scale):
    """K and V pools [n_pages, Hkv, page, D] and, for fp8, their scales [n_pages, Hkv]."""
    hkv, page, d, kv = c["hkv"], c["page"], c["d"], c["kv"]
    if c.get("pool") == "paired":
        buf = torch.empty((n_pages, hkv, 2, page, d), device=DEV, dtype=DTYPES[kv])
        k, v = buf[:, :, 0], buf[:, :, 1]
    else:
        k = torch.empty((n_pages, hkv, page, d), device=DEV, dtype=DTYPES[kv])
        v = torch.empty_like(k)
    ks, vs = [], []
    step = max(1, (1 << 27) // (hkv * page * d))
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        for pool, sc, mul in ((k, ks, key_scale), (v, vs, None)):
            x = _normal(gen, (n, hkv, page, d), _row_dtype(c))
            if mul is not None:
                x.mul_(mul.to(x.dtype))
            if kv == "fp8":
                s = _scale_for(x.abs().amax(dim=(2, 3)).float())
                sc.append(s)
                x = x.float() / s[:, :, None, None]
            pool[i:i + n].copy_(x)
    return k, v, (torch.cat(ks), torch.cat(vs)) if kv == "fp8" else None


def _table(gen, need, n_pages, cols=None):
    perm = torch.randperm(n_pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((len(need), cols or max(max(need), 1)), -1, device=DEV, dtype=torch.int32)
    off = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[off:off + n]
        off += n
    return table


def _packed(c, gen, total, key_scale):
    """q, k and v rows of ``total`` tokens: views of one fused projection, or apart."""
    hq, hkv, d = c["hkv"] * c["g"], c["hkv"], c["d"]
    buf = _normal(gen, (total, hq + 2 * hkv, d), _row_dtype(c))
    buf[:, hq:hq + hkv].mul_(key_scale.to(buf.dtype).transpose(0, 1))
    parts = buf.split([hq, hkv, hkv], dim=1)
    return parts if c["fused"] else tuple(x.contiguous() for x in parts)


def _prepare_rotary(c, gen, s):
    s["q"], s["k"], _ = _packed(c, gen, c["n"], _channel_scale(gen, c["hkv"], c["d"]))
    start = torch.randint(c["far"], (1,), device=DEV, generator=gen)
    s["pos"] = ((torch.arange(c["n"], device=DEV) + start) % c["far"]).to(torch.int32)
    _rotary_state(c, s)


def _prepare_write(c, gen, s):
    new, past = _new_past(c)
    page = c["page"]
    scale = _channel_scale(gen, c["hkv"], c["d"])
    need = [-(-(a + b) // page) for a, b in zip(new, past)]
    n_pages = sum(need) + 3
    s["pool_k"], s["pool_v"], s["scales"] = _pool(c, gen, n_pages, scale)
    s["table"] = _table(gen, need, n_pages)
    s["cu"], s["seq"] = _cu(new), _i32(past)
    s["q"], s["k"], s["v"] = _packed(c, gen, sum(new), scale)
    # the touched pages' rows, from the first token of the page that the new ones begin in
    s["from"] = _i32([p // page * page for p in past])
    back = [n + p % page for n, p in zip(new, past)]
    s["cu_back"], s["n_back"] = _cu(back), sum(back)
    _rotary_state(c, s)


def _prepare_read(c, gen, s):
    count, first = _new_past(c)
    need = [-(-(a + b) // c["page"]) for a, b in zip(count, first)]
    n_pages = sum(need) + 3
    s["pool_k"], s["pool_v"], s["scales"] = _pool(c, gen, n_pages, _channel_scale(gen, c["hkv"], c["d"]))
    s["table"] = _table(gen, need, n_pages)
    s["from"], s["cu_back"], s["n_back"] = _i32(first), _cu(count), sum(count)


def _prepare_select(c, gen, s):
    rows, vocab = c["batch"] * c["beams"], c["vocab"]
    # (the projection's output: rows begin at multiples of 16 bytes)
    s["logits"] = _normal(gen, (rows, -(-vocab // 8) * 8), DTYPES[c["dt"]]).mul_(2.5)[:, :vocab]
    s["scores"] = _normal(gen, (c["batch"], c["beams"]), torch.float32).mul_(3).sub_(12)
    s["done"] = torch.rand((c["batch"], c["beams"]), device=DEV, generator=gen) < 0.25 if c["done"] else None


def _parents(c):
    """Each group's rows continue some of its rows: the better ones more often."""
    r = random.Random(c["len_seed"] * 8 + 5)
    return [g * c["ways"] + min(r.randrange(c["ways"]), r.randrange(c["ways"]))
            for g in range(c["groups"]) for _ in range(c["ways"])]


def _prepare_reorder(c, gen, s):
    """``groups`` prompts, each with ``ways`` rows that share its pages and have tails of their own."""
    page, ways = c["page"], c["ways"]
    prompts = _lens(c, "lo", "hi", c["groups"], 0)
    seq = [prompts[i // ways] + c["tail"] for i in range(c["groups"] * ways)]
    whole = [prompts[i // ways] // page for i in range(len(seq))]
    tails = [-(-n // page) - w for n, w in zip(seq, whole)]
    n_pages = sum(whole[::ways]) + sum(tails) + c["spare"] + len(seq)
    perm = torch.randperm(n_pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((len(seq), max(-(-n // page) for n in seq) + 2), -1, device=DEV, dtype=torch.int32)
    off = 0
    for i, (w, t) in enumerate(zip(whole, tails)):
        if i % ways == 0:
            table[i:i + ways, :w] = perm[off:off + w]
            off += w
        table[i, w:w + t] = perm[off:off + t]
        off += t
    s["pools"] = []
    scale = _channel_scale(gen, c["hkv"], c["d"])
    for _ in range(c["layers"]):
        k, v, scales = _pool(c, gen, n_pages, scale)
        s["pools"] += [k, v, *(scales or ())]
    s["table"], s["seq"] = table, _i32(seq)
    s["refs"] = torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)
    s["parents"] = _i32(_parents(c))


def prepare(case, seed):
    s = {"case": case, "ws": {}}
    with torch.no_grad():
        globals()["_prepare_" + case["kind"]](case, _gen(seed), s)
    return s


# ------------------------------------------------------------------ plain forms

def _scale_for(largest):
    """The least power of two (2^-126 at least) that brings ``largest`` down to 448 or less."""
    m, e = torch.frexp(largest)  # largest = m 2^e, 448 = 0.875 2^9
    s = torch.ldexp(torch.ones_like(largest), (e - 9 + (m > 0.875)).clamp_min(-126))
    return torch.where(largest > 0, s, LOWEST_SCALE)


def _rotated(s, x, pos):
    """Rows ``x [T, H, D]`` at positions ``pos [T]``, in 32 bits."""
    c = s["case"]
    r = c["rot"]
    angle = pos.double()[:, None] * s["w"]
    cos, sin = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = x.float()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if c["layout"] == "half" else (x[..., :r:2], x[..., 1:r:2])
    pair = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat(pair, -1) if c["layout"] == "half" else torch.stack(pair, -1).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_rotary(s):
    return tuple(_rotated(s, s[x], s["pos"]).to(s[x].dtype) for x in ("q", "k"))


def _places(s, first, cu, n, page):
    """Sequence, position, page and place in it of each of ``n`` packed tokens."""
    i = torch.arange(n, device=DEV)
    b = torch.searchsorted(cu[1:], i, right=True)
    pos = first.long()[b] + i - cu.long()[b]
    return b, pos, s["table"][b, pos // page].long(), pos % page


def _rows_of(pool, scale, pages, at, dtype):
    x = pool[pages, :, at].float()
    return (x if scale is None else x * scale[pages][:, :, None]).to(dtype)


def _read(s, dtype):
    c = s["case"]
    _, _, pages, at = _places(s, s["from"], s["cu_back"], s["n_back"], c["page"])
    ks, vs = s["scales"] or (None, None)
    return _rows_of(s["pool_k"], ks, pages, at, dtype), _rows_of(s["pool_v"], vs, pages, at, dtype)


def _plain_read(s):
    return _read(s, _row_dtype(s["case"]))


def _quantised(s, pool, scale, x, pages, at):
    """Rows ``x [T, Hkv, D]`` into fp8 pages; pages with earlier tokens may get a larger scale."""
    page = s["case"]["page"]
    largest = torch.zeros_like(scale).index_reduce_(0, pages, x.abs().amax(-1), "amax")
    # the page a sequence's new tokens begin in, where it has earlier ones
    past = s["seq"].long()
    begun = s["table"][torch.arange(past.numel(), device=DEV), (past // page).clamp_max(s["table"].shape[1] - 1)].long()
    begun, held = begun[past % page > 0], (past % page)[past % page > 0]
    before = scale[begun]
    scale[pages] = _scale_for(largest)[pages]
    scale[begun] = torch.where(largest[begun] <= LARGEST_CODE * before, before, scale[begun])
    again = (pool[begun].float() * (before / scale[begun])[:, :, None, None]).to(pool.dtype)
    mine = torch.arange(page, device=DEV)[None, None, :, None] < held[:, None, None, None]
    raw = pool.view(torch.uint8)
    raw[begun] = torch.where(mine, again.view(torch.uint8), raw[begun])
    raw[pages, :, at] = (x / scale[pages][:, :, None]).to(pool.dtype).view(torch.uint8)


def _plain_write(s):
    c = s["case"]
    _, pos, pages, at = _places(s, s["seq"], s["cu"], s["k"].shape[0], c["page"])
    q, k = _rotated(s, s["q"], pos).to(s["q"].dtype), _rotated(s, s["k"], pos)
    lens = s["seq"] + (s["cu"][1:] - s["cu"][:-1])
    if c["kv"] != "fp8":
        s["pool_k"][pages, :, at] = k.to(s["pool_k"].dtype)
        s["pool_v"][pages, :, at] = s["v"]
        return q, lens, s["pool_k"], s["pool_v"]
    _quantised(s, s["pool_k"], s["scales"][0], k, pages, at)
    _quantised(s, s["pool_v"], s["scales"][1], s["v"].float(), pages, at)
    return q, lens, *_read(s, torch.bfloat16), *s["scales"]


def _plain_select(s):
    c = s["case"]
    batch, beams, vocab, n = c["batch"], c["beams"], c["vocab"], c["n"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = x - x.exp().sum(-1, keepdim=True).log()
    keys = x.view(batch, beams, vocab) + s["scores"].double()[:, :, None]
    if s["done"] is not None:
        ended = torch.full_like(keys[0, 0], -math.inf)
        keys = torch.where(s["done"][:, :, None], ended, keys)
        keys[:, :, 0] = torch.where(s["done"], s["scores"].double(), keys[:, :, 0])
    keys = keys.view(batch, -1)
    least = keys.topk(n, sorted=True).values[:, -1:]
    # equal keys go to the lowest index: all that reach the n-th, in order, best first, n of each
    b, at = (keys >= least).nonzero(as_tuple=True)
    found = keys[b, at]
    order = torch.argsort(found, descending=True, stable=True)
    order = order[torch.argsort(b[order], stable=True)]
    b, at, found = b[order], at[order], found[order]
    rank = torch.arange(b.numel(), device=DEV) - torch.searchsorted(b, b)
    at, found = at[rank < n].view(batch, n), found[rank < n].view(batch, n)
    parents = at // vocab + torch.arange(batch, device=DEV)[:, None] * beams
    return found.float(), (at % vocab).to(torch.int32), parents.to(torch.int32)


def _plain_reorder(s):
    table, refs, page = s["table"], s["refs"], s["case"]["page"]
    rows, cols = table.shape
    parents, i = s["parents"].long(), torch.arange(rows, device=DEV)
    # the row that takes its parent's pages over: the parent itself, else the lowest one
    first = torch.full((rows,), rows, device=DEV).scatter_reduce(0, parents, torch.where(parents == i, -1, i), "amin")
    heir = (parents == i) | (first[parents] == i)
    lens = s["seq"].long()[parents]
    taken = table[parents]
    at = torch.arange(cols, device=DEV)[None]
    new = torch.where(heir[:, None] | (at < (lens // page)[:, None]), taken, -1)
    refs.copy_(torch.bincount(new[new >= 0].long(), minlength=refs.numel()))
    part = (~heir & (lens % page > 0)).nonzero().flatten()
    fresh = (refs == 0).nonzero().flatten()[:part.numel()]
    old = taken[part, (lens // page)[part]].long()
    new[part, (lens // page)[part]] = fresh.to(torch.int32)
    refs[fresh] = 1
    for pool in s["pools"]:
        pool[fresh] = pool[old]
    table.copy_(new)
    s["seq"].copy_(lens)
    return table, s["seq"], refs, torch.ones_like(s["parents"]), s["pools"]


# ------------------------------------------------------------------ one pass

def _own_run(s):
    import interattn_amd as ia

    c, kind = s["case"], s["case"]["kind"]
    if kind == "rotary":
        return ia.apply_rotary(s["q"], s["k"], s["pos"], s["plan"])
    if kind == "write":
        lens = torch.empty_like(s["seq"])
        q, lens = ia.rotary_append_kv(s["q"], s["k"], s["v"], s["plan"], s["pool_k"], s["pool_v"], s["table"], s["seq"],
                                      None if c["single"] else s["cu"], scales=s["scales"], new_seq_lens=lens)
        if c["kv"] != "fp8":
            return q, lens, s["pool_k"], s["pool_v"]
        k, v = ia.read_kv(s["pool_k"], s["pool_v"], s["table"], s["from"], s["cu_back"], s["n_back"],
                          scales=s["scales"], out_dtype=torch.bfloat16)
        return q, lens, k, v, *s["scales"]
    if kind == "read":
        return ia.read_kv(s["pool_k"], s["pool_v"], s["table"], s["from"], s["cu_back"], s["n_back"],
                          scales=s["scales"], out_dtype=_row_dtype(c))
    if kind == "select":
        return ia.beam_select(s["logits"], s["scores"], c["n"], done=s["done"], workspace=s["ws"])
    ok = ia.reorder_sequences(s["pools"], s["table"], s["seq"], s["refs"], s["parents"], page_size=c["page"],
                              workspace=s["ws"])
    return s["table"], s["seq"], s["refs"], ok, s["pools"]


def run(state):
    with torch.no_grad():
        if own:
            return _own_run(state)
        return globals()["_plain_" + state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, kind = case, case["kind"]
    if kind == "select":
        return {"bytes": c["batch"] * c["beams"] * c["vocab"] * BYTES[c["dt"]] + 12 * c["batch"] * c["n"], "flops": 0}
    hkv, d = c["hkv"], c["d"]
    if kind == "reorder":
        parents, ways = _parents(c), c["ways"]
        seq = [n + c["tail"] for n in _lens(c, "lo", "hi", c["groups"], 0) for _ in range(ways)]
        copies = sum(len(set(range(len(seq))) & {i for i, p in enumerate(parents) if p == r}) - 1
                     for r in set(parents) if seq[r] % c["page"])
        page_bytes = c["layers"] * (2 * hkv * c["page"] * d * BYTES[c["kv"]] + (8 * hkv if c["kv"] == "fp8" else 0))
        changed = sum(-(-seq[i] // c["page"]) for i, p in enumerate(parents) if p != i)
        return {"bytes": 2 * copies * page_bytes + 8 * changed + 8 * len(seq), "flops": 0}
    rb = 4 if _row_dtype(c) == torch.float32 else 2
    if kind == "rotary":
        return {"bytes": 2 * c["n"] * hkv * (c["g"] + 1) * d * rb + 4 * c["n"],
                "flops": 3 * c["n"] * hkv * (c["g"] + 1) * c["rot"]}
    new, past = _new_past(c)
    held = hkv * (2 * d * BYTES[c["kv"]] + (8 / c["page"] if c["kv"] == "fp8" else 0))  # K and V of one cached token
    rows = hkv * 2 * d * rb  # of one packed token
    if kind == "read":
        return {"bytes": sum(new) * (held + rows), "flops": 0}
    q = 2 * sum(new) * hkv * c["g"] * d * rb
    back = 0
    if c["kv"] == "fp8":
        back = sum(n + p % c["page"] for n, p in zip(new, past)) * (held + hkv * 2 * d * 2)
    return {"bytes": q + sum(new) * (rows + held) + back, "flops": 3 * sum(new) * hkv * (c["g"] + 1) * c["rot"]}


# ------------------------------------------------------------------ the definition, in 64 bits

def _turned(c, s, x, pos):
    """Pairs as complex numbers, turned by their angles."""
    r, x = c["rot"], x.double()
    if c["layout"] == "half":
        z = torch.complex(x[:, :, :r // 2], x[:, :, r // 2:r])
    else:
        z = torch.view_as_complex(x[:, :, :r].reshape(x.shape[0], x.shape[1], r // 2, 2).contiguous())
    angle = pos.double()[:, None, None] * s["w"]
    z = z * torch.polar(torch.full_like(angle, s["amplitude"]), angle)
    out = x.clone()
    if c["layout"] == "half":
        out[:, :, :r // 2], out[:, :, r // 2:r] = z.real, z.imag
    else:
        out[:, :, 0:r:2], out[:, :, 1:r:2] = z.real, z.imag
    return out


def _to_code(y):
    """The nearest e4m3 value, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _exact_write(c, s):
    """Page by page of each sequence: its scale, what it held and what is new."""
    new, past = _new_past(c)
    page, hkv, d = c["page"], c["hkv"], c["d"]
    pos = torch.cat([torch.arange(p, p + n, device=DEV) for n, p in zip(new, past)])
    q = _turned(c, s, s["q"], pos)
    rows = _turned(c, s, s["k"], pos), s["v"].double()
    lens = None
    if c["kv"] != "fp8":
        pools = [s["pool_k"].double(), s["pool_v"].double()]
        start = 0
        for b, (n, p) in enumerate(zip(new, past)):
            at = torch.arange(p, p + n, device=DEV)
            for pool, x in zip(pools, rows):
                pool[s["table"][b].long()[at // page], :, at % page] = x[start:start + n]
            start += n
        return q, lens, *pools
    back, scales = ([], []), [x.double() for x in s["scales"]]
    for pool, scale, x, out in zip((s["pool_k"], s["pool_v"]), scales, rows, back):
        start = 0
        for b, (n, p) in enumerate(zip(new, past)):
            first = p // page
            count = -(-(p + n) // page) - first
            pages = s["table"][b, first:first + count].long()
            held = pool[pages].float().double()  # codes [count, Hkv, page, D]
            grid = torch.zeros((count * page, hkv, d), device=DEV, dtype=torch.float64)
            grid[p % page:p % page + n] = x[start:start + n]
            grid = grid.view(count, page, hkv, d).transpose(1, 2)
            most = grid.abs().amax(dim=(2, 3))
            pick = torch.exp2(torch.ceil(torch.log2(most.clamp_min(2.0 ** -200) / 448)).clamp_min(-126))
            if p % page:
                had = scale[pages[0]]
                pick[0] = torch.where(most[0] <= 448 * had, had, pick[0])
                old = _to_code(held[0] * (had / pick[0])[:, None, None]) * pick[0][:, None, None]
            val = _to_code(grid / pick[:, :, None, None]) * pick[:, :, None, None]
            if p % page:
                val[0, :, :p % page] = old[:, :p % page]
            scale[pages] = pick
            out.append(val.transpose(1, 2).reshape(count * page, hkv, d)[:p % page + n])
            start += n
    return q, lens, torch.cat(back[0]), torch.cat(back[1]), *scales


def exact(case, seed):
    """64-bit outputs of the kinds that compute numbers; pages that only move, lengths and tokens are none."""
    c, kind = case, case["kind"]
    if kind == "reorder":
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if kind == "rotary":
            return _turned(c, s, s["q"], s["pos"]), _turned(c, s, s["k"], s["pos"])
        if kind == "write":
            return _exact_write(c, s)
        if kind == "select":
            logp = torch.log_softmax(s["logits"].double(), -1).view(c["batch"], c["beams"], c["vocab"])
            if s["done"] is not None:
                logp[s["done"]] = -math.inf
                logp[:, :, 0] = logp[:, :, 0].masked_fill(s["done"], 0.0)
            total = (logp + s["scores"].double()[:, :, None]).flatten(1)
            return torch.sort(total, dim=1, descending=True).values[:, :c["n"]], None, None
        count, first = _new_past(c)
        outs = ([], [])
        for b, (n, f) in enumerate(zip(count, first)):
            at = torch.arange(f, f + n, device=DEV)
            pages = s["table"][b].long()[at // c["page"]]
            for i, x in enumerate(("pool_k", "pool_v")):
                v = s[x].view(torch.uint8) if c["kv"] == "fp8" else s[x]
                v = v[pages, :, at % c["page"]]
                if c["kv"] == "fp8":
                    v = v.view(DTYPES["fp8"]).float().double() * s["scales"][i].double()[pages][:, :, None]
                outs[i].append(v.double())
        return torch.cat(outs[0]), torch.cat(outs[1])
