"""Operators of prompt processing and of page sharing, as a serving program calls them.

With ``own`` false, ``run`` computes each operator in its plain form: elementary torch
operations in 32 bits, rounded once at the end.  With ``own`` true it makes the calls of
the package's entry points.  Kinds:

  prompt   ``ia.prompt_attention``: causal attention over packed prompts of different
           lengths, K and V as the projection left them
  paged    ``ia.paged_prompt_attention``: the new tokens of each sequence over the whole
           sequence in the paged pool (a chunk of a long prompt, a prompt behind a cached
           prefix, single tokens)
  prefix   ``ia.shared_prefix_decode``: one decode step of a batch whose sequences share
           long prefixes, each prefix's K/V read once for all of its sequences
  append   ``ia.append_prompt_kv``: the K/V rows of packed prompts into the pages
  fork     ``ia.free_sequences``, ``ia.fork_sequences``, ``ia.reserve_pages``: old
           continuations dropped, new ones forked from their prompts, pages for the
           tokens they are about to write
  copy     ``ia.copy_pages``: pages of every layer's pools copied to other pages
  compact  ``ia.compact_pages``: live pages moved to the front of the pools

Values are those the path meets: unit-variance queries and values, keys with a scale per
(kv head, channel) as rotary keys have; pages in random order; fp8 pages scaled by their
largest magnitude.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f32": 4, "fp8": 1}
DEV = "cuda"
SCORES_AT_ONCE = 1 << 27  # elements of the largest score matrix the plain forms hold


# ------------------------------------------------------------------ the cases

def listed():
    llama = {"hkv": 8, "g": 4, "d": 128}
    return [
        # one short prompt: latency
        dict(llama, name="prompt 1x333", kind="prompt", n=1, lo=333, hi=333, kv="bf16", fused=True, len_seed=0),
        # a packed batch of chat prompts, groups of 8 query heads, small heads
        dict(name="prompt g8 24x1-2000", kind="prompt", n=24, hkv=4, g=8, d=64, lo=1, hi=2000, kv="bf16", fused=True,
             len_seed=11),
        # long prompts: the matrix cores' share
        dict(llama, name="prompt 2x8192", kind="prompt", n=2, lo=8192, hi=8192, kv="bf16", fused=False, len_seed=0),
        # chunks of four long prompts, each over what its sequence has cached
        dict(llama, name="paged 4x256 at 16k-32k", kind="paged", n=4, lo=256, hi=256, past_lo=16000, past_hi=32500,
             kv="bf16", page=16, layout="split", len_seed=2),
        # a float32 model's prompts behind short cached prefixes, single tokens among them
        dict(name="paged f32 8x1-500 at 0-1500", kind="paged", n=8, hkv=4, g=2, d=64, lo=1, hi=500, past_lo=0,
             past_hi=1500, kv="f32", page=16, layout="split", len_seed=3),
        # 32 continuations of one long document
        dict(llama, name="prefix 32 on 32k", kind="prefix", members="32", shared_lo=32768, shared_hi=32768, lo=1,
             hi=1000, kv="bf16", page=16, layout="split", len_seed=4),
        # several system prompts of different lengths, quantised pages, sequences without one
        dict(llama, name="prefix fp8 5+1+9+4 on 1k-8k", kind="prefix", members="5+1+9+4", shared_lo=1000,
             shared_hi=8200, lo=0, hi=700, kv="fp8", page=16, layout="paired", len_seed=5),
        # the K/V of one short prompt into its pages: latency
        dict(llama, name="append 1x37", kind="append", n=1, lo=37, hi=37, past_lo=100, past_hi=100, kv="bf16", page=16,
             layout="split", fused=True, len_seed=0),
        # the K/V of a batch of prompts
        dict(llama, name="append 16x500-4000", kind="append", n=16, lo=500, hi=4000, past_lo=0, past_hi=300, kv="bf16",
             page=16, layout="split", fused=True, len_seed=6),
        # eight continuations of each of two prompts, over eight layers
        dict(name="fork 2x8 at 2k-6k", kind="fork", hkv=8, d=128, page=16, kv="bf16", layers=8, prompts=2, ways=8,
             lo=2000, hi=6000, reserve=40, spare=400, len_seed=7),
        # pages of a sequence moved aside (fp8 pools with their scales)
        dict(name="copy 700", kind="copy", hkv=8, d=128, page=16, kv="fp8", layers=4, count=700, pages=2000,
             len_seed=8),
        # a long-running server's pool, half of its pages free
        dict(name="compact 16k", kind="compact", hkv=8, d=128, page=16, kv="bf16", layers=2, pages=16384, live=0.5,
             seq_pages=200, len_seed=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "paged", "paged", "paged", "prefix", "prefix", "prefix",
                       "append", "fork", "copy", "compact"])
    g = rng.choice([1, 2, 4, 4, 8, 8, 6])
    hkv = rng.choice([1, 2, 4, 8, 8])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64])
    layout = rng.choice(["split", "paired"])
    len_seed = rng.randrange(1 << 20)
    base = dict(kind=kind, hkv=hkv, d=d, len_seed=len_seed)
    if kind == "prompt":
        kv = rng.choice(["bf16", "bf16", "bf16", "f32"])
        hi = _log(rng, 1, 8192 if kv == "bf16" else 2048)
        lo = hi if rng.random() < 0.4 else 1
        most = max(1, min(32, int(1.3e8 / 64 / (hi * hi)) if kv == "f32" else int(1.3e8 / (hi * hi))))
        return dict(base, n=_log(rng, 1, most), g=g, lo=lo, hi=hi, kv=kv, fused=rng.random() < 0.5)
    if kind == "paged":
        kv = rng.choice(["bf16", "bf16", "fp8", "f32"])
        hi = _log(rng, 1, 1500)
        past = _log(rng, 16, 40000 if kv != "f32" else 4000)
        most = max(1, min(16, int((6e7 if kv != "f32" else 2e6) / (hi * (past + hi)))))
        return dict(base, n=_log(rng, 1, most), g=g, lo=rng.choice([1, hi]), hi=hi,
                    past_lo=rng.choice([0, past, past // 2]), past_hi=past, kv=kv, page=page, layout=layout)
    if kind == "prefix":
        groups = rng.choice([1, 1, 2, 3, 5])
        most = _log(rng, 1, 48 // groups)
        shared = _log(rng, 100, 60000 // groups)
        return dict(base, g=g, members="+".join(str(rng.randint(1, most)) for _ in range(groups)),
                    shared_lo=rng.choice([shared, max(shared // 4, 1)]), shared_hi=shared, lo=0,
                    hi=_log(rng, 1, 1500), kv=rng.choice(["bf16", "bf16", "fp8", "f32"]), page=page, layout=layout)
    if kind == "append":
        hi = _log(rng, 1, 4000)
        return dict(base, g=g, n=_log(rng, 1, 16), lo=rng.choice([1, hi]), hi=hi, past_lo=0,
                    past_hi=_log(rng, 1, 2000), kv=rng.choice(["bf16", "f32"]), page=page, layout=layout,
                    fused=rng.random() < 0.5)
    kv = rng.choice(["bf16", "fp8", "f32"])
    layers = _log(rng, 1, 16)
    if kind == "fork":
        hi = _log(rng, 20, 12000)
        return dict(base, page=page, kv=kv, layers=layers, prompts=rng.randint(1, 4), ways=_log(rng, 1, 16),
                    lo=max(1, hi // 3), hi=hi, reserve=_log(rng, 1, 300), spare=_log(rng, 10, 600))
    bytes_page = 2 * layers * hkv * page * d * BYTES[kv]
    pages = max(8, min(_log(rng, 50, 40000), int(2 ** 31 / bytes_page)))
    if kind == "copy":
        return dict(base, page=page, kv=kv, layers=layers, pages=pages, count=_log(rng, 1, pages // 2))
    return dict(base, page=page, kv=kv, layers=layers, pages=pages, live=rng.choice([0.2, 0.5, 0.9]),
                seq_pages=_log(rng, 2, 400))


# ------------------------------------------------------------------ inputs

def _lens(c, lo, hi, count, salt):
    r = random.Random(c["len_seed"] * 8 + salt)
    return [r.randint(c[lo], c[hi]) for _ in range(count)]


def _news_pasts(c):
    return _lens(c, "lo", "hi", c["n"], 0), _lens(c, "past_lo", "past_hi", c["n"], 1)


def _members(c):
    """Sequences of each group of a prefix case."""
    return [int(x) for x in c["members"].split("+")]


def _group_lens(c):
    """Lengths of a prefix case: of each group's prefix, of each sequence's own tokens."""
    members = _members(c)
    return _lens(c, "shared_lo", "shared_hi", len(members), 0), _lens(c, "lo", "hi", sum(members), 1)


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


def _work_dtype(c):
    return torch.float32 if c["kv"] == "f32" else torch.bfloat16


def _pool(gen, n_pages, hkv, page, d, kv, layout, key_scale):
    """K and V pools [n_pages, Hkv, page, D] and, for fp8, their scales [n_pages, Hkv]."""
    if layout == "paired":
        buf = torch.empty((n_pages, hkv, 2, page, d), device=DEV, dtype=DTYPES[kv])
        k, v = buf[:, :, 0], buf[:, :, 1]
    else:
        k = torch.empty((n_pages, hkv, page, d), device=DEV, dtype=DTYPES[kv])
        v = torch.empty_like(k)
    draw_t = torch.float32 if kv == "f32" else torch.bfloat16
    ks, vs = [], []
    step = max(1, (1 << 27) // (hkv * page * d))
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        for pool, sc, mul in ((k, ks, key_scale), (v, vs, None)):
            x = _normal(gen, (n, hkv, page, d), draw_t)
            if mul is not None:
                x.mul_(mul.to(draw_t))
            if kv == "fp8":
                s = x.abs().amax(dim=(2, 3)).float().clamp_min(1e-12) / 448.0
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


def _packed(c, gen, total, key_scale, with_q):
    """q, k and v rows of ``total`` tokens: views of one fused projection, or apart."""
    hq, hkv, d, dt = c["hkv"] * c["g"] if with_q else 0, c["hkv"], c["d"], _work_dtype(c)
    buf = _normal(gen, (total, hq + 2 * hkv, d), dt)
    buf[:, hq:hq + hkv].mul_(key_scale.to(dt).transpose(0, 1))
    parts = buf.split([hq, hkv, hkv], dim=1)
    return parts if c["fused"] else tuple(x.contiguous() for x in parts)


def _prepare_prompt(c, gen, s):
    s["lens"] = _lens(c, "lo", "hi", c["n"], 0)
    s["cu"] = _cu(s["lens"])
    s["q"], s["k"], s["v"] = _packed(c, gen, sum(s["lens"]), _channel_scale(gen, c["hkv"], c["d"]), True)


def _prepare_paged(c, gen, s):
    new, past = _news_pasts(c)
    s["new"], s["lens"] = new, [a + b for a, b in zip(new, past)]
    need = [-(-n // c["page"]) for n in s["lens"]]
    n_pages = sum(need) + 3
    s["pool_k"], s["pool_v"], s["scales"] = _pool(gen, n_pages, c["hkv"], c["page"], c["d"], c["kv"], c["layout"],
                                                  _channel_scale(gen, c["hkv"], c["d"]))
    s["table"] = _table(gen, need, n_pages)
    s["cu"], s["seq"] = _cu(new), _i32(s["lens"])
    s["q"] = _normal(gen, (sum(new), c["hkv"] * c["g"], c["d"]), _work_dtype(c))


def _prepare_prefix(c, gen, s):
    shared, tails = _group_lens(c)
    page = c["page"]
    own_pages, seq, rows = [], [], []
    b = 0
    for members, n in zip(_members(c), shared):
        for _ in range(members):
            # whole shared pages stay shared; the page the prefix ends in is each sequence's own
            seq.append(n + tails[b])
            own_pages.append(-(-seq[-1] // page) - n // page)
            rows.append(n // page)
            b += 1
    n_pages = sum(own_pages) + sum(n // page for n in shared) + 3
    s["pool_k"], s["pool_v"], s["scales"] = _pool(gen, n_pages, c["hkv"], page, c["d"], c["kv"], c["layout"],
                                                  _channel_scale(gen, c["hkv"], c["d"]))
    perm = torch.randperm(n_pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((len(seq), max(-(-n // page) for n in seq)), -1, device=DEV, dtype=torch.int32)
    off = b = 0
    for members, n in zip(_members(c), shared):
        whole = perm[off:off + n // page]
        off += n // page
        first = b
        for _ in range(members):
            table[b, :rows[b]] = whole
            table[b, rows[b]:rows[b] + own_pages[b]] = perm[off:off + own_pages[b]]
            off += own_pages[b]
            if b > first and n % page:  # the shared part of the page the prefix ends in is the same in each
                src, dst = table[first, rows[b]].long(), table[b, rows[b]].long()
                for pool in (s["pool_k"], s["pool_v"]):
                    pool.view(torch.uint8)[dst, :, :n % page] = pool.view(torch.uint8)[src, :, :n % page].clone()
                for sc in s["scales"] or ():
                    sc[dst] = sc[src]
            b += 1
    s["table"], s["seq"], s["lens"] = table, _i32(seq), seq
    s["starts"], s["shared"] = _cu(_members(c)), _i32(shared)
    s["q"] = _normal(gen, (len(seq), c["hkv"] * c["g"], c["d"]), _work_dtype(c))


def _prepare_append(c, gen, s):
    new, past = _news_pasts(c)
    s["new"], s["past"] = new, past
    need = [-(-(a + b) // c["page"]) for a, b in zip(new, past)]
    n_pages = sum(need) + 3
    scale = _channel_scale(gen, c["hkv"], c["d"])
    s["pool_k"], s["pool_v"], _ = _pool(gen, n_pages, c["hkv"], c["page"], c["d"], c["kv"], c["layout"], scale)
    s["table"] = _table(gen, need, n_pages)
    s["cu"], s["seq"] = _cu(new), _i32(past)
    _, s["k"], s["v"] = _packed(c, gen, sum(new), scale, False)


def _layer_pools(c, gen, n_pages):
    """Every layer's K and V pools (and scales), as ``copy_pages`` takes them."""
    out = []
    scale = _channel_scale(gen, c["hkv"], c["d"])
    for _ in range(c["layers"]):
        k, v, scales = _pool(gen, n_pages, c["hkv"], c["page"], c["d"], c["kv"], "split", scale)
        out += [k, v, *(scales or ())]
    return out


def _refs(table, n_pages):
    used = table[table >= 0].long()
    return torch.bincount(used, minlength=n_pages).to(torch.int32)


def _prepare_fork(c, gen, s):
    """``prompts`` sequences, each with ``ways`` rows that hold older continuations of it."""
    lens = _lens(c, "lo", "hi", c["prompts"], 0)
    page, ways = c["page"], c["ways"]
    tails = _lens(c, "reserve", "reserve", c["prompts"] * ways, 1)
    need = [-(-n // page) for n in lens]
    cols = max(need) + -(-c["reserve"] // page) + 2
    own_pages = [-(-(lens[i // ways] + tails[i]) // page) - lens[i // ways] // page for i in range(len(tails))]
    n_pages = sum(need) + sum(own_pages) + c["spare"] + 2 * len(tails)
    perm = torch.randperm(n_pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((c["prompts"] * (1 + ways), cols), -1, device=DEV, dtype=torch.int32)
    off, seq = 0, list(lens)
    for p, n in enumerate(need):
        table[p, :n] = perm[off:off + n]
        off += n
    for i, n in enumerate(own_pages):
        row, whole = c["prompts"] + i, lens[i // ways] // page
        table[row, :whole] = table[i // ways, :whole]
        table[row, whole:whole + n] = perm[off:off + n]
        off += n
        seq.append(lens[i // ways] + tails[i])
    s["pools"] = _layer_pools(c, gen, n_pages)
    s["table"], s["seq"], s["refs"] = table, _i32(seq), _refs(table, n_pages)
    s["src"] = _i32([i // ways for i in range(len(tails))])
    s["dst"] = _i32([c["prompts"] + i for i in range(len(tails))])
    s["grow"] = _i32([0] * c["prompts"] + [c["reserve"]] * len(tails))


def _prepare_copy(c, gen, s):
    s["pools"] = _layer_pools(c, gen, c["pages"])
    perm = torch.randperm(c["pages"], device=DEV, generator=gen).to(torch.int32)
    s["src"], s["dst"] = perm[:c["count"]].contiguous(), perm[c["count"]:2 * c["count"]].contiguous()


def _prepare_compact(c, gen, s):
    """Sequences of about ``seq_pages`` pages, pairs of them sharing their first half."""
    s["pools"] = _layer_pools(c, gen, c["pages"])
    r = random.Random(c["len_seed"])
    left = int(c["pages"] * c["live"])
    need, shared = [], []
    while left > 0:
        half = len(need) % 2 == 1 and need[-1] // 2
        n = r.randint(1, 2 * c["seq_pages"])
        n = max(1, min(n, left))
        need.append(n + (half or 0))
        shared.append(half or 0)
        left -= n
    table = torch.full((len(need), max(need)), -1, device=DEV, dtype=torch.int32)
    perm = torch.randperm(c["pages"], device=DEV, generator=gen).to(torch.int32)
    off = 0
    for b, (n, h) in enumerate(zip(need, shared)):
        if h:
            table[b, :h] = table[b - 1, :h]
        table[b, h:n] = perm[off:off + n - h]
        off += n - h
    s["table"], s["refs"] = table, _refs(table, c["pages"])


def prepare(case, seed):
    s = {"case": case, "ws": {}}
    with torch.no_grad():
        globals()["_prepare_" + case["kind"]](case, _gen(seed), s)
    return s


# ------------------------------------------------------------------ plain forms

def _attend(q, k, v, first, scale):
    """Rows of ``q [n, Hq, D]`` at positions ``first ...`` over ``k, v [Hkv, L, D]`` (32 bits), each over
    the keys up to its own position."""
    n, hq, d = q.shape
    hkv, total = k.shape[0], k.shape[1]
    out = torch.zeros((n, hq, d), device=q.device, dtype=torch.float32)
    if total == 0 or n == 0:
        return out
    g = hq // hkv
    step = max(1, SCORES_AT_ONCE // (g * total))
    cols = torch.arange(total, device=q.device)
    for h in range(hkv):
        kt = k[h].t().contiguous()
        for i in range(0, n, step):
            rows = q[i:i + step, h * g:(h + 1) * g].float()
            m = rows.shape[0]
            s = torch.matmul(rows.reshape(m * g, d), kt).view(m, g, total) * scale
            hidden = cols[None, None, :] > first + torch.arange(i, i + m, device=q.device)[:, None, None]
            s = s.masked_fill(hidden, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            out[i:i + m, h * g:(h + 1) * g] = torch.matmul(p.view(m * g, total), v[h]).view(m, g, d)
    return out


def _rows(pool, scale, table_row, n):
    """[Hkv, n, D]: the first n tokens of one sequence, dequantised, in 32 bits."""
    page = pool.shape[2]
    pages = table_row[:-(-n // page)].long()
    x = pool[pages].float()
    if scale is not None:
        x = x * scale[pages][:, :, None, None]
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _plain_prompt(s):
    out = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
    at = 0
    for n in s["lens"]:
        k, v = (s[x][at:at + n].float().transpose(0, 1).contiguous() for x in ("k", "v"))
        out[at:at + n] = _attend(s["q"][at:at + n], k, v, 0, s["case"]["d"] ** -0.5).to(out.dtype)
        at += n
    return out


def _plain_sequences(s, new):
    """Attention of each sequence's last ``new`` tokens over all of its tokens in the pool."""
    out = torch.empty_like(s["q"])
    ks, vs = s["scales"] or (None, None)
    at = 0
    for b, (n, total) in enumerate(zip(new, s["lens"])):
        k = _rows(s["pool_k"], ks, s["table"][b], total)
        v = _rows(s["pool_v"], vs, s["table"][b], total)
        out[at:at + n] = _attend(s["q"][at:at + n], k, v, total - n, s["case"]["d"] ** -0.5).to(out.dtype)
        at += n
    return out


def _plain_append(s):
    page = s["pool_k"].shape[2]
    at = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        pos = torch.arange(past, past + n, device=DEV)
        pages = s["table"][b].long()[pos // page]
        s["pool_k"][pages, :, pos % page] = s["k"][at:at + n]
        s["pool_v"][pages, :, pos % page] = s["v"][at:at + n]
        at += n
    return s["pool_k"], s["pool_v"], s["seq"] + (s["cu"][1:] - s["cu"][:-1])


def _plain_fork(s):
    table, seq, refs, page = s["table"], s["seq"], s["refs"], s["case"]["page"]
    dst, src = s["dst"].long(), s["src"].long()
    held = table[dst]
    refs.index_add_(0, held[held >= 0].long(), torch.full_like(held[held >= 0], -1))
    table[dst] = -1
    seq[dst] = 0
    # whole pages shared, the page a prompt ends in copied to the lowest free pages
    lens = seq[src]
    whole = lens // page
    cols = torch.arange(table.shape[1], device=DEV)
    rows = torch.where(cols[None, :] < whole[:, None], table[src], -1)
    part = (lens % page > 0).nonzero().flatten()
    fresh = (refs == 0).nonzero().flatten()[:part.numel()]
    old = table[src[part], whole[part].long()].long()
    rows[part, whole[part].long()] = fresh.to(torch.int32)
    table[dst] = rows
    seq[dst] = lens
    refs.index_add_(0, rows[rows >= 0].long(), torch.ones_like(rows[rows >= 0]))
    for pool in s["pools"]:
        pool[fresh] = pool[old]
    # pages for the next tokens, the lowest free ones in the rows' order
    empty = (cols[None, :] * page < (seq + s["grow"])[:, None]) & (cols[None, :] >= (seq // page)[:, None]) & (table < 0)
    at = empty.flatten().nonzero().flatten()
    fresh = (refs == 0).nonzero().flatten()[:at.numel()]
    table.view(-1)[at] = fresh.to(torch.int32)
    refs[fresh] = 1
    return table, seq, refs, torch.ones_like(s["src"]), torch.ones_like(seq), s["pools"]


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pool in s["pools"]:
        pool[dst] = pool[src]
    return s["pools"]


def _plain_compact(s):
    table, refs = s["table"].clone(), s["refs"].clone()
    live = refs > 0
    count = live.sum()
    index = torch.arange(refs.numel(), device=DEV)
    movers = (live & (index >= count)).nonzero().flatten()
    holes = (~live & (index < count)).nonzero().flatten()
    to = index.clone()
    to[movers] = holes
    for pool in s["pools"]:
        pool[holes] = pool[movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    table = torch.where(table >= 0, to[table.clamp_min(0).long()].to(torch.int32), table)
    return table, refs, count.to(torch.int32).view(1), s["pools"]


# ------------------------------------------------------------------ one pass

def _own_run(s):
    import interattn_amd as ia

    c, kind = s["case"], s["case"]["kind"]
    if kind == "prompt":
        return ia.prompt_attention(s["q"], s["k"], s["v"], s["cu"], workspace=s["ws"])
    if kind == "paged":
        return ia.paged_prompt_attention(s["q"], s["pool_k"], s["pool_v"], s["table"], s["seq"], s["cu"],
                                         scales=s["scales"], workspace=s["ws"])
    if kind == "prefix":
        return ia.shared_prefix_decode(s["q"], s["pool_k"], s["pool_v"], s["table"], s["seq"], s["starts"],
                                       s["shared"], scales=s["scales"], workspace=s["ws"])
    if kind == "append":
        lens = ia.append_prompt_kv(s["pool_k"], s["pool_v"], s["table"], s["seq"], s["k"], s["v"], s["cu"])
        return s["pool_k"], s["pool_v"], lens
    if kind == "fork":
        ia.free_sequences(s["table"], s["seq"], s["refs"], s["dst"])
        forked = ia.fork_sequences(s["pools"], s["table"], s["seq"], s["refs"], s["src"], s["dst"],
                                   page_size=c["page"], workspace=s["ws"])
        grown = ia.reserve_pages(s["table"], s["seq"], s["refs"], s["grow"], page_size=c["page"])
        return s["table"], s["seq"], s["refs"], forked, grown, s["pools"]
    if kind == "copy":
        ia.copy_pages(s["pools"], s["src"], s["dst"])
        return s["pools"]
    table, refs = s["table"].clone(), s["refs"].clone()
    count = ia.compact_pages(s["pools"], table, refs, workspace=s["ws"])
    return table, refs, count, s["pools"]


def run(state):
    with torch.no_grad():
        if own:
            return _own_run(state)
        kind = state["case"]["kind"]
        if kind == "paged":
            return _plain_sequences(state, state["new"])
        if kind == "prefix":
            return _plain_sequences(state, [1] * len(state["lens"]))
        return globals()["_plain_" + kind](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, kind = case, case["kind"]
    hkv, d, eb = c["hkv"], c["d"], BYTES[c["kv"]]
    row = 2 * hkv * d * eb  # K and V of one token
    if kind in ("prompt", "paged", "prefix"):
        g = c["g"]
        qb = 4 if c["kv"] == "f32" else 2
        if kind == "prompt":
            new = _lens(c, "lo", "hi", c["n"], 0)
            total, tokens = list(new), sum(new)
        elif kind == "paged":
            new, past = _news_pasts(c)
            total = [a + b for a, b in zip(new, past)]
            tokens = sum(total)
        else:
            shared, tails = _group_lens(c)
            of = [n for m, n in zip(_members(c), shared) for _ in range(m)]
            new, total = [1] * len(of), [a + b for a, b in zip(of, tails)]
            tokens = sum(shared) + sum(tails)
        pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
        scales = 0 if c["kv"] != "fp8" else 2 * 4 * hkv * (tokens // c["page"])
        tables = 0 if kind == "prompt" else 4 * (tokens // c["page"])
        return {"bytes": 2 * sum(new) * hkv * g * d * qb + tokens * row + scales + tables,
                "flops": 4 * pairs * hkv * g * d}
    if kind == "append":
        return {"bytes": 2 * sum(_lens(c, "lo", "hi", c["n"], 0)) * row, "flops": 0}
    page_bytes = c["layers"] * (row * c["page"] + (8 * hkv if c["kv"] == "fp8" else 0))
    if kind == "fork":
        lens = _lens(c, "lo", "hi", c["prompts"], 0)
        n = c["ways"] * sum(1 for x in lens if x % c["page"])
        return {"bytes": 2 * n * page_bytes + 4 * 3 * c["ways"] * sum(x // c["page"] for x in lens), "flops": 0}
    if kind == "copy":
        return {"bytes": 2 * c["count"] * page_bytes, "flops": 0}
    moved = int(c["pages"] * c["live"] * (1 - c["live"]))
    return {"bytes": 2 * moved * page_bytes + 4 * 3 * c["pages"], "flops": 0}


# ------------------------------------------------------------------ the definition, in 64 bits

def _softmax_rows(q, k, v, seen, scale):
    """``q [R, D]``, ``k, v [L, D]`` float64, row r over its first ``seen[r]`` keys."""
    logits = (q @ k.T) * scale
    logits.masked_fill_(torch.arange(k.shape[0], device=q.device)[None] >= seen[:, None], -math.inf)
    return torch.softmax(logits, dim=1) @ v


def exact(case, seed):
    """64-bit outputs of the attention kinds.  The others move data and count pages: their
    outputs are no computed numbers."""
    c, kind = case, case["kind"]
    if kind not in ("prompt", "paged", "prefix"):
        return None
    s = prepare(case, seed)
    g, hkv, d = c["g"], c["hkv"], c["d"]
    new = {"prompt": s["lens"], "paged": s.get("new"), "prefix": [1] * len(s["lens"])}[kind]
    if sum(n * t for n, t in zip(new, s["lens"])) * hkv * g * d > 1e12:
        return None
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    start = 0
    for b, (n, total) in enumerate(zip(new, s["lens"])):
        if total == 0:
            start += n
            continue
        place = torch.arange(total, device=DEV)
        for h in range(hkv):
            if kind == "prompt":
                k, v = s["k"][start:start + n, h].double(), s["v"][start:start + n, h].double()
            else:
                pages, offs = s["table"][b].long()[place // c["page"]], place % c["page"]
                k, v = (s[x][:, h].view(torch.uint8 if c["kv"] == "fp8" else s[x].dtype)[pages, offs]
                        for x in ("pool_k", "pool_v"))
                if c["kv"] == "fp8":
                    k, v = (x.view(DTYPES["fp8"]).float().double() * sc[pages, h, None].double()
                            for x, sc in zip((k, v), s["scales"]))
                k, v = k.double(), v.double()
            most = max(1, (1 << 26) // (g * total))
            for i in range(0, n, most):
                q = s["q"][start + i:start + min(i + most, n), h * g:(h + 1) * g].double()
                seen = torch.arange(total - n + i + 1, total - n + i + 1 + q.shape[0], device=DEV)
                o = _softmax_rows(q.reshape(-1, d), k, v, seen.repeat_interleave(g), d ** -0.5)
                out[start + i:start + i + q.shape[0], h * g:(h + 1) * g] = o.view(q.shape)
        start += n
    return out
