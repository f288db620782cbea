"""The serving step's operators together: prompts turned into the cache, decode steps on it,
beams selected and their pages reordered, over several steps; and the paged runner on an 8-bit
cache."""

import math

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import beam as B
from oracle import rotary as R
from tests._util import announce

pytestmark = pytest.mark.gpu

HKV, G, D, PAGE, VOCAB, LAYERS = 2, 2, 64, 16, 97, 2
HQ = HKV * G


class Toy:
    """Two attention layers between an embedding and its transpose; weights in float32."""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        width = HQ * D
        self.emb = rng.standard_normal((VOCAB, width)).astype(np.float32)
        self.qkv = [(rng.standard_normal((width, (HQ + 2 * HKV) * D)) / math.sqrt(width)).astype(np.float32)
                    for _ in range(LAYERS)]
        self.out = [(rng.standard_normal((width, width)) / math.sqrt(width)).astype(np.float32) for _ in range(LAYERS)]
        self.head = (rng.standard_normal((width, VOCAB)) * 0.3 / math.sqrt(width)).astype(np.float32)


class Plain:
    """Beam search in 64 bits with every beam's keys and values copied."""

    def __init__(self, toy, w):
        self.toy, self.w = toy, w

    def step(self, tokens, caches):
        """``tokens`` of one sequence behind ``caches`` (a (K, V) list per layer, extended in place)."""
        x = self.toy.emb[tokens].astype(np.float64)
        for layer in range(LAYERS):
            y = (x @ self.toy.qkv[layer].astype(np.float64)).reshape(len(tokens), -1, D)
            q, k, v = y[:, :HQ], y[:, HQ:HQ + HKV], y[:, HQ + HKV:]
            past = caches[layer][0].shape[0]
            pos = np.arange(past, past + len(tokens))
            q, k = R.turn(q, pos, self.w), R.turn(k, pos, self.w)
            ks, vs = caches[layer] = (np.concatenate([caches[layer][0], k]), np.concatenate([caches[layer][1], v]))
            kk, vv = ks.repeat(G, 1), vs.repeat(G, 1)
            s = np.einsum("qhd,khd->hqk", q, kk) * D ** -0.5
            s = np.where(np.arange(len(ks))[None, None] > pos[None, :, None], -np.inf, s)
            p = np.exp(s - s.max(-1, keepdims=True))
            o = np.einsum("hqk,khd->qhd", p / p.sum(-1, keepdims=True), vv)
            x = x + o.reshape(len(tokens), -1) @ self.toy.out[layer].astype(np.float64)
        return x @ self.toy.head.astype(np.float64)


class Served:
    """The same on this library: a paged cache of ``rows`` rows, shared by all layers' pools."""

    def __init__(self, toy, device, rows, max_len, n_pages, kv_dtype):
        self.dev = device
        self.w = [[torch.from_numpy(x).to(device) for x in xs] for xs in (toy.qkv, toy.out)]
        self.emb, self.head = torch.from_numpy(toy.emb).to(device), torch.from_numpy(toy.head).to(device)
        self.plan = ia.rotary_plan(D, base=100.0, device=device)
        shape = (n_pages, HKV, PAGE, D)
        self.pools = [tuple(torch.zeros(shape, device=device).to(kv_dtype) for _ in "kv") for _ in range(LAYERS)]
        fp8 = kv_dtype == torch.float8_e4m3fn
        self.rows = torch.bfloat16 if fp8 else kv_dtype
        self.scales = [tuple(torch.ones(shape[:2], device=device) for _ in "kv") if fp8 else None for _ in range(LAYERS)]
        self.tensors = [t for p in self.pools for t in p] + [t for s in self.scales if s for t in s]
        self.table = torch.full((rows, -(-max_len // PAGE)), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(rows, device=device, dtype=torch.int32)
        self.refs = torch.zeros(n_pages, device=device, dtype=torch.int32)
        self.ws = {}

    def ints(self, x):
        return torch.tensor(x, device=self.dev, dtype=torch.int32)

    def forward(self, tokens, cu, attend):
        x = self.emb[tokens]
        for layer in range(LAYERS):
            y = (x @ self.w[0][layer]).view(x.shape[0], -1, D).to(self.rows)
            q, k, v = y.split([HQ, HKV, HKV], 1)
            (pk, pv), sc = self.pools[layer], self.scales[layer]
            q, after = ia.rotary_append_kv(q, k, v, self.plan, pk, pv, self.table, self.lens, cu, scales=sc,
                                           new_seq_lens=torch.empty_like(self.lens))
            x = x + attend(layer, q, after).reshape(x.shape[0], -1) @ self.w[1][layer]
        self.lens.copy_(after)
        return x @ self.head


def search(device, kv_dtype, prompts, beams, steps, check):
    batch = len(prompts)
    rows = batch * beams
    toy = Toy(5)
    longest = max(map(len, prompts)) + steps + 1
    s = Served(toy, device, rows, longest, rows * (-(-longest // PAGE)) + 4, kv_dtype)
    # prompts into the first row of each request's beams
    counts = [len(prompts[i // beams]) if i % beams == 0 else 0 for i in range(rows)]
    cu = s.ints([0, *np.cumsum(counts)])
    assert bool(ia.reserve_pages(s.table, s.lens, s.refs, s.ints(counts), page_size=PAGE).all())

    def prompt(layer, q, after):
        (pk, pv), sc = s.pools[layer], s.scales[layer]
        out = ia.paged_prompt_attention(q, pk, pv, s.table, after, cu, scales=sc, workspace=s.ws,
                                        out_dtype=torch.float32)
        check(layer, q, after, cu, out, s)
        return out

    logits = s.forward(torch.tensor(sum(prompts, []), device=device), cu, prompt)
    last = (cu[1:] - 1).view(batch, beams)[:, :1].expand(batch, beams).reshape(-1).long()
    scores = torch.full((batch, beams), -math.inf, device=device)
    scores[:, 0] = 0
    logits = logits[last]
    shared, starts = s.ints([len(p) for p in prompts]), s.ints(range(0, rows + 1, beams))
    one_each = s.ints(range(rows + 1))

    def decode(layer, q, after):
        (pk, pv), sc = s.pools[layer], s.scales[layer]
        out = ia.shared_prefix_decode(q, pk, pv, s.table, after, starts, shared, scales=sc, workspace=s.ws,
                                      out_dtype=torch.float32)
        check(layer, q, after, one_each, out, s)
        return out

    history = []
    for _ in range(steps):
        scores, tokens, parents = ia.beam_select(logits, scores, beams, workspace=s.ws)
        ok = ia.reorder_sequences(s.tensors, s.table, s.lens, s.refs, parents.view(-1), page_size=PAGE, workspace=s.ws)
        grown = ia.reserve_pages(s.table, s.lens, s.refs, torch.ones_like(s.lens), page_size=PAGE, workspace=s.ws)
        logits = s.forward(tokens.view(-1).long(), None, decode)
        history.append((scores, tokens, parents))
        assert bool(ok.all()) and bool(grown.all())
    torch.cuda.synchronize()
    table, refs = s.table.cpu().numpy(), s.refs.cpu().numpy()
    assert np.array_equal(np.bincount(table[table >= 0], minlength=len(refs)), refs)
    return toy, s, [[x.cpu().numpy() for x in h] for h in history]


def prompts_of(lens, seed=1):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, VOCAB, n).tolist() for n in lens]


@pytest.mark.parametrize("lens,beams,steps", [([21, 5], 3, 20), ([16], 4, 18), ([1, 40, 33], 2, 17)])
def test_beam_search_is_the_plain_one(device, lens, beams, steps):
    """float32 pools: the same tokens and parents at every step, scores within what float32
    attention over two layers adds up to (measured against 64 bits the bar is 2^-24 for each of
    the 4 (D + width) roundings of a layer's sums, per step)."""
    announce(f"beam search {lens} {beams}")
    prompts = prompts_of(lens)
    toy, _, got = search(device, torch.float32, prompts, beams, steps, lambda *a: None)
    plain = Plain(toy, ia.rotary_frequencies(D, base=100.0)[0])
    for b, prompt in enumerate(prompts):
        caches = [[(np.zeros((0, HKV, D)), np.zeros((0, HKV, D)))] * LAYERS]
        logits = plain.step(prompt, caches[0])[-1:].repeat(beams, 0)
        caches = [list(caches[0]) for _ in range(beams)]
        scores = np.full((1, beams), -np.inf)
        scores[0, 0] = 0
        for step in range(steps):
            keys = B.keys(logits, scores)
            place = B.select(keys, beams)[0]
            scores, tokens, parents = keys[:, place], place % VOCAB, place // VOCAB
            assert got[step][1][b].tolist() == tokens.tolist(), (b, step)
            assert (got[step][2][b] - b * beams).tolist() == parents.tolist(), (b, step)
            bar = (step + 1) * LAYERS * 4 * (D + HQ * D) * 2.0 ** -24 * 8
            assert np.abs(got[step][0][b] - scores[0]).max() <= bar
            caches = [list(caches[p]) for p in parents]
            logits = np.concatenate([plain.step([t], c) for t, c in zip(tokens, caches)])


@pytest.mark.parametrize("lens,beams,steps", [([21, 5], 3, 20), ([1, 50], 4, 18)])
def test_beam_search_on_an_8_bit_cache(device, lens, beams, steps):
    """Attention of every step over the rows that the cache holds, read back, in 64 bits; what
    the cache holds is within half a step of e4m3 of what was written.  fp8 pools are attended
    in bf16 products (queries and weights rounded to 2^-8 each, three roundings with the output
    kept in float32): bar 4 * 2^-8 of the values' largest magnitude."""
    announce(f"beam search, 8 bits {lens} {beams}")

    def check(layer, q, after, cu, out, s):
        (pk, pv), sc = s.pools[layer], s.scales[layer]
        n = after.tolist()
        rows = s.ints([0, *np.cumsum(n)])
        k, v = ia.read_kv(pk, pv, s.table, torch.zeros_like(after), rows, sum(n), scales=sc, out_dtype=torch.float32)
        torch.cuda.synchronize()
        k, v, q, out = (x.double().cpu() for x in (k, v, q, out))
        edges, at = cu.tolist(), 0
        for b, total in enumerate(n):
            new = edges[b + 1] - edges[b]
            for i in range(new):
                seen = total - new + i + 1
                for h in range(HQ):
                    kk, vv = k[at:at + seen, h // G], v[at:at + seen, h // G]
                    want = torch.softmax(kk @ q[edges[b] + i, h] * D ** -0.5, 0) @ vv
                    off = float((out[edges[b] + i, h] - want).abs().max())
                    assert off <= 4 * 2.0 ** -8 * max(float(vv.abs().max()), 1e-6), (layer, b, i, h, off)
            at += total

    _, s, got = search(device, torch.float8_e4m3fn, prompts_of(lens), beams, steps, check)
    for scores, tokens, parents in got:
        assert np.isfinite(scores).all() and (np.diff(scores, axis=1) <= 0).all()
    for scales in s.scales:
        for x in scales:
            x = x.cpu().numpy()
            assert (np.frexp(x)[0] == 0.5).all()  # powers of two


def test_the_paged_runner_on_an_8_bit_cache(device):
    """What the pools hold after a prompt and some decode steps is what the model cached, to
    e4m3: half a step of the value, 2^-4, or of the smallest codes, 2^-10 scales, where pages
    whose scale rose on the way add 2^-10 of each smaller scale: 2^-9 in all.  All blocks
    selected: the logits are the bf16 cache's but for that; finite here."""
    pytest.importorskip("transformers")
    from tests.test_gpu_decode import _dense_batch_greedy, _model
    from interattn_amd.decode import PagedTopkDecodeRunner, condition_block_decode_context

    for native, full in ((True, 0), (False, 1)):
        announce(f"paged runner, 8 bits {native}")
        model = _model(device, dtype=torch.bfloat16, head_dim=128)
        ids = torch.randint(0, 256, (2, 70), generator=torch.Generator().manual_seed(3)).to(device)
        tokens, _ = _dense_batch_greedy(model, ids, 20)
        runner = PagedTopkDecodeRunner(model=model, batch_size=2, max_seq_len=128, block_size=32, k=8,
                                       full_attention_layers=full, native_prompt=native, kv_dtype=torch.float8_e4m3fn)
        with condition_block_decode_context(runner), torch.no_grad():
            out = model(input_ids=ids, use_cache=True, logits_to_keep=1)
            for step in range(20):
                out = model(input_ids=tokens[:, step:step + 1], past_key_values=out.past_key_values, use_cache=True,
                            logits_to_keep=1)
                assert bool(torch.isfinite(out.logits).all())
        cu = torch.tensor([0, 90, 180], device=device, dtype=torch.int32)
        first = torch.zeros(2, device=device, dtype=torch.int32)
        for i, layer in enumerate(out.past_key_values.layers):
            assert runner.seq_lens[i].tolist() == [90, 90]
            pk, pv = runner.pools[i]
            got = ia.read_kv(pk, pv, runner.block_table, first, cu, 180, scales=runner.scales[i], out_dtype=torch.float32)
            torch.cuda.synchronize()
            for x, want, scale in zip(got, (layer.keys, layer.values), runner.scales[i]):
                want = want.transpose(1, 2).reshape(180, *x.shape[1:]).double()
                pages = runner.block_table[:, :6].long()
                s = scale[pages].repeat_interleave(16, 1)[:, :90].reshape(180, -1, 1).double()
                bar = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -9 * s)
                assert bool(((x.double() - want).abs() <= bar).all())
    for refused, kv in ((model, torch.float16), (_model(device), torch.float8_e4m3fn)):
        with pytest.raises(ValueError, match="kv_dtype"):
            PagedTopkDecodeRunner(model=refused, batch_size=2, max_seq_len=128, block_size=32, k=8, kv_dtype=kv)
    with pytest.raises(ValueError, match="divides block_size"):
        PagedTopkDecodeRunner(model=model, batch_size=2, max_seq_len=128, block_size=16, page_size=32, k=8,
                              kv_dtype=torch.float8_e4m3fn)
