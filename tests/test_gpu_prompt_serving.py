"""The prompt, prefix and page calls together, as a server uses them: prompts of different
lengths prefilled and put into pages, forked, continued by another chunk, decoded step by
step behind their shared prefixes, freed and compacted; every attention output against
float64 attention of a host copy of each row's tokens.  And the paged runner's prefill on
this path against a dense model.  Bars: those of the prompt attention tests."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import check, reference

pytestmark = pytest.mark.gpu


class Server:
    """One layer's pool, its page state, and a host copy of every row's K and V."""

    def __init__(self, device, rows, cols, n_pages, hq, hkv, d, page, seed):
        self.dev, self.page, self.hq, self.hkv, self.d = device, page, hq, hkv, d
        self.gen = torch.Generator(device=device)
        self.gen.manual_seed(seed)
        pool = torch.zeros((n_pages, hkv, 2, page, d), device=device, dtype=torch.bfloat16)
        self.pool = (pool[:, :, 0], pool[:, :, 1])
        self.table = torch.full((rows, cols), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(rows, device=device, dtype=torch.int32)
        self.refs = torch.zeros(n_pages, device=device, dtype=torch.int32)
        self.host = [torch.zeros((2, 0, hkv, d)) for _ in range(rows)]
        self.ws = {}

    def i32(self, x):
        return torch.tensor(x, device=self.dev, dtype=torch.int32)

    def rows(self, n, heads):
        return torch.randn((n, heads, self.d), device=self.dev, generator=self.gen).to(torch.bfloat16)

    def reserve(self, grow):
        ok = ia.reserve_pages(self.table, self.lens, self.refs, self.i32(grow), page_size=self.page, workspace=self.ws)
        assert ok.tolist() == [1] * len(grow)

    def extend(self, new):
        """Every row takes ``new[row]`` tokens; attention of those over the row's whole."""
        self.reserve(new)
        total = sum(new)
        k, v, q = self.rows(total, self.hkv), self.rows(total, self.hkv), self.rows(total, self.hq)
        cu = self.i32([sum(new[:i]) for i in range(len(new) + 1)])
        lens = ia.append_prompt_kv(*self.pool, self.table, self.lens, k, v, cu)
        self.lens.copy_(lens)
        out = ia.paged_prompt_attention(q, *self.pool, self.table, self.lens, cu, workspace=self.ws)
        at = 0
        for row, n in enumerate(new):
            self.host[row] = torch.cat([self.host[row], torch.stack([k[at:at + n], v[at:at + n]]).float().cpu()], 1)
            have = self.host[row].shape[1]
            want, mag = reference(q[at:at + n], *self.host[row], have - n, self.d ** -0.5)
            check(out[at:at + n], want, mag, "bf16", have, ("extend", row))
            at += n
        assert self.lens.tolist() == [h.shape[1] for h in self.host]
        return q, k, v, cu, out

    def step(self, starts, shared):
        """One decode step of every row that has tokens (rows without none are at the end)."""
        rows = sum(h.shape[1] > 0 for h in self.host)
        self.reserve([1] * rows + [0] * (len(self.host) - rows))
        k, v, q = self.rows(rows, self.hkv), self.rows(rows, self.hkv), self.rows(rows, self.hq)
        ia.append_kv(*self.pool, self.table[:rows], self.lens[:rows], k, v)
        out = ia.shared_prefix_decode(q, *self.pool, self.table[:rows], self.lens[:rows], self.i32(starts),
                                      self.i32(shared), workspace=self.ws)
        for row in range(rows):
            new = torch.stack([k[row:row + 1], v[row:row + 1]]).float().cpu()
            self.host[row] = torch.cat([self.host[row], new], 1)
            n = self.host[row].shape[1]
            want, mag = reference(q[row:row + 1], *self.host[row], n - 1, self.d ** -0.5)
            check(out[row:row + 1], want, mag, "bf16", n, ("step", row))


def test_a_server_s_day(device):
    announce("server")
    s = Server(device, 9, 20, 90, 8, 2, 64, 16, 3)
    # two prompts, prefilled alone: packed attention equals the paged call over the same pages
    q, k, v, cu, out = s.extend([45, 0, 0, 0, 130, 0, 0, 0, 0])
    packed = ia.prompt_attention(q, k, v, cu, workspace={})
    at = 0
    for row, n in ((0, 45), (4, 130)):
        want, mag = reference(q[at:at + n], k[at:at + n], v[at:at + n], 0, s.d ** -0.5)
        check(packed[at:at + n], want, mag, "bf16", n, ("packed", row))
        at += n
    # three continuations of the first, two of the second
    src, dst = [0, 0, 0, 4, 4], [1, 2, 3, 5, 6]
    ok = ia.fork_sequences([*s.pool], s.table, s.lens, s.refs, s.i32(src), s.i32(dst), page_size=16, workspace=s.ws)
    assert ok.tolist() == [1] * 5
    for a, b in zip(src, dst):
        s.host[b] = s.host[a].clone()
    # the whole pages of a prompt are held once
    assert int((s.refs > 0).sum()) == 2 + 8 + 4 + 3 and int(s.refs.max()) == 4
    for _ in range(3):
        s.step([0, 4, 7], [45, 130])
    # another chunk for some of them, then more steps
    s.extend([20, 1, 0, 33, 0, 17, 5, 0, 0])
    for _ in range(2):
        s.step([0, 4, 7], [45, 130])
    # two rows end; the pool closes up; the rest goes on, one of them without its old group
    ia.free_sequences(s.table, s.lens, s.refs, s.i32([6, 5]))
    s.host[5] = s.host[6] = s.host[7]
    live = ia.compact_pages([*s.pool], s.table, s.refs, workspace=s.ws)
    torch.cuda.synchronize()
    n = int(live)
    assert bool((s.refs[:n] > 0).all()) and bool((s.refs[n:] == 0).all()) and int(s.table.max()) < n
    assert s.refs[:n].tolist() == torch.bincount(s.table[s.table >= 0].long(), minlength=n).tolist()
    for _ in range(2):
        s.step([0, 4], [45])
    assert s.host[0].shape[1] == 45 + 20 + 7


def test_prefill_and_decode_replay_in_a_graph(device):
    """Append, paged prompt attention and shared-prefix decode captured once, replayed over
    changing rows and lengths with eager calls between; every replay equals the eager call
    bit for bit."""
    announce("prompt graph")
    s = Server(device, 4, 12, 60, 8, 2, 128, 16, 5)
    s.extend([30, 50, 0, 17])
    s.reserve([60, 60, 60, 60])
    cu = s.i32([0, 5, 5, 12, 20])
    k, v, q, q1 = s.rows(20, 2), s.rows(20, 2), s.rows(20, 8), s.rows(4, 8)
    starts, shared, past = s.i32([0, 2, 4]), s.i32([16, 0]), s.lens.clone()
    s.table[1, 0] = s.table[0, 0]
    ws, out, one = {}, torch.zeros_like(q), torch.zeros_like(q1)
    lens = torch.zeros_like(past)

    def run(ws, out, one):
        ia.append_prompt_kv(*s.pool, s.table, past, k, v, cu, new_seq_lens=lens)
        ia.paged_prompt_attention(q, *s.pool, s.table, lens, cu, out=out, workspace=ws)
        ia.shared_prefix_decode(q1, *s.pool, s.table, lens, starts, shared, out=one, workspace=ws)

    run(ws, out, one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph):
            run(ws, out, one)
    torch.cuda.current_stream().wait_stream(side)
    for i, sizes in enumerate([[5, 5, 12, 20], [0, 9, 9, 20], [20, 20, 20, 20], [1, 2, 3, 4]]):
        cu.copy_(s.i32([0] + sizes))
        past.copy_(s.i32([30 + i, 47 - i, 3 * i, 17]))
        for x in (k, v, q, q1):
            x.copy_(torch.randn(x.shape, device=device, generator=s.gen))
        want, want1 = torch.full_like(q, 9.0), torch.full_like(q1, 9.0)
        out.fill_(9.0)
        run({}, want, want1)
        torch.cuda.synchronize()
        before = lens.tolist()
        lens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == before == [a + b for a, b in zip([30 + i, 47 - i, 3 * i, 17], [
            y - x for x, y in zip([0] + sizes, sizes)])]
        assert torch.equal(out, want) and torch.equal(one, want1), i
        assert bool((out[sizes[-1]:] == 9.0).all())


def test_calls_on_a_side_stream_and_twice_at_once(device):
    """Two streams, each with its own workspace, run the same calls over each other."""
    announce("prompt streams")
    s = Server(device, 3, 80, 260, 8, 2, 128, 16, 7)
    s.extend([1100, 900, 1200])
    q, q1 = s.rows(30, 8), s.rows(3, 8)
    cu, starts, shared = s.i32([0, 10, 20, 30]), s.i32([0, 1]), s.i32([0])
    want = ia.paged_prompt_attention(q, *s.pool, s.table, s.lens, cu, workspace={})
    want1 = ia.shared_prefix_decode(q1, *s.pool, s.table, s.lens, starts, shared, workspace={})
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            ws = {}
            for _ in range(5):
                a = ia.paged_prompt_attention(q, *s.pool, s.table, s.lens, cu, workspace=ws)
                b = ia.shared_prefix_decode(q1, *s.pool, s.table, s.lens, starts, shared, workspace=ws)
            got.append((a, b, ws))
    torch.cuda.synchronize()
    for a, b, _ in got:
        assert torch.equal(a, want) and torch.equal(b, want1)


def test_refusals_with_device_tensors(device):
    announce("prompt refusals")
    s = Server(device, 2, 4, 8, 8, 2, 64, 16, 1)
    q, k = s.rows(5, 8), s.rows(5, 2)
    cu = s.i32([0, 2, 5])
    host = torch.zeros(3, dtype=torch.int32)
    bad = [
        lambda: ia.prompt_attention(q, k, k, host),
        lambda: ia.prompt_attention(q, k.float(), k, cu),
        lambda: ia.prompt_attention(q, k.float(), k.float(), cu),
        lambda: ia.prompt_attention(q, k[:4], k[:4], cu),
        lambda: ia.prompt_attention(q, k[:, :1], k, cu),
        lambda: ia.prompt_attention(q[..., ::2], k, k, cu),
        lambda: ia.prompt_attention(q, k, k, cu.long()),
        lambda: ia.prompt_attention(q, k, k, cu[:0]),
        lambda: ia.prompt_attention(q, k, k, cu, out=torch.empty_like(k)),
        lambda: ia.prompt_attention(q, k, k, cu, out=torch.empty_like(q).half()),
        lambda: ia.prompt_attention(q.half(), k, k, cu),
        lambda: ia.prompt_attention(q[:, :7], k, k, cu),
        lambda: ia.paged_prompt_attention(q, *s.pool, s.table, s.lens[:1], cu),
        lambda: ia.paged_prompt_attention(q, *s.pool, s.table[:1], s.lens, cu),
        lambda: ia.paged_prompt_attention(q, s.pool[0].to(torch.float8_e4m3fn), s.pool[1].to(torch.float8_e4m3fn),
                                          s.table, s.lens, cu),
        lambda: ia.shared_prefix_decode(q, *s.pool, s.table, s.lens, cu, cu),
        lambda: ia.shared_prefix_decode(q[:2], *s.pool, s.table, s.lens, cu[:1], cu[:1]),
        lambda: ia.append_prompt_kv(*s.pool, s.table, s.lens, k, k, cu, new_seq_lens=s.lens),
        lambda: ia.append_prompt_kv(*s.pool, s.table, s.lens, k.float(), k.float(), cu),
        lambda: ia.append_prompt_kv(*s.pool, s.table, s.lens, k[:4], k, cu),
        lambda: ia.append_prompt_kv(*s.pool, s.table, s.lens, q, q, cu),
        lambda: ia.copy_pages([s.pool[0], s.pool[1][:7]], cu, cu),
        lambda: ia.copy_pages([s.pool[0]], cu, cu[:2]),
        lambda: ia.fork_sequences([s.pool[0][:7]], s.table, s.lens, s.refs, cu, cu, page_size=16),
        lambda: ia.fork_sequences([s.pool[0]], s.table, s.lens, s.refs, cu, cu, page_size=0),
        lambda: ia.fork_sequences([s.pool[0]], s.table.t(), s.lens, s.refs, cu, cu, page_size=16),
        lambda: ia.reserve_pages(s.table, s.lens, s.refs, cu, page_size=16),
        lambda: ia.free_sequences(s.table, s.lens, s.refs.long(), cu),
        lambda: ia.compact_pages([s.pool[0]], s.table.long(), s.refs),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
    torch.cuda.synchronize()


@pytest.mark.parametrize("full_layers", [0, 1])
def test_paged_runner_with_its_prefill_on_this_path(full_layers, device):
    """k >= every block is exact attention, so prefill and a batch-2 teacher-forced decode give
    the dense model's logits, as the SDPA prefill does (the same bar)."""
    from tests.test_gpu_decode import _dense_batch_greedy, _model, _paged_runner_logits

    announce(f"paged runner, native prompt, full_layers={full_layers}")
    model = _model(device)
    ids = torch.randint(0, 256, (2, 150), generator=torch.Generator().manual_seed(6)).to(device)
    ref_tok, ref_logits = _dense_batch_greedy(model, ids, 5)
    got, runner = _paged_runner_logits(model, ids, ref_tok, max_seq_len=256, block_size=32, k=8,
                                       full_attention_layers=full_layers, native_prompt=True)
    for i, (a, b) in enumerate(zip(got, ref_logits)):
        err = (a - b).abs().max().item()
        assert err < 1e-3, f"step {i}: max |logit diff| {err}"
    for seq in runner.seq_lens:
        assert seq.cpu().tolist() == [155] * 2
