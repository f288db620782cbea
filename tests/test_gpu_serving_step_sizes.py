"""The serving step's operators at offsets past 32 bits, on streams of their own and in place."""

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import beam as B
from tests._util import announce

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pages_past_32_bits(device, kv):
    """Pools of more than 2^31 elements: rows of the last pages written and read back."""
    announce(f"long cache {kv}")
    hkv, d, page, n_pages = 8, 128, 16, 140000
    pool_t = BF16 if kv == "bf16" else FP8
    pk, pv = (torch.empty((n_pages, hkv, page, d), device=device, dtype=pool_t) for _ in "kv")
    assert pk.numel() > 2 ** 31
    scales = None if kv == "bf16" else tuple(torch.ones((n_pages, hkv), device=device) for _ in "kv")
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2], [131071, 131072, 131073]], device=device, dtype=torch.int32)
    cu, seq = torch.tensor([0, 45, 80], device=device, dtype=torch.int32), torch.tensor([0, 10], device=device, dtype=torch.int32)
    rows = torch.randn((80, 2 * hkv, d), device=device).to(BF16)
    k, v = rows.split(hkv, 1)
    _, lens = ia.rotary_append_kv(None, k, v, None, pk, pv, table, seq, cu, scales=scales)
    got = ia.read_kv(pk, pv, table, seq, cu, 80, scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == [45, 45]
    for x, want in zip(got, (k, v)):
        if kv == "bf16":
            assert torch.equal(x, want)
        else:  # half a step of e4m3, or of its smallest codes times the largest scale here
            off = (x.double() - want.double()).abs()
            assert bool((off <= torch.maximum(2.0 ** -4 * want.double().abs(), torch.tensor(2.0 ** -10, device=device))).all())
    # the rows lie where the table says
    if kv == "bf16":
        assert torch.equal(pk[n_pages - 2, :, 12], k[44]) and torch.equal(pv[131073, :, 12], v[79])


def test_rows_past_32_bits(device):
    """Token strides that reach past 2^31 elements."""
    announce("rotary, long strides")
    stride = 2 ** 30
    buf = torch.empty(2 * stride + 2 * 64, device=device, dtype=BF16)
    q = buf.as_strided((3, 2, 64), (stride, 64, 1))
    q.copy_(torch.randn((3, 2, 64), device=device))
    plan, pos = ia.rotary_plan(64, device=device), torch.tensor([5, 70, 900], device=device, dtype=torch.int32)
    want, _ = ia.apply_rotary(q.contiguous(), None, pos, plan)
    ia.apply_rotary(q, None, pos, plan, q_out=q)
    torch.cuda.synchronize()
    assert torch.equal(q.contiguous(), want)


def test_logits_past_32_bits(device):
    announce("beam select, long")
    batch, beams, vocab = 4200, 4, 131072
    logits = torch.empty((batch * beams, vocab), device=device, dtype=BF16)
    assert logits.numel() > 2 ** 31
    logits.fill_(-3.0)
    spots = torch.tensor([7, 130000, 64000, 131071], device=device)
    logits[:, spots] = torch.tensor([5.0, 6.0, 4.0, 5.5], device=device, dtype=BF16)
    scores = torch.arange(beams, device=device, dtype=torch.float32).neg().mul(10).expand(batch, beams).contiguous()
    s, tok, par = ia.beam_select(logits, scores, 4)
    torch.cuda.synchronize()
    assert torch.equal(tok, torch.tensor([130000, 131071, 7, 64000], device=device, dtype=torch.int32).expand(batch, 4))
    assert torch.equal(par, (torch.arange(batch, device=device, dtype=torch.int32) * beams)[:, None].expand(batch, 4))
    keys = B.keys(logits[:beams].double().cpu().numpy(), scores[:1].cpu().numpy())
    want = np.sort(keys[0])[::-1][:4]
    assert np.abs(s[-1].cpu().numpy() - want).max() <= 2.0 ** -21 + 2.0 ** -24 * np.abs(want).max()


def test_on_a_stream_of_its_own(device):
    """Everything on a side stream that waits for its inputs, results read after it is waited for."""
    announce("side stream")
    side = torch.cuda.Stream()
    hkv, d, page = 2, 64, 16
    pk, pv = (torch.zeros((9, hkv, page, d), device=device).to(FP8) for _ in "kv")
    scales = tuple(torch.ones((9, hkv), device=device) for _ in "kv")
    table = torch.arange(8, device=device, dtype=torch.int32).view(2, 4)
    plan, ws = ia.rotary_plan(d, device=device), {}
    q, k, v = (torch.randn((2, h, d), device=device).to(BF16) for h in (4, 2, 2))
    logits, scores = torch.randn((2, 500), device=device), torch.zeros((1, 2), device=device)
    refs = torch.bincount(table.flatten().long(), minlength=9).to(torch.int32)
    results = []
    for stream in (torch.cuda.current_stream(), side):
        a, b, sc = pk.clone(), pv.clone(), tuple(s.clone() for s in scales)
        t, r, lens = table.clone(), refs.clone(), torch.tensor([3, 20], device=device, dtype=torch.int32)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            qo, _ = ia.rotary_append_kv(q, k, v, plan, a, b, t, lens, scales=sc)
            best, tokens, parents = ia.beam_select(logits, scores, 2, workspace=ws)
            ok = ia.reorder_sequences([a, b, *sc], t, lens, r, parents.view(-1), page_size=page, workspace=ws)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        results.append([x.clone() for x in (qo, best, tokens, parents, ok, t, lens, r, a.view(torch.uint8), b.view(torch.uint8), *sc)])
    assert all(torch.equal(x, y) for x, y in zip(*results))


@pytest.mark.parametrize("counts", [[40, 3, 1], [1, 1, 1]])
def test_queries_may_be_turned_in_place(device, counts):
    announce(f"write, queries in place {counts}")
    hkv, d, page = 2, 128, 16
    total = sum(counts)
    table = torch.arange(12, device=device, dtype=torch.int32).view(3, 4)
    seq = torch.tensor([5, 0, 17], device=device, dtype=torch.int32)
    cu = torch.tensor([0, *np.cumsum(counts)], device=device, dtype=torch.int32)
    plan = ia.rotary_plan(d, layout="interleaved", device=device)
    buf = torch.randn((total, 6 + 2 * hkv, d), device=device).to(BF16)
    q, k, v = buf.split([6, hkv, hkv], 1)
    pools = [torch.zeros((12, hkv, page, d), device=device, dtype=BF16) for _ in range(4)]
    rest = buf[:, 6:].clone()
    want, _ = ia.rotary_append_kv(q, k, v, plan, *pools[:2], table, seq, cu)
    got, _ = ia.rotary_append_kv(q, k, v, plan, *pools[2:], table, seq, cu, q_out=q)
    torch.cuda.synchronize()
    assert got.data_ptr() == buf.data_ptr() and torch.equal(buf[:, :6], want) and torch.equal(buf[:, 6:], rest)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_summaries_follow_an_8_bit_cache(device):
    """Block summaries refreshed after every written token are those of a full rebuild, pages whose
    scale rises on the way too (a page lies within a block)."""
    announce("8-bit summaries")
    hkv, d, page, block, cols = 2, 64, 16, 32, 6
    table = torch.randperm(2 * cols, device=device).to(torch.int32).view(2, cols)
    pk, pv = (torch.zeros((2 * cols, hkv, page, d), device=device).to(FP8) for _ in "kv")
    scales = tuple(torch.ones((2 * cols, hkv), device=device) for _ in "kv")
    seq, cu = torch.zeros(2, device=device, dtype=torch.int32), torch.tensor([0, 30, 51], device=device, dtype=torch.int32)
    rows = torch.randn((51, hkv, d), device=device).to(BF16)
    seq = ia.append_prompt_kv(pk, pv, table, seq, rows, rows, cu, scales=scales)
    summ = ia.build_block_summaries(pk, pv, table, seq, block, nb_max=3, full=True, scales=scales)
    for step in range(20):
        old = seq.clone()
        x = (torch.randn((2, hkv, d), device=device) * 2.0 ** (step % 5)).to(BF16)
        ia.append_kv(pk, pv, table, seq, x, -x, scales=scales)
        ia.update_block_summaries(summ, pk, pv, table, old, seq, block, max_new_tokens=1, scales=scales)
        want = ia.build_block_summaries(pk, pv, table, seq, block, nb_max=3, full=True, scales=scales)
        torch.cuda.synchronize()
        for key in ("k_bar", "v_bar", "k_max", "k_min", "block_valid_counts"):
            for b in range(2):
                n = -(-int(seq[b]) // block)
                got, exp = (s[key][b, :, :n] if s[key].dim() == 4 else s[key][b, :n] for s in (summ, want))
                assert torch.equal(got, exp), (step, key)
