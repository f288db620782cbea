"""K/V into pages, 8-bit ones too, and back, against page-by-page oracles.

Codes, scales and re-encoded rows are compared bit for bit where nothing is turned (the
rows are exact inputs, scales are powers of two).  Turned keys: float32 sums are off by the
rotation's bar (tests/test_gpu_rotary.py), codes by half a step of e4m3 more: 2^-4 of the value,
2^-10 scales where it is subnormal."""

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import quantise as Q
from oracle import rotary as R
from tests._util import announce

pytestmark = pytest.mark.gpu

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def codes(pool):
    """(e4m3 has two NaN codes, 0x7F and 0xFF: one here)"""
    c = pool.view(torch.uint8).cpu().numpy()
    return np.where(c == 0xFF, 0x7F, c)


def make_pool(gen, n_pages, hkv, page, d, dtype, paired, device):
    """A pool of old contents: what no call writes has to stay."""
    if paired:
        buf = torch.empty((n_pages, hkv, 2, page, d), device=device, dtype=dtype)
        k, v = buf[:, :, 0], buf[:, :, 1]
    else:
        k, v = (torch.empty((n_pages, hkv, page, d), device=device, dtype=dtype) for _ in "kv")
    for p in (k, v):
        if dtype == FP8:
            c = torch.randint(0, 256, p.shape, device=device, generator=gen).to(torch.uint8)
            p.view(torch.uint8).copy_(torch.where((c & 0x7F) == 0x7F, torch.zeros_like(c), c))
        else:
            p.normal_(generator=gen)
    return k, v


def make_table(gen, n_seq, cols, n_pages, device):
    return torch.randperm(n_pages, device=device, generator=gen)[:n_seq * cols].to(torch.int32).view(n_seq, cols)


def cu_of(counts, device):
    return torch.tensor([0, *np.cumsum(counts)], device=device, dtype=torch.int32)


def oracle_write(pool, scale, table, past, counts, rows, page):
    """Codes and scales after the rows [tokens, Hkv, D] were written (numpy, in place)."""
    at = 0
    for b, (p, n) in enumerate(zip(past, counts)):
        done = 0
        while done < n:
            pos = p + done
            lo, take = pos % page, min(n - done, page - pos % page)
            pg = table[b, pos // page] if pos // page < table.shape[1] else -1
            if 0 <= pg < pool.shape[0]:
                for h in range(pool.shape[1]):
                    pool[pg, h], scale[pg, h] = Q.write_page(pool[pg, h], scale[pg, h], lo,
                                                             rows[at + done:at + done + take, h])
            done += take
        at += n


def setup(device, seed, n_seq, hkv, page, d, cols, paired=False, dtype=FP8, spare=3):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    n_pages = n_seq * cols + spare
    k, v = make_pool(g, n_pages, hkv, page, d, dtype, paired, device)
    table = make_table(g, n_seq, cols, n_pages, device)
    scales = None
    if dtype == FP8:
        scales = tuple(torch.exp2(torch.randint(-6, 3, (n_pages, hkv), device=device, generator=g).float()) for _ in "kv")
    return g, k, v, table, scales


def check_fp8(pool_k, pool_v, scales, before, table, past, counts, k, v, page):
    for pool, scale, (c0, s0), rows in ((pool_k, scales[0], before[0], k), (pool_v, scales[1], before[1], v)):
        want_c, want_s = c0.copy(), s0.copy()
        oracle_write(want_c, want_s, table.cpu().numpy(), past, counts, rows.float().cpu().numpy().astype(np.float64), page)
        assert np.array_equal(scale.cpu().numpy(), want_s)
        assert np.array_equal(codes(pool), want_c)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d,page,hkv,paired,past,counts", [
    (128, 16, 2, False, [0, 5, 16, 31, 40], [1, 40, 16, 3, 0]),
    (64, 16, 1, True, [7, 0], [9, 100]),
    (128, 32, 8, True, [3, 17, 32, 0], [20, 70, 5, 1]),
    (64, 64, 3, False, [50, 10, 63], [100, 6, 2]),
    (128, 48, 1, False, [47, 20], [49, 28]),
    (64, 128, 2, True, [100, 0, 5], [200, 128, 100]),
    (128, 256, 1, False, [255, 3], [2, 250]),
])
def test_codes_and_scales(device, dtype, d, page, hkv, paired, past, counts):
    """Rows of sizes that make some begun pages keep their scale and others change it."""
    announce(f"8-bit write {dtype} {d} {page} {past} {counts}")
    cols = max(-(-(p + n) // page) for p, n in zip(past, counts)) + 1
    g, pk, pv, table, scales = setup(device, page + d, len(past), hkv, page, d, cols, paired)
    total = sum(counts) + 4  # rows of no sequence behind
    mag = torch.exp2(torch.randint(-8, 9, (total, hkv, 1), device=device, generator=g).float())
    k, v = ((torch.randn((total, hkv, d), device=device, generator=g) * mag).to(dtype) for _ in "kv")
    before = [(codes(p).copy(), s.cpu().numpy().copy()) for p, s in zip((pk, pv), scales)]
    seq, cu = torch.tensor(past, device=device, dtype=torch.int32), cu_of(counts, device)
    lens = ia.append_prompt_kv(pk, pv, table, seq, k, v, cu, scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == [a + b for a, b in zip(past, counts)] and seq.tolist() == past
    check_fp8(pk, pv, scales, before, table, past, counts, k, v, page)


def test_values_at_the_edges(device):
    """Zeros, subnormals of the code, the least scale, values that are not finite, the largest
    ones, sums of a page that only the last row sets; a kept scale that is no power of two."""
    announce("8-bit write, edges")
    d, page, hkv = 64, 16, 1
    cases = [
        [0.0], [2.0 ** -140], [1e-38, -1e-30], [3.3e38, 1.0, -2.0 ** -100], [float("inf"), 3.0], [float("nan"), -0.5],
        [float("-inf"), float("nan")], [448.0, 448.0 * 2.0 ** -15, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10],
        [1.75, 1.7500001], [449.0], [0.06250001, 0.0625],
    ]
    g, pk, pv, table, scales = setup(device, 1, len(cases), hkv, page, d, 1)
    rows = torch.zeros((len(cases) * 8, hkv, d), device=device)
    for i, vals in enumerate(cases):
        for j, x in enumerate(vals):
            rows[8 * i + j % 8, 0, (5 * j) % d] = x
        rows[8 * i + 7, 0, 63] = vals[0]
    counts, past = [8] * len(cases), [0] * len(cases)
    cu = cu_of(counts, device)
    before = [(codes(p).copy(), s.cpu().numpy().copy()) for p, s in zip((pk, pv), scales)]
    v = -rows.flip(2)
    lens = ia.append_prompt_kv(pk, pv, table, torch.zeros(len(cases), device=device, dtype=torch.int32), rows, v, cu,
                               scales=scales)
    torch.cuda.synchronize()
    check_fp8(pk, pv, scales, before, table, past, counts, rows, v, page)
    # begun pages: scales that are no powers of two, that are 0, not finite or too small
    for i, s in enumerate([0.3, 0.0, float("inf"), float("nan"), 1e-40, -1.0, 0.7, 2.0, 1e-3, 5.0, 1.1]):
        scales[0][table[i, 0].long()] = s
        scales[1][table[i, 0].long()] = s
    before = [(codes(p).copy(), s.cpu().numpy().copy()) for p, s in zip((pk, pv), scales)]
    k2, v2 = (torch.randn((len(cases), hkv, d), device=device, generator=g) * 100 for _ in "kv")
    ia.append_kv(pk, pv, table, lens, k2, v2, scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == [9] * len(cases)
    check_fp8(pk, pv, scales, before, table, [8] * len(cases), [1] * len(cases), k2, v2, page)


@pytest.mark.parametrize("page", [16, 32])
def test_token_by_token(device, page):
    """40 single tokens whose sizes rise and fall, every step against the oracle."""
    announce(f"8-bit write, token by token {page}")
    n_seq, hkv, d = 3, 2, 128
    g, pk, pv, table, scales = setup(device, 9, n_seq, hkv, page, d, 4)
    seq = torch.tensor([0, 13, 30], device=device, dtype=torch.int32)
    for step in range(40):
        size = 2.0 ** ((step * 7) % 11 - 5)
        k, v = ((torch.randn((n_seq, hkv, d), device=device, generator=g) * size).bfloat16() for _ in "kv")
        past = seq.tolist()
        before = [(codes(p).copy(), s.cpu().numpy().copy()) for p, s in zip((pk, pv), scales)]
        ia.append_kv(pk, pv, table, seq, k, v, scales=scales)
        torch.cuda.synchronize()
        assert seq.tolist() == [min(p + 1, 4 * page) if p < 4 * page else p for p in past]
        check_fp8(pk, pv, scales, before, table, past, [1] * n_seq, k, v, page)


def test_one_by_one_is_all_at_once(device):
    """A page written token by token holds what one written at once does, but for values that
    were subnormal on the way (here none: sizes within 2^5 of each other)."""
    announce("8-bit write, one by one")
    n, hkv, d, page = 37, 2, 64, 16
    g, pk, pv, table, scales = setup(device, 4, 1, hkv, page, d, 3)
    rows = torch.sign(torch.randn((n, hkv, d), device=device, generator=g)) * (
        1 + 31 * torch.rand((n, hkv, d), device=device, generator=g))
    pk2, pv2, sc2 = pk.clone(), pv.clone(), tuple(s.clone() for s in scales)
    cu = cu_of([n], device)
    ia.append_prompt_kv(pk, pv, table, torch.zeros(1, device=device, dtype=torch.int32), rows, -rows, cu, scales=scales)
    seq = torch.zeros(1, device=device, dtype=torch.int32)
    for i in range(n):
        ia.append_kv(pk2, pv2, table, seq, rows[i:i + 1], -rows[i:i + 1], scales=sc2)
    torch.cuda.synchronize()
    one, two = (ia.read_kv(a, b, table, torch.zeros(1, device=device, dtype=torch.int32), cu, n, scales=s, out_dtype=F32)
                for a, b, s in ((pk, pv, scales), (pk2, pv2, sc2)))
    # values were rounded once: against the largest scale a page ever has, 2^-4 relative
    for a, b, x in zip(one, two, (rows, -rows)):
        assert torch.equal(a, b)
        assert bool(((a - x).abs() <= x.abs() * 2.0 ** -4).all())


@pytest.mark.parametrize("kv,dtype", [("bf16", BF16), ("f32", F32), ("fp8", BF16), ("fp8", F32)],
                         ids=["bf16", "f32", "fp8-bf16", "fp8-f32"])
@pytest.mark.parametrize("d,page,rot,layout,hkv,group,past,counts,paired", [
    (128, 16, 128, "half", 2, 4, [0, 5, 30], [3, 40, 1], False),
    (64, 32, 32, "interleaved", 4, 2, [100, 0], [50, 33], True),
    (128, 64, 70, "half", 1, 3, [60], [75], False),
    (64, 16, 10, "interleaved", 1, 1, [0, 1], [0, 17], False),
    (128, 128, 128, "half", 2, 1, [100, 0], [60, 128], False),        # pages of more parts than waves
    (64, 256, 26, "half", 1, 2, [7, 250], [500, 30], False),
    (128, 256, 64, "interleaved", 1, 1, [200], [300], True),
])
def test_turned_keys_and_queries(device, kv, dtype, d, page, rot, layout, hkv, group, past, counts, paired):
    announce(f"turned write {kv} {dtype} {d} {page} {rot} {layout}")
    pool_t = {"bf16": BF16, "f32": F32, "fp8": FP8}[kv]
    cols = max(-(-(p + n) // page) for p, n in zip(past, counts)) + 1
    g, pk, pv, table, scales = setup(device, rot, len(past), hkv, page, d, cols, paired, pool_t)
    total, hq = sum(counts), hkv * group
    buf = torch.randn((total, hq + 2 * hkv, d), device=device, generator=g).to(dtype)
    q, k, v = buf.split([hq, hkv, hkv], 1)
    plan = ia.rotary_plan(rot, base=1000.0, layout=layout, factor=1.25, device=device)
    w, _ = ia.rotary_frequencies(rot, base=1000.0)
    seq, cu = torch.tensor(past, device=device, dtype=torch.int32), cu_of(counts, device)
    where = np.concatenate([np.arange(p, p + n) for p, n in zip(past, counts)])
    old = [p.view(torch.uint8).clone() for p in (pk, pv)]
    qo, lens = ia.rotary_append_kv(q, k, v, plan, pk, pv, table, seq, cu, scales=scales)
    got_k, got_v = ia.read_kv(pk, pv, table, seq, cu, total, scales=scales, out_dtype=F32)
    torch.cuda.synchronize()
    assert lens.tolist() == [a + b for a, b in zip(past, counts)]
    x64 = [x.double().cpu().numpy() for x in (q, k, v)]
    for got, x in ((qo, x64[0]), (got_k, x64[1])):
        want = R.turn(x, where, w, layout, 1.25)
        pair = np.abs(R.turn(np.abs(x), where * 0, w, layout, 1.25))  # |x| factor, then its pair's sum
        size = pair.copy()
        if layout == "half":
            size[..., :rot // 2] = size[..., rot // 2:rot] = pair[..., :rot // 2] + pair[..., rot // 2:rot]
        else:
            size[..., 0:rot:2] = size[..., 1:rot:2] = pair[..., 0:rot:2] + pair[..., 1:rot:2]
        bar = 8 * 2.0 ** -24 * size
        if x is x64[0]:
            bar = bar + (2.0 ** -8 * size if dtype == BF16 else 0)  # (half a step of bf16: eps / 2)
        elif kv == "bf16":
            bar = bar + 2.0 ** -8 * size
        elif kv == "fp8":
            rows = scale_rows(scales[0], table, past, counts, page)
            bar = bar * (1 + 2.0 ** -4) + np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * rows[:, :, None])
        off = np.abs(got.double().cpu().numpy() - want)
        assert (off <= bar).all(), (off - bar).max()
    if kv == "fp8":
        rows = scale_rows(scales[1], table, past, counts, page)
        off = np.abs(got_v.double().cpu().numpy() - x64[2])
        assert (off <= np.maximum(2.0 ** -4 * np.abs(x64[2]), 2.0 ** -10 * rows[:, :, None])).all()
    else:
        assert torch.equal(got_v, v.float())
        # nothing but the sequences' rows is written
        for pool, before in zip((pk, pv), old):
            now = pool.view(torch.uint8).clone()
            for b, (p, n) in enumerate(zip(past, counts)):
                for t in range(p, p + n):
                    pg = table[b, t // page]
                    now[pg, :, t % page] = before[pg, :, t % page]
            assert torch.equal(now, before)


def scale_rows(scale, table, past, counts, page):
    """[tokens, Hkv]: each packed token's page scale."""
    s, t = scale.cpu().numpy().astype(np.float64), table.cpu().numpy()
    return np.concatenate([s[t[b, np.arange(p, p + n) // page]] for b, (p, n) in enumerate(zip(past, counts)) if n]
                          or [np.zeros((0, s.shape[1]))])


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_single_tokens_with_and_without_cu(device, kv):
    """The decode form, in place and not, is the packed form of one token each; explicit
    positions turn to themselves; a negative length is left alone, its query still turned."""
    announce(f"single tokens {kv}")
    n_seq, hkv, hq, d, page = 6, 2, 8, 128, 16
    g, pk, pv, table, scales = setup(device, 2, n_seq, hkv, page, d, 5, False, BF16 if kv == "bf16" else FP8)
    plan = ia.rotary_plan(d, device=device)
    q, k, v = (torch.randn((n_seq, h, d), device=device, generator=g).bfloat16() for h in (hq, hkv, hkv))
    past = [0, 15, 16, 79, 80, -3]  # 80 is past the table
    seq = torch.tensor(past, device=device, dtype=torch.int32)
    cu = torch.arange(n_seq + 1, device=device, dtype=torch.int32)
    results = []
    for form in range(4):
        a, b = pk.clone(), pv.clone()
        sc = None if scales is None else tuple(s.clone() for s in scales)
        lens = seq.clone()
        if form == 0:
            qo, out = ia.rotary_append_kv(q, k, v, plan, a, b, table, lens, cu, scales=sc)
            assert lens.tolist() == past
        elif form == 1:
            qo, out = ia.rotary_append_kv(q, k, v, plan, a, b, table, lens, scales=sc)
            assert out is lens
        elif form == 2:
            qo, out = ia.rotary_append_kv(q, k, v, plan, a, b, table, lens, scales=sc, new_seq_lens=torch.empty_like(lens))
            assert lens.tolist() == past
        else:
            qo, out = ia.rotary_append_kv(q, k, v, plan, a, b, table, lens, scales=sc, positions=seq.clone(),
                                          q_out=torch.empty_like(q))
        torch.cuda.synchronize()
        assert out.tolist() == [1, 16, 17, 80, 80, -3]
        results.append((qo, a.view(torch.uint8), b.view(torch.uint8), *(sc or ())))
    want_q, _ = ia.apply_rotary(q, None, seq, plan)
    for r in results:
        assert torch.equal(r[0], want_q)
        assert all(torch.equal(x, y) for x, y in zip(r, results[0]))


@pytest.mark.parametrize("kv,dtype", [("bf16", BF16), ("f32", F32), ("fp8", BF16), ("fp8", F32)],
                         ids=["bf16", "f32", "fp8-bf16", "fp8-f32"])
@pytest.mark.parametrize("d,page,rot,layout,hq,hkv,paired", [
    (128, 16, 128, "half", 128, 8, False),         # more rows than a workgroup has places for
    (64, 32, 32, "interleaved", 32, 32, True),
    (128, 16, 70, "half", 12, 4, True),            # a pair a lane
    (64, 48, 10, "half", 5, 1, False),
    (64, 256, 0, "half", 40, 8, False),
    (128, 64, 96, "interleaved", 0, 2, False),     # no queries
])
def test_single_tokens_of_many_heads(device, kv, dtype, d, page, rot, layout, hq, hkv, paired):
    """The form for single tokens writes what the packed form does, bit for bit: scales that stay
    and that rise, pages that begin, end and are missing, explicit positions."""
    announce(f"single tokens of many heads {kv} {dtype} {d} {page} {rot} {layout} {hq}+{hkv}")
    past = [0, 3, page - 1, page, 2 * page - 1, 2 * page, -1, 7, 2 * page + 9, page + 2]
    n = len(past)
    g, pk, pv, table, scales = setup(device, rot + hq, n, hkv, page, d, 3, paired,
                                     {"bf16": BF16, "f32": F32, "fp8": FP8}[kv])
    table[7, 0] = -1
    mag = torch.exp2(torch.randint(-6, 8, (n, hq + 2 * hkv, 1), device=device, generator=g).float())
    buf = (torch.randn((n, hq + 2 * hkv, d), device=device, generator=g) * mag).to(dtype)
    buf[5, hq, 3], buf[9, hq + hkv, d - 1] = float("inf"), float("nan")
    q, k, v = buf.split([hq, hkv, hkv], 1)
    plan = ia.rotary_plan(rot, base=300.0, layout=layout, factor=0.75, device=device)
    cu = torch.arange(n + 1, device=device, dtype=torch.int32)
    where = torch.randint(-5, 9000, (n,), device=device, generator=g, dtype=torch.int32)
    for positions in (None, where):
        results = []
        for form in range(3):
            a, b = pk.clone(), pv.clone()
            sc = None if scales is None else tuple(s.clone() for s in scales)
            lens = torch.tensor(past, device=device, dtype=torch.int32)
            out = None if not hq else torch.empty_like(q) if form < 2 else buf.clone()[:, :hq]
            qo, new = ia.rotary_append_kv(q if hq else None, k, v, plan, a, b, table, lens, cu if form == 0 else None,
                                          positions=positions, scales=sc, q_out=out,
                                          new_seq_lens=torch.empty_like(lens) if form == 1 else None)
            torch.cuda.synchronize()
            assert (new is lens) == (form == 2)
            assert new.tolist() == [p + (p >= 0 and i != 7) for i, p in enumerate(past)]
            results.append((new, a.view(torch.uint8), b.view(torch.uint8), *(sc or ()), *([qo.contiguous().view(torch.uint8)] if hq else [])))
        assert any(not torch.equal(x, y) for x, y in zip(results[0][1:], (pk.view(torch.uint8),)))
        for r in results[1:]:
            assert all(torch.equal(x, y) for x, y in zip(r, results[0]))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_sequences_without_new_rows(device, kv):
    """A begun page of a sequence that gets no rows keeps its codes and its scale, whatever the
    rows before and behind its place in the batch are; a batch of no rows at all."""
    announce(f"write, sequences without rows {kv}")
    hkv, d, page = 2, 64, 16
    past, counts = [5, 0, 8, 16, 3], [0, 3, 0, 2, 0]
    g, pk, pv, table, scales = setup(device, 9, 5, hkv, page, d, 2, False, FP8 if kv == "fp8" else BF16)
    if scales:
        for s in scales:
            s.fill_(2.0 ** -6)
    total = sum(counts)
    k, v, q = (torch.full((total + 1, hkv, d), 1e4, device=device, dtype=BF16)[1:] for _ in "kvq")
    seq = torch.tensor(past, device=device, dtype=torch.int32)
    idle = [b for b, n in enumerate(counts) if n == 0]
    mine = table[idle].flatten().long()
    state = [pk.view(torch.uint8), pv.view(torch.uint8), *(scales or ())]
    before = [x.clone() for x in state]
    plan = ia.rotary_plan(d, device=device)
    _, lens = ia.rotary_append_kv(q, k, v, plan, pk, pv, table, seq, cu_of(counts, device), scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == [a + b for a, b in zip(past, counts)]
    assert all(torch.equal(x[mine], y[mine]) for x, y in zip(state, before))
    before = [x.clone() for x in state]
    _, lens = ia.rotary_append_kv(q[:0], k[:0], v[:0], plan, pk, pv, table, seq, cu_of([0] * 5, device), scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == past and all(torch.equal(x, y) for x, y in zip(state, before))


def test_missing_pages(device):
    """A position without a page is skipped, the length counts up to the first of them, and
    queries are turned all the same."""
    announce("8-bit write, missing pages")
    hkv, d, page = 1, 64, 16
    g, pk, pv, table, scales = setup(device, 3, 3, hkv, page, d, 4)
    table[0, 1], table[1, 0], table[2, 2] = -1, 10 ** 6, -7
    past, counts = [5, 0, 20], [40, 10, 44]
    total = sum(counts)
    k, v, q = (torch.randn((total, hkv, d), device=device, generator=g) for _ in "kvq")
    plan = ia.rotary_plan(0, device=device)
    before = [(codes(p).copy(), s.cpu().numpy().copy()) for p, s in zip((pk, pv), scales)]
    qo, lens = ia.rotary_append_kv(q, k, v, plan, pk, pv, table, torch.tensor(past, device=device, dtype=torch.int32),
                                   cu_of(counts, device), scales=scales)
    torch.cuda.synchronize()
    assert lens.tolist() == [16, 0, 32] and torch.equal(qo, q)
    check_fp8(pk, pv, scales, before, table, past, counts, k, v, page)


def test_identity_table(device):
    announce("write, no table")
    pk, pv = torch.zeros((4, 1, 16, 64), device=device), torch.zeros((4, 1, 16, 64), device=device)
    rows = torch.randn((30, 1, 64), device=device)
    seq = torch.tensor([10], device=device, dtype=torch.int32)
    _, lens = ia.rotary_append_kv(None, rows, -rows, None, pk, pv, None, seq, cu_of([30], device))
    k, v = ia.read_kv(pk, pv, None, seq, cu_of([30], device), 30)
    torch.cuda.synchronize()
    assert lens.tolist() == [40] and torch.equal(k, rows) and torch.equal(v, -rows)


def test_captured_decode_step(device):
    """A captured write of single tokens, lengths in place, replayed with the program's own
    work between: every replay as the eager call on a copy."""
    announce("8-bit write, captured")
    n_seq, hkv, hq, d, page = 4, 2, 4, 64, 16
    g, pk, pv, table, scales = setup(device, 6, n_seq, hkv, page, d, 3)
    plan = ia.rotary_plan(d, device=device)
    q, k, v = (torch.randn((n_seq, h, d), device=device, generator=g).bfloat16() for h in (hq, hkv, hkv))
    seq, qo = torch.tensor([0, 3, 15, 16], device=device, dtype=torch.int32), torch.empty_like(q)
    start = seq.clone()
    ia.rotary_append_kv(q, k, v, plan, pk, pv, table, seq, scales=scales, q_out=qo)
    torch.cuda.synchronize()
    seq.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ia.rotary_append_kv(q, k, v, plan, pk, pv, table, seq, scales=scales, q_out=qo)
    for step in range(6):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=device, generator=g) * 2.0 ** (step % 3))
        a, b, sc, lens = pk.clone(), pv.clone(), tuple(s.clone() for s in scales), seq.clone()
        want, _ = ia.rotary_append_kv(q, k, v, plan, a, b, table, lens, scales=sc)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(seq, lens) and torch.equal(qo, want)
        assert torch.equal(a.view(torch.uint8), pk.view(torch.uint8))
        assert torch.equal(b.view(torch.uint8), pv.view(torch.uint8))
        assert all(torch.equal(x, y) for x, y in zip(sc, scales))


# ------------------------------------------------------------------ reading back

@pytest.mark.parametrize("kv", ["bf16", "f32", "fp8"])
@pytest.mark.parametrize("out", [BF16, F32], ids=["to-bf16", "to-f32"])
@pytest.mark.parametrize("d,page,hkv,paired", [(128, 16, 8, True), (64, 32, 3, False)])
def test_read_back(device, kv, out, d, page, hkv, paired):
    announce(f"read {kv} {out} {d} {page}")
    pool_t = {"bf16": BF16, "f32": F32, "fp8": FP8}[kv]
    g, pk, pv, table, scales = setup(device, d, 4, hkv, page, d, 6, paired, pool_t)
    if scales:
        for s in scales:
            s.mul_(1 + torch.rand(s.shape, device=device, generator=g))
        pk.view(torch.uint8)[table[0, 0].long(), 0, 0, 0] = 0x7F  # a NaN code stays one
    table[2, 1] = -1
    starts, counts = [0, 7, page - 3, -2], [page * 6 + 5, 0, 2 * page, 5]
    total = sum(counts)
    given = [torch.full((total + 3, hkv, d), 9.0, device=device, dtype=out) for _ in "kv"]
    got = ia.read_kv(pk, pv, table, torch.tensor(starts, device=device, dtype=torch.int32), cu_of(counts, device),
                     total + 3, scales=scales, out_dtype=out, k_out=given[0], v_out=given[1])
    torch.cuda.synchronize()
    t = table.cpu()
    for x, pool, i in ((got[0], pk, 0), (got[1], pv, 1)):
        x, p = x.cpu(), pool.cpu().float()
        if scales:
            p = p * scales[i].cpu()[:, :, None, None]
        at = 0
        for b, (s, n) in enumerate(zip(starts, counts)):
            for j in range(n):
                pos = s + j
                pg = int(t[b, pos // page]) if 0 <= pos < 6 * page else -1
                want = p[pg, :, pos % page].to(out) if pg >= 0 else torch.zeros((hkv, d), dtype=out)
                assert torch.equal(torch.nan_to_num(x[at + j], nan=5.0), torch.nan_to_num(want, nan=5.0)), (b, j)
            at += n
        assert bool((x[total:] == 9).all())


def test_write_and_read_refusals(device):
    g, pk, pv, table, scales = setup(device, 0, 2, 2, 16, 64, 3)
    plan = ia.rotary_plan(64, device=device)
    rows = torch.zeros((2, 2, 64), device=device)
    q = torch.zeros((2, 4, 64), device=device)
    seq, cu = torch.zeros(2, device=device, dtype=torch.int32), torch.arange(3, device=device, dtype=torch.int32)
    f32 = torch.zeros((7, 2, 16, 64), device=device)
    seq3 = ia.sequence_scales(scales, table)
    bad = [
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu),  # no scales
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu, scales=(*scales, seq3)),
        lambda: ia.rotary_append_kv(q, rows.half(), rows.half(), plan, pk, pv, table, seq, cu, scales=scales),
        lambda: ia.rotary_append_kv(q, rows, rows.bfloat16(), plan, pk, pv, table, seq, cu, scales=scales),
        lambda: ia.rotary_append_kv(q.bfloat16(), rows, rows, plan, pk, pv, table, seq, cu, scales=scales),
        lambda: ia.rotary_append_kv(q[:, :3], rows, rows, plan, pk, pv, table, seq, cu, scales=scales),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu[:2], scales=scales),
        lambda: ia.rotary_append_kv(q[:1], rows[:1], rows[:1], plan, pk, pv, table, seq, scales=scales),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu, scales=scales, new_seq_lens=seq),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu, scales=scales, positions=seq[:1]),
        lambda: ia.rotary_append_kv(None, rows, rows, plan, pk, pv, table, seq, cu, scales=scales, q_out=q),
        lambda: ia.rotary_append_kv(q, rows, rows, ia.rotary_plan(128, device=device), pk, pv, table, seq, cu, scales=scales),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, scales=scales, positions=seq),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu, scales=scales, positions=cu[1:], new_seq_lens=cu[1:]),
        lambda: ia.rotary_append_kv(q, rows, rows, plan, pk, pv, table, seq, cu, scales=scales, q_out=q[:1].expand(2, 4, 64)),
        lambda: ia.read_kv(pk, pv, table, seq, cu, 1 << 31, scales=scales),
        lambda: ia.append_prompt_kv(f32, f32, table, seq, rows, rows, cu, scales=scales),
        lambda: ia.append_kv(f32, f32, table, seq, rows, rows, scales=scales),
        lambda: ia.append_prompt_kv(pk, pv, table, seq, rows, rows, cu),
        lambda: ia.read_kv(pk, pv, table, seq, cu, 2),
        lambda: ia.read_kv(pk, pv, table, seq, cu, -1, scales=scales),
        lambda: ia.read_kv(pk, pv, table, seq, cu, 2, scales=scales, out_dtype=torch.half),
        lambda: ia.read_kv(pk, pv, table, seq, cu, 2, scales=scales, k_out=rows.bfloat16()[:1]),
        lambda: ia.read_kv(pk, pv, table, seq[:1], cu, 2, scales=scales),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    # nothing to do
    lens = ia.append_prompt_kv(pk, pv, table[:0], seq[:0], rows[:0], rows[:0], cu[:1], scales=scales)
    assert lens.shape == (0,)
    k, v = ia.read_kv(pk, pv, table[:0], seq[:0], cu[:1], 0, scales=scales)
    assert k.shape == (0, 2, 64) and k.dtype == BF16
