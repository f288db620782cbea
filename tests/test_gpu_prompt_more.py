"""Forms of the prompt and page calls that the other tests leave out: cut keys with values
that are not finite, single tokens beside ``paged_decode``, more page tensors than one launch
takes."""

import math

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, paged, reference
from tests.test_gpu_prompt_edges import i32
from tests.test_gpu_prompt_hidden import check_values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,hq", [("bf16", 64), ("bf16", 8), ("f32", 64), ("f32", 8)])
def test_cut_keys_with_seen_and_hidden_values(kv, hq, device):
    """Three new tokens over 2,600 keys, which are cut: an infinity that all rows see in the
    first piece, a NaN in the last that only the last row sees."""
    announce(f"cut keys, seen and hidden {kv} {hq}")
    hkv, d, page, total, new = 1, 128, 32, 2600, 3
    pk, pv, _, table = paged(device, [total], hkv, d, page, kv, "split", 5)
    at = lambda t: (int(table[0, t // page]), 0, t % page)  # noqa: E731
    pv[(*at(70), 4)], pv[(*at(total - 1), 9)], pv[(*at(total - 1), 4)] = math.inf, math.nan, -math.inf
    q = torch.randn((new, hq, d), device=device).to(DT[kv])
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, [total]), i32(device, [0, new]), workspace={})
    torch.cuda.synchronize()
    want, mag = reference(q, gather(pk, None, table[0], total), gather(pv, None, table[0], total), total - new, d ** -0.5)
    assert bool((want[:2, :, 4] == math.inf).all()) and bool(torch.isfinite(want[:2, :, 9]).all())
    check_values(out, want, mag, kv, total, kv)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_cut_keys_with_a_missing_page_at_any_scale(scale, kv, device):
    announce(f"cut keys, missing page, scale {scale} {kv}")
    hq, hkv, d, page, total, new = 64, 1, 64, 16, 2100, 2
    pk, pv, _, table = paged(device, [total], hkv, d, page, kv, "split", 6)
    k, v = gather(pk, None, table[0], total), gather(pv, None, table[0], total)
    keep = torch.tensor([not (160 <= t < 176 or 2064 <= t < 2080) for t in range(total)], device=k.device)
    table[0, 10], table[0, 129] = -1, pk.shape[0]
    q = torch.randn((new, hq, d), device=device).to(DT[kv])
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, [total]), i32(device, [0, new]), scale=scale,
                                    workspace={})
    torch.cuda.synchronize()
    n = int(keep.sum())
    want, mag = reference(q, k[keep], v[keep], n - new, scale)
    check(out, want, mag, kv, n, (scale, kv))


@pytest.mark.parametrize("kv", ["bf16", "f32", "fp8"])
def test_single_tokens_beside_the_dense_decode(kv, device):
    """New lengths of one are a decode step.  Each side is within its bar of the float64
    result, so they are within the sum of both of each other."""
    announce(f"single tokens beside paged_decode {kv}")
    hkv, hq, d, page = 2, 8, 128, 16
    lens = [1, 16, 700, 333, 64, 65]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, "paired", 6)
    q = torch.randn((len(lens), hq, d), device=device).to(DT["f32" if kv == "f32" else "bf16"])
    seq = i32(device, lens)
    one = ia.paged_prompt_attention(q, pk, pv, table, seq, i32(device, list(range(len(lens) + 1))), scales=scales,
                                    workspace={})
    dense = ia.paged_decode(q, pk, pv, table, seq, max_seq_len=max(lens), scales=scales, workspace={})
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        k, v = gather(pk, scales and scales[0], table[b], n), gather(pv, scales and scales[1], table[b], n)
        want, mag = reference(q[b:b + 1], k, v, n - 1, d ** -0.5)
        check(one[b:b + 1], want, mag, kv, n, ("prompt", b))
        check(dense[b:b + 1], want, mag, kv, n, ("decode", b))


def test_page_calls_over_sixty_tensors(device):
    """A model of 30 layers: more tensors than one launch takes, in every call that moves pages."""
    announce("sixty page tensors")
    page, n_pages, rows = 16, 40, 5
    gen = torch.Generator(device=device)
    gen.manual_seed(1)
    pools = [torch.randn((n_pages, 2, page, 8), device=device, generator=gen) for _ in range(60)]
    host = [p.cpu().clone() for p in pools]
    table = torch.full((rows, 8), -1, dtype=torch.int32)
    table[0, :4] = torch.tensor([30, 7, 22, 39])  # 55 tokens: three whole pages and a part
    table[4, :2] = torch.tensor([35, 3])
    lens = torch.tensor([55, 0, 0, 0, 20], dtype=torch.int32)
    refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)
    table, lens, refs = table.to(device), lens.to(device), refs.to(device)
    ok = ia.fork_sequences(pools, table, lens, refs, i32(device, [0, 0, 4]), i32(device, [1, 2, 3]), page_size=page,
                           workspace={})
    torch.cuda.synchronize()
    assert ok.tolist() == [1, 1, 1] and lens.tolist() == [55, 55, 55, 20, 20]
    assert table[1].tolist() == [30, 7, 22, 0, -1, -1, -1, -1] and table[2, :4].tolist() == [30, 7, 22, 1]
    assert table[3, :2].tolist() == [35, 2]
    for p, h in zip(pools, host):
        h[0], h[1], h[2] = h[39], h[39], h[3]
        assert torch.equal(p.cpu(), h)
    ia.copy_pages(pools, i32(device, [7, 35]), i32(device, [20, 21]))
    torch.cuda.synchronize()
    for p, h in zip(pools, host):
        h[20], h[21] = h[7], h[35]
        assert torch.equal(p.cpu(), h)
    # held: 0 1 2 3 7 22 30 35 39, so 22 30 35 39 move to 4 5 6 8
    before = [h[table.cpu().clamp_min(0).long()] for h in host]
    assert ia.compact_pages(pools, table, refs, workspace={}).tolist() == [9]
    torch.cuda.synchronize()
    assert table[0, :4].tolist() == [5, 7, 4, 8] and table[4, :2].tolist() == [6, 3]
    assert refs[:9].tolist() == [1, 1, 1, 1, 3, 3, 2, 3, 1] and not bool(refs[9:].any())
    held = (table >= 0).cpu()
    for p, b in zip(pools, before):
        assert torch.equal(p.cpu()[table.cpu().clamp_min(0).long()][held], b[held])
