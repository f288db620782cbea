"""V that is not finite: a row has what the tokens it sees give it, +inf, -inf or NaN in their
channels and finite values in the others, whatever the tokens hidden from it hold.  Bars:
those of the prompt attention tests."""

import math

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, packed, paged, reference
from tests.test_gpu_prompt_edges import i32

pytestmark = pytest.mark.gpu


def check_values(got, want, mag, kv, keys, what):
    """``check`` where ``want`` is finite, the same infinity or NaN elsewhere."""
    g, odd = got.detach().cpu(), ~torch.isfinite(want)
    assert bool(odd.any()), what
    same = (g.double() == want) | (torch.isnan(g) & torch.isnan(want))
    assert bool(same[odd].all()), (what, int((~same[odd]).sum()))
    check(torch.where(odd, torch.zeros_like(g), g), want.masked_fill(odd, 0), mag.masked_fill(odd, 0), kv, keys, what)


# query heads, kv heads (tiles of 128 rows, but of 32 for the float32 group of 4)
SHAPES = [("bf16", 128, 64, 1), ("bf16", 64, 40, 1), ("f32", 64, 64, 1), ("f32", 128, 40, 1), ("bf16", 128, 4, 1),
          ("bf16", 64, 8, 2), ("f32", 128, 4, 1)]


@pytest.mark.parametrize("kv,d,hq,hkv", SHAPES)
def test_seen_infinities_and_hidden_ones(kv, d, hq, hkv, device):
    """Every row past token 5 sees an infinity in channel 3; tokens 100 on bring NaN and the
    other infinity into channel 9, and into channel 3 itself."""
    announce(f"seen and hidden {kv} {d} {hq}x{hkv}")
    n = 106
    q, k, v, cu = packed(device, [n, 4], hq, hkv, d, kv, False, d)
    v = v.clone()
    v[5, 0, 3] = math.inf
    v[100, 0, 9], v[101, 0, 9], v[101, 0, 3] = math.inf, math.nan, -math.inf
    v[102, -1, 11], v[103, -1, 11] = -math.inf, -math.inf
    out = ia.prompt_attention(q, k, v, cu, workspace={})
    torch.cuda.synchronize()
    want, mag = reference(q[:n], k[:n], v[:n], 0, d ** -0.5)
    assert float(want[100, 0, 3]) == math.inf and math.isnan(float(want[101, 0, 3]))
    assert bool(torch.isfinite(want[:100, :, 9]).all()) and bool(torch.isfinite(out[n:]).all())
    check_values(out[:n], want, mag, kv, n, (kv, d))


@pytest.mark.parametrize("hq", [64, 8])
def test_fp8_codes_and_page_scales(hq, device):
    """fp8: a NaN code that is seen, one that is hidden, and pages whose scales are not
    finite (K's: the scores of its tokens; V's: their values) behind some of the rows."""
    announce(f"fp8 seen and hidden, {hq} heads")
    hkv, d, page, total, new = 1, 64, 16, 150, 12
    pk, pv, scales, table = paged(device, [total], hkv, d, page, "fp8", "split", 7)
    nan = torch.tensor([0x7f], device=device, dtype=torch.uint8)
    raw = pv.view(torch.uint8)
    raw[int(table[0, 0]), 0, 2, 3] = nan
    raw[int(table[0, 8]), 0, 141 % page, 9] = nan
    scales[1][int(table[0, 9]), 0] = math.nan  # tokens 144..149
    q = torch.randn((new, hq, d), device=device).to(torch.bfloat16)
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, [total]), i32(device, [0, new]), scales=scales,
                                    workspace={})
    torch.cuda.synchronize()
    k, v = gather(pk, scales[0], table[0], total), gather(pv, scales[1], table[0], total)
    want, mag = reference(q, k, v, total - new, d ** -0.5)
    seen = 144 - (total - new)  # rows before see none of the page with the NaN scale
    assert bool(torch.isfinite(want[:3, :, 9]).all()) and bool(torch.isnan(want[seen:]).all())
    assert bool(torch.isnan(out[seen:]).all())
    check_values(out[:seen], want[:seen], mag[:seen], "fp8", total, hq)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_prefix_members_that_end_before_it(kv, device):
    """Ten members of eight query heads; the first tokens hold an infinity that all see, the
    last ones a NaN that the shorter members do not."""
    announce(f"prefix seen and hidden {kv}")
    hkv, hq, d, page, shared = 1, 8, 64, 16, 200
    lens = [230, 210, 199, 150, 201, 64, 230, 190, 200, 63]
    pk, pv, _, table = paged(device, [230] * 10, hkv, d, page, kv, "split", 13)
    for i in range(1, 10):
        table[i, :12] = table[0, :12]
        for pool in (pk, pv):  # (the page that the prefix ends in)
            pool[int(table[i, 12]), :, :8] = pool[int(table[0, 12]), :, :8].clone()
    pv[int(table[0, 0]), 0, 1, 5] = -math.inf
    pv[int(table[0, 11]), 0, 191 % page, 6] = math.nan
    pv[int(table[0, 11]), 0, 189 % page, 5] = math.inf
    q = torch.randn((10, hq, d), device=device).to(DT[kv])
    out = ia.shared_prefix_decode(q, pk, pv, table, i32(device, lens), i32(device, [0, 10]), i32(device, [shared]),
                                  workspace={})
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        want, mag = reference(q[b:b + 1], gather(pk, None, table[b], n), gather(pv, None, table[b], n), n - 1, d ** -0.5)
        check_values(out[b:b + 1], want, mag, kv, n, (kv, b))
