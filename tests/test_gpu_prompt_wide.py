"""Tiles of 128 rows at their edges: scales of zero, scores past 2^31, values that are not
finite.  Bars: those of the prompt attention tests."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, packed, paged
from tests.test_gpu_prompt_edges import i32, reference_heads

pytestmark = pytest.mark.gpu

# groups above 32 always take tiles of 128 rows
WIDE = [("bf16", 128), ("bf16", 64), ("f32", 128), ("f32", 64)]


@pytest.mark.parametrize("kv,d", WIDE)
@pytest.mark.parametrize("scale", [0.0, 1e-45])
def test_scale_of_zero_is_the_mean_of_the_visible_values(scale, kv, d, device):
    announce(f"wide, scale {scale} {kv} {d}")
    lens, hq, hkv = [70, 3], 64, 1
    q, k, v, cu = packed(device, lens, hq, hkv, d, kv, True, 8)
    out = ia.prompt_attention(q, k, v, cu, scale=scale)
    torch.cuda.synchronize()
    for at, n in ((0, 70), (70, 3)):
        want, mag = reference_heads(q[at:at + n], k[at:at + n], v[at:at + n], 0, scale)
        check(out[at:at + n], want, mag, kv, n, (scale, at))


@pytest.mark.parametrize("kv", ["bf16", "f32", "fp8"])
def test_scale_of_zero_with_a_missing_page(kv, device):
    """A page that is not there lies before the causal border."""
    announce(f"wide, scale 0, missing page {kv}")
    new, total, hq, hkv, d, page = 9, 150, 64, 1, 64, 16
    pk, pv, scales, table = paged(device, [total], hkv, d, page, kv, "split", 4)
    k, v = gather(pk, scales and scales[0], table[0], total), gather(pv, scales and scales[1], table[0], total)
    keep = torch.tensor([not 32 <= t < 48 for t in range(total)], device=k.device)
    table[0, 2] = -1
    q = torch.randn((new, hq, d), device=device).to(DT["f32" if kv == "f32" else "bf16"])
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, [total]), i32(device, [0, new]), scale=0.0,
                                    scales=scales, workspace={})
    torch.cuda.synchronize()
    want, mag = reference_heads(q, k[keep], v[keep], total - 16 - new, 0.0)
    check(out, want, mag, kv, total, kv)
