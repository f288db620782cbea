"""Tiles of 128 rows at their edges: scales of zero, scores past 2^31, values that are not
finite.  Bars: those of the prompt attention tests."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, packed, paged, reference
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


def far_scores(device, n, hq, d, kv, top, negative):
    """q and k whose scores of token j are ``+-64 * 2^top * b[j]`` exactly, b distinct bf16
    values in [1, 2): neighbours differ by 2^(top - 1) or more, so that a row's softmax is
    one at its largest score and zero elsewhere to any precision."""
    q = torch.zeros((n, hq, d), device=device, dtype=DT[kv])
    q[..., :64] = 2.0 ** (top // 2)
    order = torch.randperm(128, generator=torch.Generator().manual_seed(top))[:n]
    b = (1 + order.float() / 128).to(device)
    k = torch.zeros((n, 1, d), device=device, dtype=DT[kv])
    k[..., :64] = (b * 2.0 ** (top - top // 2) * (-1 if negative else 1))[:, None, None].to(DT[kv])
    best = [max(range(i + 1), key=lambda j: -int(order[j]) if negative else int(order[j])) for i in range(n)]
    return q, k, best


@pytest.mark.parametrize("negative", [False, True])
@pytest.mark.parametrize("top", [11, 28, 60])
@pytest.mark.parametrize("kv,d,hq", [("bf16", 128, 64), ("bf16", 64, 40), ("f32", 64, 64), ("bf16", 128, 4)])
def test_scores_far_out(kv, d, hq, top, negative, device):
    """Finite scores from 2^17 to 2^67 in size: every row is the value at its largest score.
    ``scale`` 1: log2 units are 1.44 times the scores, gaps at least 2^10."""
    announce(f"far scores {kv} {d} {hq} 2^{top} {negative}")
    n = 100
    q, k, best = far_scores(device, n, hq, d, kv, top, negative)
    v = torch.randn((n, 1, d), device=device).to(DT[kv])
    cu = i32(device, [0, n])
    out = ia.prompt_attention(q, k, v, cu, scale=1.0)
    torch.cuda.synchronize()
    assert torch.equal(out, v[best].expand(n, hq, d))


def test_far_scores_in_pages_and_prefixes(device):
    """The same through the pool: a single token of 64 heads, and a group of nine sequences."""
    announce("far scores, pages")
    n, d, page = 100, 128, 16
    q, k, best = far_scores(device, n, 64, d, "bf16", 40, False)
    v = torch.randn((n, 1, d), device=device).to(torch.bfloat16)
    pk, pv = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 12)).view(7, page, 1, d).transpose(1, 2) for x in (k, v))
    table = torch.arange(7, device=device, dtype=torch.int32)[None]
    out = ia.paged_prompt_attention(q[:1], pk, pv, table, i32(device, [n]), i32(device, [0, 1]), scale=1.0, workspace={})
    lens = [100, 97, 100, 98, 100, 99, 100, 100, 97]
    many = ia.shared_prefix_decode(q[:9, :8], pk, pv, table.expand(9, 7).contiguous(), i32(device, lens),
                                   i32(device, [0, 9]), i32(device, [97]), scale=1.0, workspace={})
    torch.cuda.synchronize()
    assert torch.equal(out[0], v[best[n - 1]].expand(64, d))
    for b, m in enumerate(lens):
        assert torch.equal(many[b], v[best[m - 1]].expand(8, d)), b


@pytest.mark.parametrize("low", [-1, -2 ** 31])
def test_negative_lengths_leave_the_other_members_alone(low, device):
    announce(f"negative length {low}")
    hkv, hq, d, page, shared = 1, 8, 64, 16, 96
    lens = [120, low, 110, 101, 97, low, 100, 120, 99]
    pk, pv, _, table = paged(device, [120] * 9, hkv, d, page, "bf16", "split", 13)
    table[:, :6] = table[0, :6].clone()
    q = torch.randn((9, hq, d), device=device).to(torch.bfloat16)
    out = ia.shared_prefix_decode(q, pk, pv, table, i32(device, lens), i32(device, [0, 9]), i32(device, [shared]),
                                  workspace={})
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        if n < 0:
            assert bool((out[b] == 0).all())
            continue
        want, mag = reference(q[b:b + 1], gather(pk, None, table[b], n), gather(pv, None, table[b], n), n - 1, d ** -0.5)
        check(out[b:b + 1], want, mag, "bf16", n, b)
