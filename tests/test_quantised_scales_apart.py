"""Keys and values of a write have pools and scales of their own: one tensor for both would be
written by the waves of both."""

import pytest
import torch

import interattn_amd as ia
from interattn_amd import _native as N
from tests._util import announce

P = 1 << 32  # an aligned address that nothing follows
D, HKV, PAGES = 128, 2, 9


def write(single, k_scale, v_scale, stride, v_pool=P + (1 << 31), dtype=N.IA_FP8_E4M3):
    kv = N.PagedKV(P + (1 << 30), v_pool, dtype, 16, PAGES, HKV * 16 * D, 16 * D, D, HKV * 16 * D, 16 * D, D, P - 4096, 4, 4)
    if dtype == N.IA_FP8_E4M3:
        kv.k_scale, kv.v_scale, kv.scale_page_stride = k_scale, v_scale, stride
    rows = N.PackedKV(P + (1 << 28), P + (1 << 29), N.IA_BF16, HKV * D, D, HKV * D, D)
    return N.lib().ia_rotary_append_kv(None, None, rows, kv, None if single else P, P + 4096, P + 8192, None, 5,
                                       5 if single else 40, HKV, D, None)


def refused(rc, text):
    msg = N.lib().ia_last_error().decode()
    assert rc == N.IA_ERR_INVALID and text in msg, (rc, msg)


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("k_scale,v_scale,stride", [
    (P, P, HKV), (P, P + 4, 2 * HKV), (P + 4, P, HKV), (P, P + 4 * HKV, HKV), (P + 4 * HKV * (PAGES - 1), P, HKV),
])
def test_shared_scales(single, k_scale, v_scale, stride):
    refused(write(single, k_scale, v_scale, stride), "k_scale and v_scale")


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("dtype", [N.IA_FP8_E4M3, N.IA_BF16])
def test_one_pool_for_both(single, dtype):
    refused(write(single, P, P + (1 << 20), HKV, P + (1 << 30), dtype), "pools")


@pytest.mark.gpu
@pytest.mark.parametrize("single", [False, True])
def test_scales_side_by_side(device, single):
    """Views of one ``[n_pages, 2, Hkv]`` tensor, and of ``[2, n_pages, Hkv]``, as two tensors."""
    announce(f"fp8 scales side by side {single}")
    g = torch.Generator(device=device)
    g.manual_seed(1)
    k, v = (torch.randn((5, HKV, D), device=device, generator=g).mul_(m).bfloat16() for m in (1.0, 30.0))
    table = torch.randperm(PAGES, device=device)[:5].view(5, 1).to(torch.int32)
    cu = None if single else torch.arange(6, device=device, dtype=torch.int32)
    lens = torch.arange(5, device=device, dtype=torch.int32)
    got = []
    for scales in (torch.ones((2, PAGES, HKV), device=device), torch.ones((PAGES, 2, HKV), device=device).transpose(0, 1),
                   (torch.ones((PAGES, HKV), device=device), torch.ones((PAGES, HKV), device=device))):
        pools = [torch.zeros((PAGES, HKV, 16, D), device=device).to(torch.float8_e4m3fn) for _ in "kv"]
        _, after = ia.rotary_append_kv(None, k, v, None, *pools, table, lens.clone(), cu, scales=(scales[0], scales[1]))
        torch.cuda.synchronize()
        got.append([after, *(x.view(torch.uint8) for x in pools), scales[0], scales[1]])
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    assert not torch.equal(got[0][3], got[0][4])
