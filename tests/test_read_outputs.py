"""Rows read back go to two outputs that lie apart."""

import pytest
import torch

import interattn_amd as ia
from interattn_amd import _native as N
from tests._util import announce

P = 1 << 32  # an aligned address that nothing follows
D, HKV, TOKENS = 128, 2, 9


@pytest.mark.parametrize("dtype,size", [(N.IA_BF16, 2), (N.IA_F32, 4)])
@pytest.mark.parametrize("rows", [0, 1, -1, TOKENS - 1, 0.5])
def test_outputs_that_meet(dtype, size, rows):
    kv = N.PagedKV(P + (1 << 30), P + (1 << 31), N.IA_BF16, 16, 9, HKV * 16 * D, 16 * D, D, HKV * 16 * D, 16 * D, D,
                   P - 4096, 4, 4)
    rc = N.lib().ia_read_kv(kv, P, P + int(rows * HKV * D * size), dtype, P - 8192, P - 12288, 2, TOKENS, HKV, D, None)
    assert rc == N.IA_ERR_INVALID and "overlap" in N.lib().ia_last_error().decode()


@pytest.mark.gpu
def test_neighbours_in_one_buffer(device):
    announce("read, outputs that are neighbours")
    pool = [torch.randn((4, HKV, 16, D), device=device).bfloat16() for _ in "kv"]
    table = torch.tensor([[3, 1]], device=device, dtype=torch.int32)
    starts = torch.tensor([5], device=device, dtype=torch.int32)
    cu = torch.tensor([0, TOKENS], device=device, dtype=torch.int32)
    out = torch.zeros((2, TOKENS, HKV, D), device=device, dtype=torch.bfloat16)
    want = ia.read_kv(*pool, table, starts, cu, TOKENS)
    ia.read_kv(*pool, table, starts, cu, TOKENS, k_out=out[1], v_out=out[0])
    torch.cuda.synchronize()
    assert torch.equal(out[1], want[0]) and torch.equal(out[0], want[1])
    with pytest.raises(ValueError, match="overlap"):
        ia.read_kv(*pool, table, starts, cu, TOKENS, k_out=out[0], v_out=out[0])
