"""Outputs of the prompt-side attention calls are the caller's: a later call with the same
workspace leaves an earlier result alone, in a captured graph too."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import packed, paged
from tests.test_gpu_prompt_edges import i32

pytestmark = pytest.mark.gpu


def calls(device):
    """(call of n rows in a workspace, name) of each entry point."""
    hq, hkv, d, page = 8, 2, 64, 16
    q, k, v, _ = packed(device, [300], hq, hkv, d, "bf16", False, 3)
    pk, pv, _, table = paged(device, [400] * 8, hkv, d, page, "bf16", "split", 4)
    lens, starts, shared = i32(device, [400] * 8), i32(device, [0, 1]), i32(device, [16])
    cu = {n: i32(device, [0, n]) for n in (5, 7, 8, 100, 300)}
    return {
        "packed": lambda n, ws: ia.prompt_attention(q[:n], k[:n], v[:n], cu[n], workspace=ws),
        "paged": lambda n, ws: ia.paged_prompt_attention(q[:n], pk, pv, table[:1], lens[:1], cu[n], workspace=ws),
        "prefix": lambda n, ws: ia.shared_prefix_decode(q[:n], pk, pv, table[:n], lens[:n], starts, shared, workspace=ws),
    }


@pytest.mark.parametrize("name", ["packed", "paged", "prefix"])
def test_a_later_call_leaves_a_result_alone(name, device):
    announce(f"outputs, {name}")
    call, ws = calls(device)[name], {}
    first = call(8, ws)
    torch.cuda.synchronize()
    kept = first.clone()
    first.add_(1)
    second = call(8, ws)
    torch.cuda.synchronize()
    assert torch.equal(second, kept) and torch.equal(first, kept + 1)


@pytest.mark.parametrize("name", ["packed", "paged", "prefix"])
def test_a_graph_keeps_the_memory_it_writes(name, device):
    """Captured after an eager call of its size; eager calls of other sizes and new tensors
    follow; replays write none of them."""
    announce(f"outputs, {name}, graph")
    call, ws = calls(device)[name], {}
    want = call(8, ws).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph):
            got = call(8, ws)
    torch.cuda.current_stream().wait_stream(side)
    where = got.data_ptr()
    del got
    for _ in range(3):
        others = [call(n, ws) for n in (5, 7)]
        others += [torch.zeros_like(want) for _ in range(64)]
        held = [t.clone() for t in others]
        graph.replay()
        torch.cuda.synchronize()
        for t, h in zip(others, held):
            assert torch.equal(t, h)
            assert not t.data_ptr() <= where < t.data_ptr() + t.numel() * t.element_size()
