"""The paged runner's prefill on the prompt calls: what it leaves to SDPA, what it refuses."""

from types import SimpleNamespace

import pytest
import torch

from interattn_amd.decode import PagedTopkDecodeRunner
from tests._util import announce

pytestmark = pytest.mark.gpu

B, HQ, HKV, D = 2, 4, 2, 64


def runner(device, native):
    layer = SimpleNamespace(self_attn=SimpleNamespace())
    model = SimpleNamespace(
        config=SimpleNamespace(num_hidden_layers=1, num_key_value_heads=HKV, num_attention_heads=HQ, head_dim=D,
                               hidden_size=HQ * D),
        parameters=lambda: iter([torch.zeros(1, device=device)]), model=SimpleNamespace(layers=[layer]))
    r = PagedTopkDecodeRunner(model=model, batch_size=B, max_seq_len=64, block_size=16, k=4, full_attention_layers=1,
                              native_prompt=native)
    return r, SimpleNamespace(layer_idx=0, training=False)


def inputs(device, t, grad):
    gen = torch.Generator(device=device)
    gen.manual_seed(t)
    return [torch.randn((B, h, t, D), device=device, generator=gen).requires_grad_(grad) for h in (HQ, HKV, HKV)]


def test_prefill_keeps_gradients(device):
    """Gradients of a weighted sum of the output against the formula's in 64 bits.  float32
    products and sums over 64 channels and 21 keys of values of order one: the bar is 2^-24
    for each of the 4 * (64 + 21) roundings on the way, with a factor 8 for the values' size."""
    announce("runner, gradients")
    t, scale = 21, D ** -0.5
    r, module = runner(device, True)
    q, k, v = inputs(device, t, True)
    out, _ = r.hybrid_attention_forward(module, q, k, v, None, scale)
    assert out.requires_grad and out.shape == (B, t, HQ, D)
    w = torch.randn(out.shape, device=device)
    got = torch.autograd.grad((out * w).sum(), (q, k, v))
    q64, k64, v64 = (x.detach().cpu().double().requires_grad_(True) for x in (q, k, v))
    kk, vv = (x.repeat_interleave(HQ // HKV, 1) for x in (k64, v64))
    s = (q64 @ kk.transpose(2, 3) * scale).masked_fill(torch.ones(t, t).triu(1).bool(), -torch.inf)
    want_out = (torch.softmax(s, -1) @ vv).transpose(1, 2)
    want = torch.autograd.grad((want_out * w.cpu().double()).sum(), (q64, k64, v64))
    torch.cuda.synchronize()
    for a, b in zip((out, *got), (want_out, *want)):
        bar = 8 * 4 * (64 + 21) * 2.0 ** -24 * max(1.0, float(b.detach().abs().max()))
        assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= bar
    assert r.seq_lens[0].tolist() == [t] * B


def test_without_gradients_both_prefills_agree(device):
    """The pools hold the same rows; the outputs are both within the bar above."""
    announce("runner, both prefills")
    t, scale = 33, D ** -0.5
    outs, pools = [], []
    for native in (False, True):
        r, module = runner(device, native)
        q, k, v = inputs(device, t, False)
        out, _ = r.hybrid_attention_forward(module, q, k, v, None, scale)
        torch.cuda.synchronize()
        outs.append(out.cpu().double())
        pools.append([p.detach()[r.block_table[:, :3].long()].cpu()[:, :, :, :, :] for p in r.pools[0]])
        assert r.seq_lens[0].tolist() == [t] * B and not out.requires_grad
    bar = 2 * 8 * 4 * (64 + 33) * 2.0 ** -24 * max(1.0, float(outs[0].abs().max()))
    assert float((outs[0] - outs[1]).abs().max()) <= bar
    for a, b in zip(*pools):
        a, b = (x.permute(0, 1, 3, 2, 4).reshape(B, -1, HKV, D)[:, :t] for x in (a, b))
        assert torch.equal(a, b)


def test_native_prefill_refuses_a_chunk(device):
    """Keys of cached tokens besides the new ones: refused before anything is written."""
    announce("runner, chunk")
    r, module = runner(device, True)
    q, k, v = inputs(device, 20, False)
    before = [p.clone() for p in r.pools[0]]
    with pytest.raises(ValueError, match="whole prompts"):
        r.hybrid_attention_forward(module, q[:, :, 12:], k, v, None, D ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, r.pools[0])) and r.seq_lens[0].tolist() == [0] * B
