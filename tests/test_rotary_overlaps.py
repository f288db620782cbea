"""Outputs of a rotation that share memory with what other workgroups read or write are refused;
views of one buffer whose rows lie apart are not."""

import pytest
import torch

import interattn_amd as ia
from interattn_amd import _native as N
from tests._util import announce

P = 1 << 32  # an aligned address that nothing follows
D, T = 128, 6
WIDE = 48 * D  # a token of 32 query, 8 key and 8 value heads in bf16 elements


def rows(at, heads, tok=WIDE, head=D, out=None, out_tok=None, out_head=None):
    return N.RotaryRows(P + 2 * at, P + 2 * (at if out is None else out), tok, head, tok if out_tok is None else out_tok,
                        head if out_head is None else out_head, heads)


def refused(rc):
    msg = N.lib().ia_last_error().decode()
    assert rc == N.IA_ERR_INVALID and "overlap" in msg, (rc, msg)


def turn(*tensors, tokens=T):
    rot = N.Rotary(P, D, 0, 1.0)
    return N.lib().ia_apply_rotary(rot, (N.RotaryRows * 2)(*tensors), len(tensors), N.IA_BF16, D, P, tokens, 0, None)


FAR = 1 << 24
K = rows(32 * D, 8)

# (the kernel is reached by none of these: two workgroups would write, or one read and one write,
# the same row)
OVERLAPS = {
    "both strides a row": [rows(0, 4, out=FAR, out_tok=D, out_head=D)],
    "tokens within the heads": [rows(0, 4, out=FAR, out_tok=2 * D)],
    "heads within the tokens": [rows(0, 4, out=FAR, out_tok=D, out_head=(T - 1) * D)],
    "expanded": [rows(0, 4, out=FAR, out_tok=0)],
    "a token later": [rows(0, 32, out=WIDE)],
    "a head later": [rows(0, 32, out=D)],
    "half a head later": [rows(0, 4, out=D // 2)],
    "the input by other strides": [rows(0, 4, tok=4 * D, out=0, out_tok=D, out_head=T * D)],
    "one output twice": [rows(0, 32, out=FAR), rows(32 * D, 8, out=FAR)],
    "outputs that meet in a head": [rows(0, 32, out=FAR), rows(32 * D, 8, out=FAR + 31 * D)],
    "q into k": [rows(0, 32, out=8 * D), K],
    "k into q": [rows(0, 32), rows(32 * D, 8, out=31 * D)],
    "k of q, q in place": [rows(0, 32), rows(4 * D, 8, out=FAR)],
    "k and q the same, in place": [rows(0, 8), rows(0, 8)],
}


@pytest.mark.parametrize("name", OVERLAPS)
def test_apply_rotary_refuses(name):
    refused(turn(*OVERLAPS[name]))


def test_one_token_has_no_token_stride():
    """Its heads are all there is to compare."""
    refused(turn(rows(0, 4, out=FAR, out_head=0), tokens=1))
    refused(turn(rows(0, 4, out=D, out_tok=0), tokens=1))


@pytest.mark.parametrize("name,q", [
    ("heads", rows(0, 32, out=FAR, out_tok=D, out_head=D)),
    ("a token later", rows(0, 32, out=WIDE)),
    ("into the keys", rows(0, 32, out=4 * D)),
    ("into the values", rows(0, 32, out=40 * D)),
    ("keys of the queries", rows(32 * D, 32, tok=WIDE)),
    ("the keys' buffer by other strides", rows(FAR, 32, out=0, out_tok=32 * D)),
])
@pytest.mark.parametrize("single", [False, True])
def test_rotary_append_refuses(name, q, single):
    cu, lens, new = P - (1 << 20), P - (1 << 19), P - (1 << 18)
    kv = N.PagedKV(P + (1 << 30), P + (1 << 31), N.IA_BF16, 16, 9, 8 * 16 * D, 16 * D, D, 8 * 16 * D, 16 * D, D, P, 4, 4)
    packed = N.PackedKV(P + 64 * D, P + 80 * D, N.IA_BF16, WIDE, D, WIDE, D)
    rot = N.Rotary(P, D, 0, 1.0)
    refused(N.lib().ia_rotary_append_kv(rot, q, packed, kv, None if single else cu, lens, new, None, T if single else 2, T,
                                        8, D, None))


# ------------------------------------------------------------------ views that lie apart

def views(device):
    """``(q, k)`` and outputs of every kind that may be given."""
    g = torch.Generator(device=device)
    g.manual_seed(1)

    def buf(*shape):
        return torch.randn(shape, device=device, generator=g).bfloat16()

    b = buf(T, 12, 64)
    yield "one projection, in place", b[:, :8], b[:, 8:10], b[:, :8], b[:, 8:10]
    b = buf(T, 24, 64)
    yield "outputs beside the inputs", b[:, :8], b[:, 8:10], b[:, 10:18], b[:, 18:20]
    b = buf(T, 4, 3, 64)  # q, k and v of a head side by side
    yield "a head's q and k, in place", b[:, :, 0], b[:, :, 1], b[:, :, 0], b[:, :, 1]
    yield "into the values", b[:, :, 0], None, b[:, :, 2], None
    b = buf(10, T, 64)  # heads first
    yield "heads first, in place", b[:8].transpose(0, 1), b[8:].transpose(0, 1), b[:8].transpose(0, 1), b[8:].transpose(0, 1)
    b = buf(4, 3 * T, 64)  # heads first, tokens of three batches
    yield "stretches of every head", b[:, :T].transpose(0, 1), None, b[:, T:2 * T].transpose(0, 1), None
    b = buf(2 * T, 4, 64)
    yield "every other token", b[::2], None, b[1::2], None
    b = buf(T, 4, 128)
    yield "halves of a row", b[:, :, :64], b[:, :, 64:], b[:, :, :64], b[:, :, 64:]
    yield "both from one", b[:, :, :64], b[:, :, :64], buf(T, 4, 64), buf(T, 4, 64)
    b, c = buf(1, 4, 64), buf(T, 4, 64)
    yield "expanded inputs", b.expand(T, 4, 64), c[:, :1].expand(T, 4, 64), buf(T, 4, 64), buf(T, 4, 64)


@pytest.mark.gpu
def test_views_that_lie_apart(device):
    pos = torch.arange(3, 3 + T, device=device, dtype=torch.int32)
    plan = ia.rotary_plan(64, device=device)
    for name, q, k, q_out, k_out in views(device):
        announce(f"rotary views, {name}")
        want_q, want_k = ia.apply_rotary(q.clone(), None if k is None else k.clone(), pos, plan)
        got_q, got_k = ia.apply_rotary(q, k, pos, plan, q_out=q_out, k_out=k_out)
        torch.cuda.synchronize()
        assert torch.equal(got_q, want_q) and (k is None or torch.equal(got_k, want_k)), name


@pytest.mark.gpu
@pytest.mark.parametrize("single", [False, True])
def test_queries_turned_in_place_beside_keys(device, single):
    """The projection's own buffer, heads of one group side by side too."""
    announce(f"rotary append, queries in place {single}")
    plan = ia.rotary_plan(64, device=device)
    n = 5
    cu = None if single else torch.tensor([0, 2, n], device=device, dtype=torch.int32)
    lens = torch.tensor([3, 40, 0, 16, 7][:n if single else 2], device=device, dtype=torch.int32)
    table = torch.randperm(20, device=device)[:lens.numel() * 4].view(-1, 4).to(torch.int32)
    for split in (lambda b: (b[:, :4], b[:, 4:6], b[:, 6:]), lambda b: (b[:, 0::4], b[:, 1::4], b[:, 2::4])):
        got = []
        for in_place in (False, True):
            b = torch.randn((n, 8, 64), device=device, generator=torch.Generator(device=device).manual_seed(3)).bfloat16()
            q, k, v = split(b)
            pools = [torch.zeros((20, 2, 16, 64), device=device, dtype=torch.bfloat16) for _ in "kv"]
            q, lens_after = ia.rotary_append_kv(q, k, v, plan, *pools, table, lens.clone(), cu,
                                                q_out=q if in_place else None)
            torch.cuda.synchronize()
            got.append([q, lens_after, *pools])
        assert all(torch.equal(x, y) for x, y in zip(*got))
