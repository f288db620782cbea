"""Rotary positions of packed rows against the rotation in 64 bits.

Bars: the sums are float32.  A turned value is a c - b s with c and s off by at most 2^-23 times
the factor (a rounding of the angle, of each step of the sums, of the product with the factor:
measured against 64 bits the bar is four half steps of 2^-24 each) and three roundings of its
own; so 8 * 2^-24 * (|a| + |b|) * factor, and for bf16 outputs half a step more: bf16 has
2^-7 between 1 and its successor, so half a step is 2^-8 of the value."""

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import rotary as R
from tests._util import announce

pytestmark = pytest.mark.gpu

SCALING = {"yarn": dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096)}


def frequencies(rot, base=10000.0, scaling=None):
    return ia.rotary_frequencies(rot, base=base, scaling=SCALING.get(scaling))


def bar_of(x, rot, layout, factor, dtype):
    """Elementwise bar of the turned rows ``x``."""
    a = np.abs(x.double().cpu().numpy())
    r = np.zeros_like(a)
    if layout == "half":
        r[..., :rot // 2] = r[..., rot // 2:rot] = a[..., :rot // 2] + a[..., rot // 2:rot]
    else:
        r[..., 0:rot:2] = r[..., 1:rot:2] = a[..., 0:rot:2] + a[..., 1:rot:2]
    bar = 8 * 2.0 ** -24 * r * factor
    return bar + (2.0 ** -8 * (r * factor) if dtype == torch.bfloat16 else 0)


def check(got, x, pos, w, layout, factor, inverse=False):
    want = R.turn(x.double().cpu().numpy(), pos.cpu().numpy(), w, layout, factor, inverse)
    rot = 2 * len(w)
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bar_of(x, rot, layout, factor, x.dtype)).all(), off.max()
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot,layout,fused,scaling", [
    (1, 1, 1, 64, 64, "half", False, None),
    (1, 32, 8, 128, 128, "half", True, None),
    (33, 32, 8, 128, 128, "interleaved", True, "yarn"),
    (257, 7, 1, 128, 96, "interleaved", False, None),
    (100, 4, 2, 128, 64, "half", True, "yarn"),
    (65, 5, 5, 64, 26, "half", False, None),     # halves of 13: no whole chunk
    (65, 3, 1, 64, 26, "interleaved", True, None),
    (40, 2, 1, 16, 16, "half", False, None),
    (19, 2, 2, 48, 48, "half", True, None),
    (11, 3, 1, 256, 250, "half", False, None),
    (300, 2, 1, 256, 256, "interleaved", False, None),
    (7, 4, 4, 80, 2, "half", True, None),
    (7, 4, 4, 80, 0, "half", True, None),
])
def test_rows_are_turned(device, dtype, tokens, hq, hkv, d, rot, layout, fused, scaling):
    announce(f"rotary {dtype} {tokens} {hq}+{hkv} {d} {rot} {layout}")
    g = torch.Generator(device=device)
    g.manual_seed(tokens * 7 + rot)
    w, factor = frequencies(rot, scaling=scaling)
    plan = ia.rotary_plan(rot, scaling=SCALING.get(scaling), layout=layout, device=device)
    buf = torch.randn((tokens, hq + hkv, d), device=device, generator=g).to(dtype)
    q, k = buf.split([hq, hkv], 1)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.randint(-3000, 200000, (tokens,), device=device, generator=g, dtype=torch.int32)
    for inverse in (False, True):
        qo, ko = ia.apply_rotary(q, k, pos, plan, inverse=inverse)
        torch.cuda.synchronize()
        check(qo, q, pos, w, layout, factor, inverse)
        check(ko, k, pos, w, layout, factor, inverse)


def test_any_position_has_its_angle(device):
    """The ends of the range, where float32 angles would be off by 100 turns: against angles
    formed with whole numbers."""
    announce("rotary, far positions")
    rot = d = 64
    plan = ia.rotary_plan(rot, device=device)
    pos = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, -123456789]
    x = torch.randn((len(pos), 2, d), device=device)
    got, none = ia.apply_rotary(x, None, torch.tensor(pos, device=device, dtype=torch.int32), plan)
    torch.cuda.synchronize()
    assert none is None
    turns = [t % (1 << 64) for t in plan.turns.tolist()]
    angle = np.array([[(p * t % (1 << 64)) / 2.0 ** 64 for t in turns] for p in pos]) * 2 * np.pi
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    v = x.double().cpu().numpy()
    a, b = v[..., :32], v[..., 32:]
    want = np.concatenate([a * c - b * s, b * c + a * s], -1)
    assert (np.abs(got.double().cpu().numpy() - want) <= bar_of(x, rot, "half", 1.0, x.dtype)).all()


def test_outputs_may_be_the_inputs_or_given(device):
    announce("rotary, in place")
    plan = ia.rotary_plan(128, device=device)
    buf = torch.randn((50, 12, 128), device=device).bfloat16()
    pos = torch.arange(50, device=device, dtype=torch.int32)
    want_q, want_k = ia.apply_rotary(buf[:, :8], buf[:, 8:10], pos, plan)
    rest = buf[:, 10:].clone()
    given = torch.full((50, 3, 8, 128), 7.0, device=device, dtype=torch.bfloat16)
    got, _ = ia.apply_rotary(buf[:, :8], None, pos, plan, q_out=given[:, 1])
    assert got.data_ptr() == given[:, 1].data_ptr() and torch.equal(given[:, 1], want_q)
    assert bool((given[:, 0] == 7).all()) and bool((given[:, 2] == 7).all())
    q, k = ia.apply_rotary(buf[:, :8], buf[:, 8:10], pos, plan, q_out=buf[:, :8], k_out=buf[:, 8:10])
    torch.cuda.synchronize()
    assert torch.equal(buf[:, :8], want_q) and torch.equal(buf[:, 8:10], want_k) and torch.equal(buf[:, 10:], rest)
    # no tokens
    q, k = ia.apply_rotary(buf[:0, :8], buf[:0, 8:10], pos[:0], plan)
    assert q.shape == (0, 8, 128) and k.shape == (0, 2, 128)


@pytest.mark.parametrize("layout,rot", [("half", 64), ("interleaved", 36), ("half", 36)])
def test_not_finite_stays_where_it_is(device, layout, rot):
    """A value that is not finite reaches its pair and nothing else; unturned channels are as
    they are."""
    announce(f"rotary, not finite {layout} {rot}")
    plan = ia.rotary_plan(rot, layout=layout, device=device)
    x = torch.randn((4, 1, 64), device=device)
    pos = torch.arange(4, device=device, dtype=torch.int32)
    clean, _ = ia.apply_rotary(x, None, pos, plan)
    y = x.clone()
    y[1, 0, 3], y[2, 0, 40], y[3, 0, 63] = float("inf"), float("nan"), float("-inf")
    got, _ = ia.apply_rotary(y, None, pos, plan)
    torch.cuda.synchronize()

    def partner(i):
        if i >= rot:
            return i
        if layout == "half":
            return (i + rot // 2) % rot
        return i ^ 1

    touched = {(t, c) for t, i in ((1, 3), (2, 40), (3, 63)) for c in (i, partner(i))}
    for t in range(4):
        for c in range(64):
            if (t, c) not in touched:
                assert got[t, 0, c] == clean[t, 0, c]
    if rot < 64:
        assert got[3, 0, 63] == float("-inf")


def test_inverse_is_the_gradient(device):
    """The transposed rotation against the formula's gradient in 64 bits, and against
    differences: the rotation is linear, so for any step e the difference of the rotation's
    outputs over the step is the product with the gradient's rows (float32: the bar of the
    values' rounding, over e)."""
    announce("rotary, gradient")
    w, factor = frequencies(32, scaling="yarn")
    for layout in ("half", "interleaved"):
        plan = ia.rotary_plan(32, scaling=SCALING["yarn"], layout=layout, device=device)
        x, g = torch.randn((9, 3, 64), device=device), torch.randn((9, 3, 64), device=device)
        pos = torch.randint(0, 5000, (9,), device=device, dtype=torch.int32)
        grad, _ = ia.apply_rotary(g, None, pos, plan, inverse=True)
        torch.cuda.synchronize()
        check(grad, g, pos, w, layout, factor, inverse=True)
        e, v = 0.5, torch.randn_like(x)
        up, _ = ia.apply_rotary(x + e * v, None, pos, plan)
        down, _ = ia.apply_rotary(x - e * v, None, pos, plan)
        slope = ((up.double() - down.double()) * g.double()).sum((1, 2)) / (2 * e)
        want = (v.double() * grad.double()).sum((1, 2))
        # 192 products of values up to about 4, each off by the bar of its row and x +- e v by 2^-24
        bar = 192 * 4 * 8 * 2.0 ** -24 * 8 * factor / (2 * e)
        assert bool(((slope - want).abs() <= bar).all())


def test_a_captured_rotation_follows_its_inputs(device):
    announce("rotary, captured")
    plan = ia.rotary_plan(64, device=device)
    q, k = torch.randn((20, 4, 64), device=device), torch.randn((20, 2, 64), device=device)
    pos = torch.arange(20, device=device, dtype=torch.int32)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ia.apply_rotary(q, k, pos, plan, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ia.apply_rotary(q, k, pos, plan, q_out=qo, k_out=ko)
    for step in range(4):
        q.normal_()
        k.normal_()
        pos.add_(1000 * step)
        want = ia.apply_rotary(q, k, pos, plan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_refusals(device):
    plan = ia.rotary_plan(64, device=device)
    x, pos = torch.zeros((4, 2, 64), device=device), torch.zeros(4, device=device, dtype=torch.int32)
    for bad in (lambda: ia.apply_rotary(x, None, pos[:3], plan), lambda: ia.apply_rotary(x, None, pos.long(), plan),
                lambda: ia.apply_rotary(x.half(), None, pos, plan), lambda: ia.apply_rotary(x, x.bfloat16(), pos, plan),
                lambda: ia.apply_rotary(x, x[:3], pos, plan), lambda: ia.apply_rotary(x[..., :32], None, pos, plan),
                lambda: ia.apply_rotary(x, None, pos, plan, q_out=x.bfloat16()),
                lambda: ia.apply_rotary(x, None, pos, plan, k_out=x),
                lambda: ia.apply_rotary(x, None, pos, plan, q_out=torch.empty_like(x[:1]).expand(4, 2, 64)),
                lambda: ia.apply_rotary(x, None, pos, plan, q_out=torch.empty_like(x[:, :1]).expand(4, 2, 64)),
                lambda: ia.apply_rotary(x.transpose(1, 2), None, pos, plan),
                lambda: ia.apply_rotary(x, None, pos, ia.rotary_plan(64, device="cpu"))):
        with pytest.raises(ValueError):
            bad()
