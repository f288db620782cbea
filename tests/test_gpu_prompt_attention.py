"""Prompt attention (packed and paged K/V) against float64 attention of the same inputs.

Bars, from the roundings alone.  bf16 and fp8 operands enter the products exactly.  P is
rounded to bf16: half a step of its 8 significant bits, 2^-8 relative to it, which moves a
row by at most 2^-8 A with A = sum p |v| (p the float64 softmax weights).  The output is
rounded to its type: 2^-8 |want| for bf16, 2^-24 |want| for float32.  Scores are float32
sums of D products (|s| stays below 2^5 here: errors below 128 * 2^-24 * 2^5 = 2^-12), so
the exponentials and the float32 sums over the keys add less than 2^-11 A.
    bf16, fp8:  |got - want| <= (2^-8 + 2^-11) A + half a step of the output
float32 caches have no rounded P: the scores' and the sums' errors, 2^-24 relative to each
of D products, of the keys' terms and of the exponential's argument:
    f32:        |got - want| <= 2^-24 * 8 * (keys + 128) A + 2^-24 |want|
"""

import math

import pytest
import torch

import interattn_amd as ia
from tests._util import announce

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}


def reference(q, k, v, first, scale):
    """(attention, its bound A) of rows ``q [n, Hq, D]`` at positions first.. over ``k, v [L, Hkv, D]``."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    n, hq, d = q.shape
    total, hkv, _ = k.shape
    out, mag = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
        for i in range(n):
            seen = min(first + i + 1, total)
            if seen <= 0:
                continue
            p = torch.softmax(kh[:seen] @ q[i, h] * scale, 0)
            out[i, h] = p @ vh[:seen]
            mag[i, h] = p @ vh[:seen].abs()
    return out, mag


def check(got, want, mag, kv, keys, what):
    g = got.detach().cpu().double()
    if kv == "f32":
        bar = 2.0 ** -24 * 8 * (keys + 128) * mag + 2.0 ** -24 * want.abs()
    else:
        bar = (2.0 ** -8 + 2.0 ** -11) * mag + (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24) * want.abs()
    worst = float(((g - want).abs() - bar).max()) if g.numel() else 0.0
    finite = bool(torch.isfinite(g).all())
    assert finite and worst <= 1e-30, (what, finite, worst)


def packed(device, lens, hq, hkv, d, kv, fused, seed, extra=0):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    total = sum(lens) + extra
    buf = torch.randn((total, hq + 2 * hkv, d), device=device, generator=gen).to(DT[kv])
    parts = buf.split([hq, hkv, hkv], dim=1)
    if not fused:
        parts = tuple(x.contiguous() for x in parts)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], device=device, dtype=torch.int32)
    return (*parts, cu)


PACKED = [
    # lens, hq, hkv, d, kv, fused
    ([1], 4, 1, 128, "bf16", False),
    ([5], 1, 1, 64, "bf16", False),
    ([16, 1, 0, 17, 33], 8, 2, 128, "bf16", True),
    ([64], 4, 1, 128, "bf16", False),
    ([65, 63, 128], 8, 8, 64, "bf16", True),
    ([333], 32, 8, 128, "bf16", True),
    ([700, 2, 129], 6, 1, 128, "bf16", False),
    ([257], 16, 2, 64, "bf16", True),
    ([100], 64, 1, 64, "bf16", False),
    ([40], 3, 3, 128, "f32", True),
    ([1, 70, 0, 200], 8, 2, 64, "f32", False),
    ([300], 8, 1, 128, "f32", True),
    ([31, 32], 32, 1, 128, "f32", False),
    ([0, 0], 4, 2, 64, "bf16", False),
]


@pytest.mark.parametrize("c", PACKED, ids=[f"{c[4]}-{c[3]}-{c[1]}x{c[2]}-{'.'.join(map(str, c[0]))}" for c in PACKED])
def test_packed(c, device):
    lens, hq, hkv, d, kv, fused = c
    announce(f"prompt {c}")
    q, k, v, cu = packed(device, lens, hq, hkv, d, kv, fused, len(lens) + d, extra=3)
    out = torch.full((q.shape[0], hq, d), 7.0, device=device, dtype=DT[kv])
    ia.prompt_attention(q, k, v, cu, out=out, workspace={})
    torch.cuda.synchronize()
    at = 0
    for n in lens:
        want, mag = reference(q[at:at + n], k[at:at + n], v[at:at + n], 0, d ** -0.5)
        check(out[at:at + n], want, mag, kv, n, (c, n))
        at += n
    assert bool((out[at:] == 7.0).all()), "rows of no sequence changed"


def paged(device, lens, hkv, d, page, kv, layout, seed, spare=2, table_pad=1):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    need = [math.ceil(n / page) for n in lens]
    n_pages = sum(need) + spare
    x = torch.randn((2, n_pages, hkv, page, d), device=device, generator=gen)
    scales = None
    if kv == "fp8":
        sc = x.abs().amax(dim=(3, 4)) / 448.0
        x = x / sc[..., None, None]
        scales = (sc[0].contiguous(), sc[1].contiguous())
    if layout == "paired":
        buf = x.to(DT[kv]).permute(1, 2, 0, 3, 4).contiguous()
        pk, pv = buf[:, :, 0], buf[:, :, 1]
    else:
        pk, pv = x[0].to(DT[kv]), x[1].to(DT[kv])
    perm = torch.randperm(n_pages, device=device, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + table_pad), -1, device=device, dtype=torch.int32)
    off = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[off:off + n]
        off += n
    return pk, pv, scales, table


def gather(pool, scale, row, n):
    page = pool.shape[2]
    pages = row[:math.ceil(n / page)].long()
    x = pool[pages].float().double()
    if scale is not None:
        x = x * scale[pages].double()[:, :, None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:n]


PAGED = [
    # new, past, hq, hkv, d, page, kv, layout
    ([1], [0], 4, 1, 128, 16, "bf16", "split"),
    ([1, 1, 1], [15, 16, 4000], 32, 8, 128, 16, "bf16", "paired"),
    ([3, 0, 9], [1000, 50, 7], 8, 2, 64, 32, "bf16", "split"),
    ([8], [2500], 4, 1, 128, 48, "bf16", "split"),
    ([200, 1, 64], [0, 777, 1300], 8, 2, 128, 16, "bf16", "paired"),
    ([40], [3000], 16, 2, 64, 64, "bf16", "split"),
    ([1, 2, 30], [600, 0, 77], 8, 2, 128, 16, "fp8", "split"),
    ([100, 5], [700, 2000], 16, 2, 64, 32, "fp8", "paired"),
    ([70], [1900], 12, 2, 128, 16, "fp8", "split"),
    ([1, 33], [300, 10], 4, 2, 128, 16, "f32", "split"),
    ([60, 4], [900, 1500], 4, 4, 64, 32, "f32", "paired"),
    ([25], [1400], 8, 2, 128, 16, "f32", "split"),
]


@pytest.mark.parametrize("c", PAGED, ids=[f"{c[6]}-{c[4]}-{c[2]}x{c[3]}-{i}" for i, c in enumerate(PAGED)])
def test_paged(c, device):
    new, past, hq, hkv, d, page, kv, layout = c
    announce(f"paged prompt {c}")
    lens = [a + b for a, b in zip(new, past)]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, layout, d + page)
    gen = torch.Generator(device=device)
    gen.manual_seed(5)
    q = torch.randn((sum(new), hq, d), device=device, generator=gen).to(DT["f32" if kv == "f32" else "bf16"])
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device=device, dtype=torch.int32)
    seq = torch.tensor(lens, device=device, dtype=torch.int32)
    out = ia.paged_prompt_attention(q, pk, pv, table, seq, cu, scales=scales, workspace={})
    torch.cuda.synchronize()
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        k = gather(pk, scales and scales[0], table[b], total)
        v = gather(pv, scales and scales[1], table[b], total)
        want, mag = reference(q[at:at + n], k, v, total - n, d ** -0.5)
        check(out[at:at + n], want, mag, kv, total, (c, b))
        at += n
