"""What the prompt-side attention calls do at their edges: values that are not finite in
places a row must not see, pages that are not there, offsets that disagree with the data,
odd strides, scales of any sign, streams, graphs and shared workspaces."""

import math

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, packed, paged, reference

pytestmark = pytest.mark.gpu


def i32(device, values):
    return torch.tensor(values, device=device, dtype=torch.int32)


@pytest.mark.parametrize("kv,d,n", [("bf16", 128, 70), ("bf16", 64, 20), ("f32", 128, 40), ("f32", 64, 9)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_tokens_that_are_not_finite(kv, d, n, bad, device):
    """A later token whose K or V is not finite leaves the rows before it as they are; the
    rows that see it are not finite (NaN, or the infinity itself)."""
    announce(f"hidden {bad} {kv} {d} {n}")
    hq, hkv = 8, 2
    q, k, v, cu = packed(device, [n, 5], hq, hkv, d, kv, False, n)
    k, v = k.clone(), v.clone()
    at = n - 6
    v[at, 0, 3] = bad
    k[at + 2, 1, 5] = bad
    out = ia.prompt_attention(q, k, v, cu, workspace={})
    torch.cuda.synchronize()
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[at + 2, 1, 5], clean_v[at, 0, 3] = 0, 0
    want, mag = reference(q[:n], clean_k[:n], clean_v[:n], 0, d ** -0.5)
    check(out[:at], want[:at], mag[:at], kv, n, "rows before")
    # kv head 1 sees a clean token at `at`, head 0 one at `at + 2`
    check(out[:at + 2, 4:], want[:at + 2, 4:], mag[:at + 2, 4:], kv, n, "head 1")
    assert not bool(torch.isfinite(out[at:n, :4, 3]).any())
    assert bool(torch.isfinite(out[n:]).all())
    rest = torch.ones(d, dtype=torch.bool)
    rest[3] = False
    check(out[at:n, :4][..., rest], want[at:, :4][..., rest], mag[at:, :4][..., rest], kv, n, "other dims")


def reference_heads(q, k, v, first, scale):
    """``reference`` by whole heads, for long inputs whose values are all finite."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    (n, hq, d), (total, hkv, _) = q.shape, k.shape
    hidden = torch.arange(total)[None] > first + torch.arange(n)[:, None]
    out, mag = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    for h in range(hq):
        p = torch.softmax((q[:, h] @ k[:, h * hkv // hq].T * scale).masked_fill(hidden, -math.inf), -1)
        out[:, h], mag[:, h] = p @ v[:, h * hkv // hq], p @ v[:, h * hkv // hq].abs()
    return out, mag


# enough rows that every launch takes its tiles of 128 (the small cases run in tiles of 32)
LARGE = [
    ([900, 300, 65], 32, 8, 128, "bf16", True),
    ([1500, 1, 40], 16, 2, 64, "bf16", False),
    ([130], 64, 1, 128, "f32", True),
    ([90], 64, 1, 64, "f32", False),
]


@pytest.mark.parametrize("c", LARGE, ids=[f"{c[4]}-{c[3]}-{c[1]}x{c[2]}" for c in LARGE])
def test_packed_in_tiles_of_128_rows(c, device):
    lens, hq, hkv, d, kv, fused = c
    announce(f"prompt large {c}")
    q, k, v, cu = packed(device, lens, hq, hkv, d, kv, fused, 17)
    out = ia.prompt_attention(q, k, v, cu, workspace={})
    torch.cuda.synchronize()
    at = 0
    for n in lens:
        want, mag = reference_heads(q[at:at + n], k[at:at + n], v[at:at + n], 0, d ** -0.5)
        check(out[at:at + n], want, mag, kv, n, (c, n))
        at += n


@pytest.mark.parametrize("kv,d,page", [("bf16", 128, 16), ("fp8", 128, 32), ("fp8", 64, 16)])
def test_paged_in_tiles_of_128_rows(kv, d, page, device):
    announce(f"paged large {kv} {d}")
    new, past, hq, hkv = [400, 1, 330], [1000, 700, 0], 32, 8
    lens = [a + b for a, b in zip(new, past)]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, "paired", 31)
    q = torch.randn((sum(new), hq, d), device=device).to(torch.bfloat16)
    cu = i32(device, [0, 400, 401, 731])
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, lens), cu, scales=scales, workspace={})
    torch.cuda.synchronize()
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        k, v = gather(pk, scales and scales[0], table[b], total), gather(pv, scales and scales[1], table[b], total)
        want, mag = reference_heads(q[at:at + n], k, v, total - n, d ** -0.5)
        check(out[at:at + n], want, mag, kv, total, b)
        at += n


def test_hidden_tokens_that_are_not_finite_in_tiles_of_128_rows(device):
    announce("hidden, large")
    n, hq, hkv, d = 700, 32, 8, 128
    q, k, v, cu = packed(device, [n], hq, hkv, d, "bf16", False, 5)
    want, mag = reference_heads(q, k, v, 0, d ** -0.5)
    k, v = k.clone(), v.clone()
    v[650, 2, 9], k[333, 5, 1], v[20, 7, 100] = math.nan, math.nan, math.inf
    out = ia.prompt_attention(q, k, v, cu, workspace={})
    torch.cuda.synchronize()
    sees = torch.zeros(n, hq, d, dtype=torch.bool)
    sees[650:, 8:12, 9], sees[333:, 20:24, :], sees[20:, 28:32, 100] = True, True, True
    assert not bool(torch.isfinite(out.cpu()[sees]).any())
    got = torch.where(sees, want, out.cpu().double())
    check(got.to(torch.bfloat16), torch.where(sees, got.to(torch.bfloat16).double(), want), mag, "bf16", n, "unseen")


@pytest.mark.parametrize("kv", ["bf16", "f32", "fp8"])
def test_rows_past_a_sequence_and_missing_pages(kv, device):
    """Pool rows behind a sequence's end hold NaN; table entries are -1 or past the pool:
    neither reaches the output, which is the attention of the keys that are there."""
    announce(f"missing pages {kv}")
    hkv, hq, d, page = 2, 8, 64, 16
    lens, new = [100, 45, 33], [40, 3, 33]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, "split", 9, spare=6)
    if kv != "fp8":
        for b, n in enumerate(lens):
            if n % page:
                last = int(table[b, n // page])
                pk[last, :, n % page:] = math.nan
                pv[last, :, n % page:] = math.nan
    table[0, 1], table[0, 3], table[1, 0] = -1, pk.shape[0], 1 << 30
    q = torch.randn((sum(new), hq, d), device=device).to(DT["f32" if kv == "f32" else "bf16"])
    cu = i32(device, [0, 40, 43, 76])
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, lens), cu, scales=scales, workspace={})
    torch.cuda.synchronize()
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        row = table[b].clone()
        gone = [p for p in range(-(-total // page)) if not 0 <= int(row[p]) < pk.shape[0]]
        row[gone] = 0
        k, v = gather(pk, scales and scales[0], row, total), gather(pv, scales and scales[1], row, total)
        keep = torch.tensor([t // page not in gone for t in range(total)])
        for i in range(n):
            mine = keep.clone()
            mine[total - n + i + 1:] = False
            ki, vi = k[mine.to(k.device)], v[mine.to(v.device)]
            want, mag = reference(q[at + i:at + i + 1], ki, vi, max(ki.shape[0] - 1, 0), d ** -0.5)
            check(out[at + i:at + i + 1], want, mag, kv, total, (b, i))
        at += n


def test_nothing_to_see_is_zeros(device):
    announce("nothing to see")
    hkv, hq, d, page = 1, 4, 128, 16
    pk, pv, _, table = paged(device, [64, 64, 64], hkv, d, page, "bf16", "split", 2)
    table[1] = -1
    # sequence 0 claims more new tokens than it has, 1 has no page, 2 has a negative length
    q = torch.randn((12, hq, d), device=device).to(torch.bfloat16)
    out = ia.paged_prompt_attention(q, pk, pv, table, i32(device, [2, 64, -7]), i32(device, [0, 5, 9, 12]), workspace={})
    torch.cuda.synchronize()
    assert bool((out[:3] == 0).all()) and bool((out[5:] == 0).all())
    want, mag = reference(q[3:5], gather(pk, None, table[0], 2), gather(pv, None, table[0], 2), 0, d ** -0.5)
    check(out[3:5], want, mag, "bf16", 2, "two tokens")


def test_offsets_are_clipped_to_the_rows(device):
    """cu_seqlens outside [0, tokens] is clipped; rows of no sequence keep what out held."""
    announce("clipped offsets")
    q, k, v, _ = packed(device, [50], 4, 1, 64, "bf16", False, 3)
    out = torch.full(q.shape, 3.0, device=device, dtype=torch.bfloat16)
    ia.prompt_attention(q, k, v, i32(device, [-4, 10, 10, 30]), out=out)
    torch.cuda.synchronize()
    for a, b in ((0, 10), (10, 30)):
        want, mag = reference(q[a:b], k[a:b], v[a:b], 0, 64 ** -0.5)
        check(out[a:b], want, mag, "bf16", b - a, (a, b))
    assert bool((out[30:] == 3.0).all())
    out.fill_(3.0)
    ia.prompt_attention(q, k, v, i32(device, [7, 20, 900]), out=out)
    torch.cuda.synchronize()
    for a, b in ((7, 20), (20, 50)):
        want, mag = reference(q[a:b], k[a:b], v[a:b], 0, 64 ** -0.5)
        check(out[a:b], want, mag, "bf16", b - a, (a, b))
    assert bool((out[:7] == 3.0).all())


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_any_scale(scale, kv, device):
    announce(f"scale {scale} {kv}")
    n, hq, hkv, d = 45, 4, 2, 64
    q, k, v, cu = packed(device, [n], hq, hkv, d, kv, False, 8)
    q = (q * 0.3).to(q.dtype)
    out = ia.prompt_attention(q, k, v, cu, scale=scale)
    torch.cuda.synchronize()
    want, mag = reference(q, k, v, 0, scale)
    check(out, want, mag, kv, n, scale)


def test_large_scores_and_falling_maxima(device):
    """Scores that grow and fall by hundreds over a row: the running maximum is exact."""
    announce("large scores")
    n, hq, hkv, d = 200, 2, 1, 64
    q, k, v, cu = packed(device, [n], hq, hkv, d, "f32", False, 8)
    ramp = torch.cat([torch.linspace(0, 12, 100), torch.linspace(12, -12, 100)]).to(device)
    q = torch.ones_like(q)
    k = (ramp[:, None, None] * torch.ones_like(k)).contiguous()
    out = ia.prompt_attention(q, k, v, cu)
    torch.cuda.synchronize()
    want, mag = reference(q, k, v, 0, d ** -0.5)
    # scores reach 12 * 64 / 8 = 96: an error of 64 products' roundings, 64 * 2^-24 * 96, in the
    # exponent moves a weight by as much, relatively
    assert float(((out.cpu().double() - want).abs() - (64 * 96 * 2.0 ** -24 * 4) * mag).max()) <= 1e-30


def test_odd_strides_and_types(device):
    """Head-major q, k and v, a float32 q over bf16 K/V, both output types."""
    announce("strides and types")
    n, hq, hkv, d = 77, 6, 3, 128
    gen = torch.Generator(device=device)
    gen.manual_seed(4)
    q = torch.randn((hq, n, d + 8), device=device, generator=gen).transpose(0, 1)[..., :d]
    k = torch.randn((hkv, n, 2 * d), device=device, generator=gen).to(torch.bfloat16).transpose(0, 1)[..., d:]
    v = torch.randn((n, hkv + 2, d), device=device, generator=gen).to(torch.bfloat16)[:, 1:1 + hkv]
    cu = i32(device, [0, 30, n])
    for out_dtype in (torch.float32, torch.bfloat16):
        out = ia.prompt_attention(q, k, v, cu, out_dtype=out_dtype)
        torch.cuda.synchronize()
        assert out.dtype == out_dtype
        qr = q.to(torch.bfloat16)  # (the products take bf16 operands)
        for a, b in ((0, 30), (30, n)):
            want, mag = reference(qr[a:b], k[a:b], v[a:b], 0, d ** -0.5)
            check(out[a:b], want, mag, "bf16", b - a, (out_dtype, a))


def test_identity_table_reads_a_contiguous_view(device):
    announce("identity table")
    n, hq, hkv, d, page = 90, 4, 2, 64, 32
    pool = torch.randn((2, 3, hkv, page, d), device=device).to(torch.bfloat16)
    q = torch.randn((11, hq, d), device=device).to(torch.bfloat16)
    out = ia.paged_prompt_attention(q, pool[0], pool[1], None, i32(device, [n]), i32(device, [0, 11]))
    torch.cuda.synchronize()
    k, v = (x.permute(0, 2, 1, 3).reshape(-1, hkv, d)[:n] for x in pool)
    want, mag = reference(q, k, v, n - 11, d ** -0.5)
    check(out, want, mag, "bf16", n, "identity")


def test_single_token_equals_the_dense_decode(device):
    """New lengths of one are a decode step: the same as paged_decode to rounding (both sides
    within half a step of P and of the output of the exact result)."""
    announce("single tokens")
    hkv, hq, d, page = 2, 8, 128, 16
    lens = [1, 16, 700, 333]
    pk, pv, _, table = paged(device, lens, hkv, d, page, "bf16", "paired", 6)
    q = torch.randn((4, hq, d), device=device).to(torch.bfloat16)
    seq = i32(device, lens)
    ws = {}
    one = ia.paged_prompt_attention(q, pk, pv, table, seq, i32(device, [0, 1, 2, 3, 4]), workspace=ws)
    for b, n in enumerate(lens):
        want, mag = reference(q[b:b + 1], gather(pk, None, table[b], n), gather(pv, None, table[b], n), n - 1, d ** -0.5)
        check(one[b:b + 1], want, mag, "bf16", n, b)


@pytest.mark.parametrize("kv", ["bf16", "f32", "fp8"])
def test_prefix_with_rows_and_pages_that_are_not_there(kv, device):
    """NaN behind the sequences, a member shorter than its prefix whose group sees a NaN V
    there, table entries that do not exist."""
    announce(f"prefix edges {kv}")
    hkv, hq, d, page = 1, 8, 64, 16
    lens = [200, 130, 201, 260, 210]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, "split", 21)
    shared = 192
    for i in range(1, 5):
        table[i, :min(lens[i], shared) // page] = table[0, :min(lens[i], shared) // page]
    if kv != "fp8":
        # token 150: members but the second see it; token 129 is the second's last
        pv[int(table[0, 9]), 0, 150 % page, 7] = math.nan
        pv[int(table[1, 8]), 0, 2:] = pv[int(table[0, 8]), 0, 2:]
        pv[int(table[1, 8]), 0, :2] = pv[int(table[0, 8]), 0, :2]
        pk[int(table[1, 8])] = pk[int(table[0, 8])]
        last = int(table[3, 260 // page])
        pk[last, :, 260 % page:] = math.nan
        pv[last, :, 260 % page:] = math.nan
    table[4, 12] = -1  # sequence 4's own tokens 192..207 are not there
    q = torch.randn((5, hq, d), device=device).to(DT["f32" if kv == "f32" else "bf16"])
    out = ia.shared_prefix_decode(q, pk, pv, table, i32(device, lens), i32(device, [0, 5]), i32(device, [shared]),
                                  scales=scales, workspace={})
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        row = table[b].clone()
        if b == 1 and kv == "fp8":
            row[:9] = table[0, :9]  # (its own partial page is not read: the prefix is the group's)
        row[row < 0] = 0
        k, v = gather(pk, scales and scales[0], row, n), gather(pv, scales and scales[1], row, n)
        keep = [t for t in range(n) if not (b == 4 and 192 <= t < 208)]
        k, v = k[keep], v[keep]
        want, mag = reference(q[b:b + 1], k.nan_to_num(), v.nan_to_num(), len(keep) - 1, d ** -0.5)
        dims = torch.ones(d, dtype=torch.bool)
        if kv != "fp8" and b != 1:
            dims[7] = False
            assert bool(torch.isnan(out[b, :, 7]).all()), b
        check(out[b:b + 1][..., dims], want[..., dims], mag[..., dims], kv, n, b)


def test_prefix_groups_that_decrease_stay_in_bounds(device):
    """group_starts must not decrease; one that does gives no useful rows and no fault, and
    sequences outside it are right."""
    announce("prefix decreasing groups")
    hkv, hq, d, page = 1, 4, 64, 16
    lens = [70, 80, 90, 100, 110, 60]
    pk, pv, _, table = paged(device, lens, hkv, d, page, "bf16", "split", 5)
    q = torch.randn((6, hq, d), device=device).to(torch.bfloat16)
    out = ia.shared_prefix_decode(q, pk, pv, table, i32(device, lens), i32(device, [0, 4, 2, 5, -3]),
                                  i32(device, [32, 48, 16, 64]), workspace={})
    torch.cuda.synchronize()
    n = lens[5]
    want, mag = reference(q[5:], gather(pk, None, table[5], n), gather(pv, None, table[5], n), n - 1, d ** -0.5)
    check(out[5:], want, mag, "bf16", n, "outside")


def test_prefix_batch_too_wide_for_the_held_plan(device):
    """More sequences and groups than the plan keeps in LDS: 4,500 sequences in 1,500 groups of
    three, one in nine checked against all of its tokens."""
    announce("prefix wide batch")
    hkv, hq, d, page, groups = 1, 1, 64, 16, 1500
    b = 3 * groups
    gen = torch.Generator(device=device)
    gen.manual_seed(0)
    n_pages = 64
    pk, pv = (torch.randn((n_pages, hkv, page, d), device=device, generator=gen).to(torch.bfloat16) for _ in range(2))
    lens = torch.randint(17, 40, (b,), device=device, generator=gen, dtype=torch.int32)
    table = torch.randint(0, n_pages, (b, 3), device=device, generator=gen, dtype=torch.int32)
    table[1::3, 0], table[2::3, 0] = table[::3, 0], table[::3, 0]
    q = torch.randn((b, hq, d), device=device, generator=gen).to(torch.bfloat16)
    starts = torch.arange(0, b + 1, 3, device=device, dtype=torch.int32)
    shared = torch.full((groups,), 16, device=device, dtype=torch.int32)
    out = ia.shared_prefix_decode(q, pk, pv, table, lens, starts, shared, workspace={})
    torch.cuda.synchronize()
    for i in range(0, b, 9):
        n = int(lens[i])
        want, mag = reference(q[i:i + 1], gather(pk, None, table[i], n), gather(pv, None, table[i], n), n - 1, d ** -0.5)
        check(out[i:i + 1], want, mag, "bf16", n, i)
