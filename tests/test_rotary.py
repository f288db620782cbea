"""Frequencies of rotary positions, the oracles of the serving step, and refusals (CPU only:
pointers are never followed)."""

import ctypes
import math

import numpy as np
import pytest
import torch

import interattn_amd as ia
from interattn_amd import _native as N
from interattn_amd import beam, rotary
from oracle import beam as OB
from oracle import quantise as Q
from oracle import rotary as R

P = 1 << 20  # an aligned address that nothing reads


# ------------------------------------------------------------------ frequencies

def config(dim, base, scaling):
    from transformers import LlamaConfig

    return LlamaConfig(hidden_size=dim * 4, num_attention_heads=4, head_dim=dim, max_position_embeddings=131072,
                       rope_parameters=dict(rope_theta=base, **scaling))


@pytest.mark.parametrize("dim,base,scaling", [
    (128, 10000.0, dict(rope_type="linear", factor=4.0)),
    (64, 500000.0, dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, low_freq_factor=1.0,
                        high_freq_factor=4.0)),
    (128, 500000.0, dict(rope_type="llama3", factor=32.0, original_max_position_embeddings=4096, low_freq_factor=2.0,
                         high_freq_factor=3.0)),
    (128, 10000.0, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)),
    (64, 1e6, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768, beta_fast=16.0, beta_slow=2.0,
                   truncate=False)),
    (64, 10000.0, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=2048, attention_factor=1.25)),
])
def test_frequencies_are_a_model_configs(dim, base, scaling):
    """Against the functions that models of this config use, which compute in float32: every
    frequency within a few roundings of 2^-24 (powers amplify one of the exponent: ln base of
    them)."""
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    want, factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](config(dim, base, scaling), torch.device("cpu"))
    got, got_factor = ia.rotary_frequencies(dim, base=base, scaling=scaling)
    bar = (8 + 2 * math.log(base)) * 2.0 ** -24
    # (llama3 blends two terms whose weights are themselves differences)
    bar *= 16 if scaling["rope_type"] == "llama3" else 4
    assert len(got) == dim // 2
    assert max(abs(a - float(b)) / float(b) for a, b in zip(got, want)) <= bar
    assert abs(got_factor - factor) <= 2.0 ** -40 * factor


def test_plain_frequencies():
    w, f = ia.rotary_frequencies(8, base=100.0)
    assert f == 1.0 and np.allclose(w, [1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    assert ia.rotary_frequencies(8, base=100.0, scaling={"rope_type": "default"})[0] == w
    assert ia.rotary_frequencies(0) == ([], 1.0)


def test_turns_are_whole_numbers_of_the_circle():
    """2^-64 of a turn: what a float64 frequency holds, for any sign and size."""
    w = [1.0, 1e-6, 2 * math.pi * 0.75, -0.5, 7.0]
    plan = ia.rotary_plan(10, inv_freq=w, device="cpu")
    for x, t in zip(w, plan.turns.tolist()):
        want = math.fmod(x / (2 * math.pi), 1.0) % 1.0
        got = (t % (1 << 64)) / 2.0 ** 64
        assert min(abs(got - want), 1 - abs(got - want)) <= 2.0 ** -53
    assert plan.dim == 10 and plan.layout == "half" and plan.factor == 1.0
    assert ia.rotary_plan(10, inv_freq=torch.tensor(w, dtype=torch.float64), device="cpu").turns.equal(plan.turns)
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=100)
    assert ia.rotary_plan(8, scaling=yarn, device="cpu").factor == pytest.approx(0.1 * math.log(4) + 1)
    assert ia.rotary_plan(8, scaling=yarn, factor=2.0, device="cpu").factor == 2.0


def test_base_may_stand_in_the_scaling():
    theta = {"rope_type": "default", "rope_theta": 500000.0}
    want = ia.rotary_frequencies(16, base=500000.0)
    assert ia.rotary_frequencies(16, scaling=theta) == want == ia.rotary_frequencies(16, base=500000, scaling=theta)
    assert ia.rotary_frequencies(16) == ia.rotary_frequencies(16, base=10000.0)
    assert ia.rotary_frequencies(16, scaling={"rope_type": "linear", "factor": 2.0, "rope_theta": 500000.0})[0] \
        == [x / 2 for x in want[0]]


@pytest.mark.parametrize("kw,text", [
    (dict(dim=7), "even"),
    (dict(dim=8, base=10000.0, scaling={"rope_type": "default", "rope_theta": 500000.0}), "rope_theta"),
    (dict(dim=8, scaling={"rope_type": "default", "factor": 2.0}), "factor"),
    (dict(dim=8, base=math.inf), "base"),
    (dict(dim=4, base=100.0, inv_freq=[1.0, 2.0]), "inv_freq"),
    (dict(dim=4, base=1.0, scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64}), "above 1"),
    (dict(dim=-2), "even"),
    (dict(dim=8, base=0.0), "base"),
    (dict(dim=8, layout="columns"), "layout"),
    (dict(dim=8, inv_freq=[1.0, 2.0]), "each of dim"),
    (dict(dim=4, inv_freq=[1.0, math.inf]), "finite"),
    (dict(dim=4, factor=math.nan), "finite"),
    (dict(dim=4, inv_freq=[1.0, 2.0], scaling={"rope_type": "linear", "factor": 2.0}), "inv_freq"),
    (dict(dim=4, scaling={"rope_type": "dynamic", "factor": 2.0}), "unknown rope_type"),
    (dict(dim=4, scaling={"rope_type": "linear"}), "factor"),
    (dict(dim=4, scaling={"rope_type": "linear", "factor": -1.0}), "positive"),
    (dict(dim=4, scaling={"rope_type": "yarn", "factor": 2.0}), "original_max"),
    (dict(dim=4, scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64, "mscale": 1.0}),
     "mscale"),
    (dict(dim=4, scaling={"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 64,
                          "low_freq_factor": 4.0, "high_freq_factor": 4.0}), "above"),
])
def test_plans_refuse(kw, text):
    with pytest.raises(ValueError, match=text):
        ia.rotary_plan(kw.pop("dim"), device="cpu", **kw)


# ------------------------------------------------------------------ oracles

def test_oracle_codes_are_torchs():
    """Every code, every midpoint and its neighbours, against torch's own conversion."""
    v = Q.VALUES[:0x7F]
    mids = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mids, np.nextafter(mids, 0).astype(np.float32), np.nextafter(mids.astype(np.float32), np.float32(1e9)),
                        [0.0, 2.0 ** -11, 2.0 ** -10, 2.0 ** -10 * 1.0001, 448.0, 460.0]]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(Q.encode(x), want)
    assert np.array_equal(np.nan_to_num(Q.VALUES, nan=-1.0),
                          np.nan_to_num(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy(),
                                        nan=-1.0))
    assert Q.encode([np.nan, np.inf, -np.inf]).tolist() == [0x7F] * 3


def test_oracle_scales():
    for a, s in ((0.0, 2.0 ** -126), (1e-40, 2.0 ** -126), (448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (1.75, 2.0 ** -8),
                 (3.4e38, 2.0 ** 120)):
        assert Q.page_scale(a) == s


def test_oracle_rotation_turns_back():
    rng = np.random.default_rng(0)
    x, pos = rng.standard_normal((5, 2, 16)), rng.integers(-1000, 1000, 5)
    w = rng.random(6)
    for layout in ("half", "interleaved"):
        y = R.turn(x, pos, w, layout, 2.0)
        assert np.allclose(R.turn(y, pos, w, layout, 0.5, inverse=True), x)
        assert np.array_equal(y[..., 12:], x[..., 12:])
        assert np.allclose(R.turn(x, pos * 0, w, layout), x)


def test_oracle_reorder_keeps_counts():
    rng = np.random.default_rng(1)
    for _ in range(50):
        rows, cols, page = int(rng.integers(1, 7)), int(rng.integers(1, 6)), 16
        n_pages = rows * cols + 8
        table, at = np.full((rows, cols), -1, np.int32), 0
        lens = rng.integers(0, cols * page + 1, rows).astype(np.int32)
        for i in range(rows):
            n = -(-int(lens[i]) // page)
            table[i, :n] = np.arange(at, at + n)
            at += n
        refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
        parents = rng.integers(-1, rows, rows).astype(np.int32)
        new, new_len, new_refs, ok, copies = OB.reorder(table, lens, refs, parents, page)
        assert np.array_equal(new_refs, np.bincount(new[new >= 0], minlength=n_pages)) and ok.all()
        for i, p in enumerate(parents):
            assert new_len[i] == (lens[p] if p >= 0 else 0)
            assert (new[i, :-(-int(new_len[i]) // page)] >= 0).all()
        assert all(new_refs[a] >= 1 and new_refs[b] == 1 for a, b in copies)


# ------------------------------------------------------------------ refusals

def struct(cls, base, **kw):
    s = cls(**base)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def refused(rc, code, text):
    msg = N.lib().ia_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


ROT = dict(turns=P, dim=128, interleaved=0, factor=1.0)
TURN = dict(in_=P, out=P, in_token_stride=1024, in_head_stride=128, out_token_stride=1024, out_head_stride=128, n_heads=8)
ROWS = dict(k=P, v=P, dtype=N.IA_BF16, k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128)
KV = dict(k=P, v=P, dtype=N.IA_BF16, page_size=16, n_pages=9, k_page_stride=2 * 16 * 128, k_head_stride=16 * 128,
          k_token_stride=128, v_page_stride=2 * 16 * 128, v_head_stride=16 * 128, v_token_stride=128, block_table=P,
          bt_stride=4, bt_cols=4)
FP8 = dict(KV, dtype=N.IA_FP8_E4M3, k_scale=P, v_scale=P, scale_page_stride=2)


def turn_call(rot={}, rows={}, n_tensors=1, dtype=N.IA_BF16, d=128, pos=P, tokens=5):
    arr = (N.RotaryRows * 2)(struct(N.RotaryRows, TURN, **rows), struct(N.RotaryRows, TURN))
    return N.lib().ia_apply_rotary(struct(N.Rotary, ROT, **rot), arr, n_tensors, dtype, d, pos, tokens, 0, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=N.IA_FP8_E4M3), N.IA_ERR_UNSUPPORTED, "bf16 or f32"),
    (dict(d=100), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(d=272), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(rot=dict(dim=130)), N.IA_ERR_INVALID, "at most head_dim"),
    (dict(rot=dict(dim=63)), N.IA_ERR_INVALID, "even"),
    (dict(rot=dict(turns=None)), N.IA_ERR_INVALID, "turns"),
    (dict(rot=dict(factor=math.inf)), N.IA_ERR_INVALID, "finite"),
    (dict(n_tensors=0), N.IA_ERR_INVALID, "row tensors"),
    (dict(tokens=-1), N.IA_ERR_INVALID, "tokens"),
    (dict(pos=None), N.IA_ERR_INVALID, "null"),
    (dict(rows=dict(in_=None)), N.IA_ERR_INVALID, "null"),
    (dict(rows=dict(out_token_stride=-1024)), N.IA_ERR_INVALID, "strides"),
    (dict(rows=dict(in_head_stride=132)), N.IA_ERR_INVALID, "strides"),
    (dict(rows=dict(out=P + 8)), N.IA_ERR_INVALID, "aligned"),
])
def test_apply_rotary_refuses(kw, code, text):
    refused(turn_call(**kw), code, text)


def test_apply_rotary_of_nothing():
    assert turn_call(tokens=0) == N.IA_OK
    assert turn_call(rows=dict(n_heads=0)) == N.IA_OK


def write_call(rot={}, q={}, rows={}, kv={}, base=KV, cu=P, lens=P, new=P + 4096, pos=None, n_seq=2, tokens=40, hkv=2,
               d=128, with_q=True):
    return N.lib().ia_rotary_append_kv(
        struct(N.Rotary, ROT, **rot), struct(N.RotaryRows, TURN, **q) if with_q else None,
        struct(N.PackedKV, ROWS, **rows), struct(N.PagedKV, base, **kv), cu, lens, new, pos, n_seq, tokens, hkv, d, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(lens=None), N.IA_ERR_INVALID, "null"),
    (dict(d=96), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(kv=dict(page_size=24)), N.IA_ERR_INVALID, "page_size"),
    (dict(rot=dict(dim=129)), N.IA_ERR_INVALID, "rotary"),
    (dict(rows=dict(dtype=N.IA_FP8_E4M3)), N.IA_ERR_INVALID, "f32 or bf16"),
    (dict(rows=dict(dtype=N.IA_F32)), N.IA_ERR_INVALID, "pool's dtype"),
    (dict(base=FP8, kv=dict(k_scale=None)), N.IA_ERR_INVALID, "k_scale"),
    (dict(base=FP8, kv=dict(scale_page_stride=1)), N.IA_ERR_INVALID, "scales of its own"),
    (dict(base=FP8, kv=dict(seq_scale=P)), N.IA_ERR_INVALID, "per sequence"),
    (dict(hkv=0), N.IA_ERR_INVALID, "counts"),
    (dict(tokens=-1), N.IA_ERR_INVALID, "counts"),
    (dict(rows=dict(v=None)), N.IA_ERR_INVALID, "null"),
    (dict(rows=dict(v=P + 2)), N.IA_ERR_INVALID, "aligned"),
    (dict(rows=dict(k_head_stride=4)), N.IA_ERR_INVALID, "strides"),
    (dict(cu=None), N.IA_ERR_INVALID, "one token"),
    (dict(new=P), N.IA_ERR_INVALID, "in place"),
    (dict(q=dict(n_heads=7)), N.IA_ERR_INVALID, "multiple"),
    (dict(q=dict(out=None)), N.IA_ERR_INVALID, "null"),
    (dict(q=dict(in_token_stride=4)), N.IA_ERR_INVALID, "strides"),
    (dict(q=dict(in_=P + 4)), N.IA_ERR_INVALID, "aligned"),
    (dict(n_seq=1 << 23, tokens=1 << 23, cu=None), N.IA_ERR_UNSUPPORTED, "too many"),
])
def test_write_refuses(kw, code, text):
    refused(write_call(**kw), code, text)


def test_write_and_read_of_nothing():
    assert write_call(n_seq=0, tokens=0, lens=None, new=None) == N.IA_OK
    kv = N.PagedKV(**KV)
    assert N.lib().ia_read_kv(kv, None, None, N.IA_BF16, None, None, 0, 0, 2, 128, None) == N.IA_OK


@pytest.mark.parametrize("args,code,text", [
    ((dict(), P, P, N.IA_FP8_E4M3, P, P, 2, 9, 2, 128), N.IA_ERR_INVALID, "out dtype"),
    ((dict(), P, P, N.IA_BF16, P, P, 2, 9, 2, 80), N.IA_ERR_UNSUPPORTED, "head_dim"),
    ((dict(), P, P, N.IA_BF16, P, P, -2, 9, 2, 128), N.IA_ERR_INVALID, "counts"),
    ((dict(), None, P, N.IA_BF16, P, P, 2, 9, 2, 128), N.IA_ERR_INVALID, "null"),
    ((dict(), P, P + 8, N.IA_BF16, P, P, 2, 9, 2, 128), N.IA_ERR_INVALID, "aligned"),
    ((dict(page_size=0), P, P, N.IA_BF16, P, P, 2, 9, 2, 128), N.IA_ERR_INVALID, "page_size"),
])
def test_read_refuses(args, code, text):
    refused(N.lib().ia_read_kv(struct(N.PagedKV, KV, **args[0]), *args[1:], None), code, text)


BIG = 1 << 40


def beam_call(dtype=N.IA_BF16, stride=1000, logits=P, scores=P, pad=0, batch=2, beams=4, vocab=1000, n=8, out=P, ws=P,
              nbytes=BIG):
    return N.lib().ia_beam_select(logits, dtype, stride, scores, None, pad, batch, beams, vocab, n, out, out, out, ws,
                                  nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=N.IA_FP8_E4M3), N.IA_ERR_UNSUPPORTED, "bf16 or f32"),
    (dict(beams=0), N.IA_ERR_INVALID, "beams"),
    (dict(beams=65), N.IA_ERR_INVALID, "beams"),
    (dict(n=65), N.IA_ERR_INVALID, "best"),
    (dict(n=0), N.IA_ERR_INVALID, "best"),
    (dict(vocab=1, n=5), N.IA_ERR_INVALID, "candidates"),
    (dict(batch=-1), N.IA_ERR_INVALID, "beams"),
    (dict(scores=None), N.IA_ERR_INVALID, "null"),
    (dict(stride=-5), N.IA_ERR_INVALID, "stride"),
    (dict(pad=1000), N.IA_ERR_INVALID, "pad_token"),
    (dict(logits=P + 1), N.IA_ERR_INVALID, "aligned"),
    (dict(nbytes=16), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 4), N.IA_ERR_WORKSPACE, "workspace"),
])
def test_beam_select_refuses(kw, code, text):
    refused(beam_call(**kw), code, text)


def test_beam_select_of_nothing_and_its_workspace():
    assert beam_call(batch=0) == N.IA_OK
    size = N.lib().ia_beam_select_workspace_size
    assert size(1, 65, 100, 4, N.IA_F32) == size(1, 4, 100, 65, N.IA_F32) == 0
    assert 0 < size(1, 4, 32000, 8, N.IA_F32) <= size(4, 4, 32000, 8, N.IA_F32)
    # (a launch holds 2^32 threads)
    assert size(1 << 20, 16, 1000, 4, N.IA_F32) > 0 == size(1 << 20, 17, 1000, 4, N.IA_F32)


STATE = dict(block_table=P, bt_stride=4, rows=3, cols=4, seq_lens=P, refs=P, n_pages=20, page_size=16)


def reorder_call(state={}, tensor=None, parents=P, ok=P, ws=P, nbytes=BIG):
    t = None if tensor is None else (N.PageTensor * 1)(tensor)
    return N.lib().ia_reorder_sequences(struct(N.PageState, STATE, **state), t, 0 if tensor is None else 1, parents, ok,
                                        ws, nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(parents=None), N.IA_ERR_INVALID, "null"),
    (dict(ok=None), N.IA_ERR_INVALID, "null"),
    (dict(state=dict(seq_lens=None)), N.IA_ERR_INVALID, "null"),
    (dict(state=dict(rows=8193)), N.IA_ERR_UNSUPPORTED, "8192"),
    (dict(state=dict(page_size=0)), N.IA_ERR_INVALID, "page_size"),
    (dict(state=dict(rows=8192, cols=1 << 22, bt_stride=1 << 22), nbytes=1 << 40), N.IA_ERR_UNSUPPORTED, "columns"),
    (dict(tensor=N.PageTensor(None, 64, 0, 0, 1, 1, 64, 16)), N.IA_ERR_INVALID, "non-null"),
    (dict(nbytes=8), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(ws=None), N.IA_ERR_WORKSPACE, "workspace"),
])
def test_reorder_refuses(kw, code, text):
    refused(reorder_call(**kw), code, text)


def test_reorder_of_no_rows():
    assert reorder_call(state=dict(rows=0), ws=None, nbytes=0) == N.IA_OK


def test_host_tensors_are_refused():
    x = torch.zeros((4, 2, 64))
    i = torch.zeros(4, dtype=torch.int32)
    plan = ia.rotary_plan(64, device="cpu")
    pool, table = torch.zeros((9, 2, 16, 64)), torch.zeros((4, 2), dtype=torch.int32)
    calls = [lambda: ia.apply_rotary(x, x, i, plan), lambda: ia.rotary_append_kv(x, x, x, plan, pool, pool, table, i),
             lambda: ia.read_kv(pool, pool, table, i, torch.zeros(5, dtype=torch.int32), 4),
             lambda: ia.beam_select(torch.zeros((4, 9)), torch.zeros((2, 2))),
             lambda: ia.reorder_sequences([pool], table, i, torch.zeros(9, dtype=torch.int32), i, page_size=16)]
    for call in calls:
        with pytest.raises(ValueError, match="device"):
            call()


def test_row_layouts():
    x = torch.empty((5, 8, 128), dtype=torch.bfloat16)
    assert rotary._heads(x.shape[1:], x.stride(), x.dtype, "q") == (8, 128, 1024, 128)
    one = torch.empty((5, 1, 128), dtype=torch.bfloat16)
    assert rotary._heads(one.shape[1:], one.stride(), one.dtype, "q")[3] == 0
    for bad in (x.transpose(1, 2), x.half(), x[0]):
        with pytest.raises(ValueError):
            rotary._heads(bad.shape[1:], bad.stride(), bad.dtype, "q")


def test_struct_layouts():
    assert ctypes.sizeof(N.Rotary) == 8 + 3 * 4 + 4
    assert ctypes.sizeof(N.RotaryRows) == 2 * 8 + 4 * 8 + 4 + 4
    assert beam.MAX_BEAMS == beam.MAX_BEST == 64
