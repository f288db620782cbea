"""Arguments that the prompt, prefix, append and page calls refuse, each before anything is
launched (CPU only: the pointers are never followed)."""

import ctypes
import math

import pytest
import torch

import interattn_amd as ia
from interattn_amd import _native as N
from interattn_amd import pages, prompt

P = 1 << 20  # an aligned address that nothing reads


def struct(cls, base, **kw):
    s = cls(**base)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


SHAPE = dict(n_seq=2, n_tokens=40, n_q_heads=8, n_kv_heads=2, head_dim=128, q_dtype=N.IA_BF16, q_token_stride=1024,
             q_head_stride=128)
ROWS = dict(k=P, v=P, dtype=N.IA_BF16, k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128)
KV = dict(k=P, v=P, dtype=N.IA_BF16, page_size=16, n_pages=9, k_page_stride=2 * 16 * 128, k_head_stride=16 * 128,
          k_token_stride=128, v_page_stride=2 * 16 * 128, v_head_stride=16 * 128, v_token_stride=128, block_table=P,
          bt_stride=4, bt_cols=4)
DECODE = dict(batch=3, n_q_heads=8, n_kv_heads=2, head_dim=128, q_batch_stride=1024, q_row_stride=128,
              q_dtype=N.IA_BF16)
BIG = 1 << 40  # a workspace size that covers everything


def refused(rc, code, text):
    msg = N.lib().ia_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def packed_call(shape={}, rows={}, q=P, cu=P, scale=0.1, out=P, out_dtype=N.IA_BF16, ws=P, nbytes=BIG):
    return N.lib().ia_prompt_attention(struct(N.PromptShape, SHAPE, **shape), q, struct(N.PackedKV, ROWS, **rows), cu,
                                       scale, out, out_dtype, ws, nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(shape=dict(n_seq=-1)), N.IA_ERR_INVALID, "counts"),
    (dict(shape=dict(n_tokens=-3)), N.IA_ERR_INVALID, "counts"),
    (dict(shape=dict(n_q_heads=0)), N.IA_ERR_INVALID, "counts"),
    (dict(shape=dict(n_q_heads=9)), N.IA_ERR_INVALID, "multiple"),
    (dict(shape=dict(n_q_heads=130)), N.IA_ERR_UNSUPPORTED, "group"),
    (dict(shape=dict(head_dim=96)), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(shape=dict(q_dtype=N.IA_FP8_E4M3)), N.IA_ERR_INVALID, "q dtype"),
    (dict(shape=dict(q_head_stride=132)), N.IA_ERR_INVALID, "q strides"),
    (dict(shape=dict(q_token_stride=-128)), N.IA_ERR_INVALID, "q strides"),
    (dict(rows=dict(k=None)), N.IA_ERR_INVALID, "non-null"),
    (dict(rows=dict(dtype=N.IA_FP8_E4M3)), N.IA_ERR_UNSUPPORTED, "bf16 or f32"),
    (dict(rows=dict(dtype=N.IA_F32)), N.IA_ERR_UNSUPPORTED, "fp32 q"),
    (dict(rows=dict(v_head_stride=4)), N.IA_ERR_INVALID, "strides"),
    (dict(rows=dict(k_token_stride=-256)), N.IA_ERR_INVALID, "strides"),
    (dict(rows=dict(v=P + 8)), N.IA_ERR_INVALID, "aligned"),
    (dict(q=P + 2), N.IA_ERR_INVALID, "aligned"),
    (dict(q=None), N.IA_ERR_INVALID, "null"),
    (dict(cu=None), N.IA_ERR_INVALID, "null"),
    (dict(out=None), N.IA_ERR_INVALID, "null"),
    (dict(out_dtype=N.IA_FP8_E4M3), N.IA_ERR_INVALID, "out dtype"),
    (dict(scale=math.nan), N.IA_ERR_INVALID, "finite"),
    (dict(scale=-math.inf), N.IA_ERR_INVALID, "finite"),
    (dict(shape=dict(n_tokens=2000000000, n_q_heads=128, n_kv_heads=8)), N.IA_ERR_UNSUPPORTED, "launch"),
])
def test_packed(kw, code, text):
    refused(packed_call(**kw), code, text)


def test_nothing_to_do_launches_nothing():
    assert packed_call(shape=dict(n_seq=0)) == N.IA_OK
    assert packed_call(shape=dict(n_tokens=0)) == N.IA_OK


def paged_call(shape={}, kv={}, seq=P, cu=P, ws=P, nbytes=BIG):
    return N.lib().ia_paged_prompt_attention(struct(N.PromptShape, SHAPE, **shape), P, struct(N.PagedKV, KV, **kv), seq,
                                             cu, 0.1, P, N.IA_BF16, ws, nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(kv=dict(page_size=24)), N.IA_ERR_INVALID, "page_size"),
    (dict(kv=dict(page_size=0)), N.IA_ERR_INVALID, "page_size"),
    (dict(kv=dict(dtype=N.IA_FP8_E4M3)), N.IA_ERR_INVALID, "scale"),
    (dict(kv=dict(k_token_stride=64)), N.IA_ERR_INVALID, "token stride"),
    (dict(kv=dict(bt_cols=5)), N.IA_ERR_INVALID, "block table"),
    (dict(kv=dict(v=P + 4)), N.IA_ERR_INVALID, "aligned"),
    (dict(seq=None), N.IA_ERR_INVALID, "null"),
    (dict(kv=dict(bt_stride=4096, bt_cols=4096), ws=None), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(kv=dict(bt_stride=4096, bt_cols=4096), nbytes=4096), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(kv=dict(bt_stride=4096, bt_cols=4096), ws=P + 4), N.IA_ERR_WORKSPACE, "workspace"),
])
def test_paged(kw, code, text):
    refused(paged_call(**kw), code, text)


def test_prompt_workspace_is_one_size_for_every_call_that_cuts():
    lib = N.lib()
    size = lambda **kw: lib.ia_prompt_attention_workspace_size(  # noqa: E731
        struct(N.PromptShape, SHAPE, **{k: v for k, v in kw.items() if k != "keys"}), N.IA_BF16, kw.get("keys", 1 << 17))
    one = size(n_seq=1, n_tokens=1)
    assert one > 0 and size(n_seq=4, n_tokens=200) == one and size(n_seq=3, n_tokens=3) == one
    assert size(n_seq=1, n_tokens=100, keys=100) == 0 and size(n_seq=2, n_tokens=1 << 16) == 0
    assert size(n_seq=1, n_tokens=1, head_dim=64) < one and size(n_seq=1, n_tokens=1, head_dim=72) == 0


def prefix_call(shape={}, kv={}, seq=P, starts=P, shared=P, groups=1, ws=P, nbytes=BIG, scale=0.1):
    return N.lib().ia_shared_prefix_decode(struct(N.DecodeShape, DECODE, **shape), P, struct(N.PagedKV, KV, **kv), seq,
                                           starts, shared, groups, scale, P, N.IA_BF16, ws, nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(shape=dict(batch=-1)), N.IA_ERR_INVALID, "batch"),
    (dict(groups=-1), N.IA_ERR_INVALID, "groups"),
    (dict(shape=dict(n_q_heads=7)), N.IA_ERR_INVALID, "multiple"),
    (dict(shape=dict(n_q_heads=256)), N.IA_ERR_UNSUPPORTED, "group"),
    (dict(shape=dict(head_dim=32)), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(shape=dict(batch=1 << 20)), N.IA_ERR_UNSUPPORTED, "batch"),
    (dict(shape=dict(q_row_stride=4)), N.IA_ERR_INVALID, "q strides"),
    (dict(kv=dict(page_size=40)), N.IA_ERR_INVALID, "page_size"),
    (dict(kv=dict(dtype=N.IA_F32)), N.IA_ERR_UNSUPPORTED, "fp32 q"),
    (dict(seq=None), N.IA_ERR_INVALID, "null"),
    (dict(starts=None), N.IA_ERR_INVALID, "null"),
    (dict(shared=None), N.IA_ERR_INVALID, "null"),
    (dict(ws=None), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(nbytes=1000), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 16), N.IA_ERR_WORKSPACE, "workspace"),
    (dict(scale=math.inf), N.IA_ERR_INVALID, "finite"),
])
def test_prefix(kw, code, text):
    refused(prefix_call(**kw), code, text)


def test_prefix_of_no_sequence_launches_nothing():
    assert prefix_call(shape=dict(batch=0)) == N.IA_OK


def append_call(kv={}, rows={}, cu=P, seq=P, new=2 * P, n_seq=2, tokens=9, hkv=2, d=128):
    return N.lib().ia_append_prompt_kv(struct(N.PagedKV, KV, **kv), struct(N.PackedKV, ROWS, **rows), cu, seq, new, n_seq,
                                       tokens, hkv, d, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(kv=dict(dtype=N.IA_FP8_E4M3)), N.IA_ERR_UNSUPPORTED, "bf16 or f32"),
    (dict(rows=dict(dtype=N.IA_F32)), N.IA_ERR_INVALID, "dtype"),
    (dict(rows=dict(k_token_stride=2)), N.IA_ERR_INVALID, "strides"),
    (dict(rows=dict(v=None)), N.IA_ERR_INVALID, "null"),
    (dict(rows=dict(k=P + 8)), N.IA_ERR_INVALID, "aligned"),
    (dict(new=P), N.IA_ERR_INVALID, "new_seq_lens"),
    (dict(cu=None), N.IA_ERR_INVALID, "null"),
    (dict(d=80), N.IA_ERR_UNSUPPORTED, "head_dim"),
    (dict(n_seq=-1), N.IA_ERR_INVALID, "counts"),
    (dict(hkv=0), N.IA_ERR_INVALID, "counts"),
    (dict(tokens=2000000000), N.IA_ERR_UNSUPPORTED, "tokens"),
    (dict(kv=dict(k_head_stride=3)), N.IA_ERR_INVALID, "strides"),
])
def test_append(kw, code, text):
    refused(append_call(**kw), code, text)


STATE = dict(block_table=P, bt_stride=8, rows=4, cols=8, seq_lens=P, refs=P, n_pages=20, page_size=16)
TENSOR = dict(data=P, page_stride=4096, outer_stride=0, inner_stride=0, n_outer=1, n_inner=1, run_bytes=4096,
              word_bytes=16)


def tensors(**kw):
    return (N.PageTensor * 1)(struct(N.PageTensor, TENSOR, **kw))


@pytest.mark.parametrize("kw,text", [
    (dict(data=None), "non-null"), (dict(run_bytes=0), "extents"), (dict(n_outer=0), "extents"),
    (dict(page_stride=-16), "extents"), (dict(word_bytes=8), "words"), (dict(page_stride=4100), "aligned"),
    (dict(data=P + 4), "aligned"), (dict(run_bytes=1 << 30, n_inner=2, inner_stride=1 << 30), "2 GiB"),
])
def test_page_tensors(kw, text):
    lib = N.lib()
    bad = tensors(**kw)
    state = N.PageState(**STATE)
    code = N.IA_ERR_UNSUPPORTED if "GiB" in text else N.IA_ERR_INVALID
    refused(lib.ia_copy_pages(bad, 1, P, P, 1, 20, None), code, text)
    refused(lib.ia_fork_sequences(state, bad, 1, P, P, 1, P, P, BIG, None), code, text)
    refused(lib.ia_compact_pages(state, bad, 1, P, P, BIG, None), code, text)


@pytest.mark.parametrize("kw,text", [
    (dict(block_table=None), "null"), (dict(refs=None), "null"), (dict(rows=-1), "page state"),
    (dict(bt_stride=7), "page state"), (dict(page_size=0), "page state"), (dict(refs=P + 4), "16-byte"),
    (dict(n_pages=-1), "page state"),
])
def test_page_state(kw, text):
    lib = N.lib()
    bad, good = struct(N.PageState, STATE, **kw), tensors()
    refused(lib.ia_fork_sequences(bad, good, 1, P, P, 1, P, P, BIG, None), N.IA_ERR_INVALID, text)
    refused(lib.ia_free_sequences(bad, P, 1, None), N.IA_ERR_INVALID, text)
    refused(lib.ia_reserve_pages(bad, P, P, P, BIG, None), N.IA_ERR_INVALID, text)
    refused(lib.ia_compact_pages(bad, good, 1, P, P, BIG, None), N.IA_ERR_INVALID, text)


def test_page_lists_and_workspaces():
    lib = N.lib()
    state, good = N.PageState(**STATE), tensors()
    refused(lib.ia_copy_pages(good, 1, None, P, 3, 20, None), N.IA_ERR_INVALID, "page lists")
    refused(lib.ia_copy_pages(good, 1, P, P, -1, 20, None), N.IA_ERR_INVALID, "page lists")
    refused(lib.ia_copy_pages(None, 1, P, P, 3, 20, None), N.IA_ERR_INVALID, "page tensors")
    assert lib.ia_copy_pages(good, 1, P, P, 0, 20, None) == N.IA_OK
    refused(lib.ia_fork_sequences(state, good, 1, P, P, 8193, P, P, BIG, None), N.IA_ERR_INVALID, "fork lists")
    refused(lib.ia_fork_sequences(state, good, 1, P, P, 2, None, P, BIG, None), N.IA_ERR_INVALID, "fork lists")
    refused(lib.ia_fork_sequences(state, good, 1, P, P, 2, P, P, 23, None), N.IA_ERR_WORKSPACE, "workspace")
    refused(lib.ia_fork_sequences(state, good, 1, P, P, 2, P, None, BIG, None), N.IA_ERR_WORKSPACE, "workspace")
    assert lib.ia_fork_sequences(state, good, 1, P, P, 0, P, None, 0, None) == N.IA_OK
    refused(lib.ia_free_sequences(state, None, 2, None), N.IA_ERR_INVALID, "row list")
    assert lib.ia_free_sequences(state, None, 0, None) == N.IA_OK
    refused(lib.ia_reserve_pages(state, None, P, P, BIG, None), N.IA_ERR_INVALID, "null")
    refused(lib.ia_reserve_pages(state, P, P, P, 8, None), N.IA_ERR_WORKSPACE, "workspace")
    refused(lib.ia_compact_pages(state, good, 1, None, P, BIG, None), N.IA_ERR_INVALID, "null")
    refused(lib.ia_compact_pages(state, good, 1, P, P, 8, None), N.IA_ERR_WORKSPACE, "workspace")


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8, 64)
    cu = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        ia.prompt_attention(x, x, x, cu)
    with pytest.raises(ValueError, match="device"):
        ia.paged_prompt_attention(x, x[None], x[None], table, cu[:1], cu)
    with pytest.raises(ValueError, match="device"):
        ia.shared_prefix_decode(x, x[None], x[None], table, cu[:1], cu, cu[:1])
    with pytest.raises(ValueError, match="device"):
        ia.append_prompt_kv(x[None], x[None], table, cu[:1], x, x, cu)
    for call in (lambda: ia.copy_pages([x], cu, cu), lambda: ia.free_sequences(table, cu[:1], cu, cu),
                 lambda: ia.fork_sequences([x], table, cu[:1], cu, cu, cu, page_size=16),
                 lambda: ia.reserve_pages(table, cu[:1], cu, cu[:1], page_size=16),
                 lambda: ia.compact_pages([x], table, cu)):
        with pytest.raises(ValueError, match="device"):
            call()


def test_page_layouts():
    lay = lambda t: pages._page_layout(t.shape, t.stride(), t.element_size())  # noqa: E731
    pool = torch.empty(5, 8, 16, 128, dtype=torch.bfloat16)
    assert lay(pool) == (32768, 0, 0, 1, 1, 32768, 16)
    assert lay(torch.empty(5, 8, 2, 16, 128, dtype=torch.bfloat16)[:, :, 1]) == (65536, 0, 8192, 1, 8, 4096, 16)
    assert lay(torch.empty(5, 16, 8, 128, dtype=torch.bfloat16).permute(0, 2, 1, 3)) == (32768, 0, 0, 1, 1, 32768, 16)
    assert lay(torch.empty(5, 4, 16, 3, 64)[..., 1, :]) == (4 * 16 * 3 * 256, 0, 768, 1, 64, 256, 16)
    assert lay(torch.empty(5, 3)) == (12, 0, 0, 1, 1, 12, 4)
    assert lay(torch.empty(1, 1, 1, 4)) == (16, 0, 0, 1, 1, 16, 16)
    for bad in (pool[:, :1].expand(5, 8, 16, 128), torch.empty(5, 3, dtype=torch.bfloat16), torch.empty(5, 0),
                torch.empty(5, 4, 3, 4, 3, 4, 64)[:, :, 0, :, 0, :, :32][:, :, :, :2],
                torch.empty(1, 8, 16).expand(5, 8, 16)):
        with pytest.raises(ValueError):
            lay(bad)


def test_row_layouts():
    q = torch.empty(10, 8, 128, dtype=torch.bfloat16)
    s = N.PromptShape.from_buffer_copy(prompt._q_layout(q.shape[1:], q.stride(), q.dtype, 2, 128))
    assert (s.n_q_heads, s.n_kv_heads, s.head_dim, s.q_token_stride, s.q_head_stride) == (8, 2, 128, 1024, 128)
    for heads, stride, dtype, hkv, d in (((8, 128), (1024, 128, 2), q.dtype, 2, 128), ((8,), (8, 1), q.dtype, 2, 128),
                                         ((8, 128), (1024, 128, 1), torch.float16, 2, 128),
                                         ((8, 128), (1024, 128, 1), q.dtype, 3, 128),
                                         ((8, 128), (1024, 128, 1), q.dtype, 2, 64)):
        with pytest.raises(ValueError):
            prompt._q_layout(torch.Size(heads), stride, dtype, hkv, d)
    ok = (torch.Size((2, 64)), (128, 64, 1), torch.float32)
    assert ctypes.sizeof(N.PackedKV) == len(prompt._row_layout(*ok, *ok)[0])
    for other in ((torch.Size((3, 64)), (128, 64, 1), torch.float32), (torch.Size((2, 64)), (128, 64, 2), torch.float32),
                  (torch.Size((2, 64)), (128, 64, 1), torch.bfloat16)):
        with pytest.raises(ValueError):
            prompt._row_layout(*ok, *other)


def test_struct_layouts():
    assert ctypes.sizeof(N.PromptShape) == 4 * 6 + 8 * 2
    assert ctypes.sizeof(N.PackedKV) == 8 * 2 + 8 + 8 * 4
    assert ctypes.sizeof(N.PageTensor) == 8 * 4 + 4 * 4
    assert ctypes.sizeof(N.PageState) == 8 * 2 + 4 * 2 + 8 * 2 + 8 + 8
