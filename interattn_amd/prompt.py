"""Prompt attention: causal attention of packed prompts, over their own K/V or over a
paged pool that holds them.

Packed rows put the sequences of a batch one behind the other with no padding:
``cu_seqlens [n_seq + 1] int32`` on the device holds the first row of each, and the end of
the last.  Pools, block tables and scales are those of ``ops``.  Calls launch on the
current stream of their tensors' device, never synchronise, and keep scratch in the caller's
``workspace`` dict; calls that share one must not overlap.  An output is a new tensor unless
``out`` is given: batches differ from call to call, and a kept buffer of another size would
be replaced under a captured graph that writes it.
"""

import functools

import torch

from . import _native as N
from .ops import _DTYPE_CODE, _code, _stream, paged_kv, workspace_tensor

_F32, _BF16 = torch.float32, torch.bfloat16


def device_of(ref, *others):
    """``ref``'s GPU, which has to hold every other tensor too (a kernel reads them there)."""
    dev = ref.get_device()
    if dev < 0:
        raise ValueError("interattn_amd kernels need device (cuda) tensors")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on {ref.device}, got one on {t.device}")
    return dev


def check_ints(t, name, length=None):
    """A contiguous int32 vector; returns its length."""
    if t.dtype != torch.int32 or t.dim() != 1:
        raise ValueError(f"{name} must be a contiguous int32 vector")
    n = t.shape[0]
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be a contiguous int32 vector")
    if length is not None and n != length:
        raise ValueError(f"{name} must have {length} entries, got {n}")
    return n


def launch(fn, ref, *args):
    """Call an entry point on the current stream of ``ref``'s device, with it current."""
    if torch.cuda.current_device() == ref.get_device():
        N.check(fn(*args, _stream(ref)))
    else:
        with torch.cuda.device(ref.device):
            N.check(fn(*args, _stream(ref)))


# What follows from shapes, strides and types alone is checked once per combination and kept
# as the bytes of the C struct, pointers and row counts left out; nothing is kept of a
# tensor.  That is a third of a call's host time up to the launch (an append on an 8-core
# EPYC host: 21.3 -> 14.0 us).

@functools.lru_cache(maxsize=1024)
def _q_layout(heads, stride, dtype, hkv, d):
    """``PromptShape`` bytes of packed query rows."""
    if len(heads) != 2 or (heads[1] > 1 and stride[2] != 1):
        raise ValueError("q must be [tokens, n_q_heads, D] with contiguous rows")
    if dtype not in (_F32, _BF16):
        raise ValueError("q must be float32 or bfloat16")
    if heads[1] != d:
        raise ValueError("q and the keys disagree on head_dim")
    if hkv <= 0 or heads[0] <= 0 or heads[0] % hkv:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads (grouped query attention)")
    return bytes(N.PromptShape(0, 0, heads[0], hkv, d, _DTYPE_CODE[dtype], stride[0],
                               stride[1] if heads[0] > 1 else 0))


def _prompt_shape(q, n_seq, hkv, d):
    rows = q.shape
    shape = N.PromptShape.from_buffer_copy(_q_layout(rows[1:], q.stride(), q.dtype, hkv, d))
    tokens = rows[0]
    shape.n_seq, shape.n_tokens = n_seq, tokens
    if tokens <= 1:
        shape.q_token_stride = 0  # (any stride means nothing then)
    return shape


@functools.lru_cache(maxsize=1024)
def _row_layout(k_heads, k_stride, k_dtype, v_heads, v_stride, v_dtype):
    """``(PackedKV bytes, n_kv_heads, D)`` of packed K and V rows."""
    if len(k_heads) != 2 or k_heads != v_heads:
        raise ValueError("k and v must both be [tokens, n_kv_heads, D]")
    if k_stride[2] != 1 or v_stride[2] != 1 or k_dtype != v_dtype:
        raise ValueError("k and v must share a dtype and have contiguous rows")
    one = k_heads[0] <= 1
    return bytes(N.PackedKV(None, None, _code(k_dtype, "k and v"), k_stride[0], 0 if one else k_stride[1], v_stride[0],
                            0 if one else v_stride[1])), k_heads[0], k_heads[1]


def _packed_rows(k, v):
    """``(PackedKV, tokens, n_kv_heads, D)``."""
    ks, vs = k.shape, v.shape
    held, hkv, d = _row_layout(ks[1:], k.stride(), k.dtype, vs[1:], v.stride(), v.dtype)
    tokens = ks[0]
    if vs[0] != tokens:
        raise ValueError("k and v must have the same tokens")
    rows = N.PackedKV.from_buffer_copy(held)
    rows.k, rows.v = k.data_ptr(), v.data_ptr()
    if tokens <= 1:
        rows.k_token_stride = rows.v_token_stride = 0
    return rows, tokens, hkv, d


_POOLS = {}  # layouts of pools -> (PagedKV bytes, n_kv_heads, D)


def _pool(pool_k, pool_v, block_table, scales, n_seq):
    """``(PagedKV, n_kv_heads, D)``: ``ops.paged_kv``'s struct, its table of ``n_seq`` rows."""
    key = [pool_k.shape, pool_k.stride(), pool_k.dtype, pool_v.shape, pool_v.stride(), pool_v.dtype]
    if block_table is not None:
        rows = block_table.shape
        if rows[0] != n_seq:
            raise ValueError("block_table must have a row for each sequence")
        key += (rows, block_table.stride(), block_table.dtype)
    ks = vs = None
    if scales is not None:
        ks, vs = scales[:2]
        key += (ks.shape, ks.stride(), ks.dtype, vs.shape, vs.stride(), vs.dtype)
    key = tuple(key)
    held = _POOLS.get(key)
    if held is None:
        kv, _ = paged_kv(pool_k, pool_v, block_table, scales if ks is None else (ks, vs))
        kv.k = kv.v = kv.block_table = kv.k_scale = kv.v_scale = None
        if len(_POOLS) >= 1024:
            _POOLS.clear()
        held = _POOLS[key] = bytes(kv), pool_k.shape[1], pool_k.shape[3]
    held, hkv, d = held
    kv = N.PagedKV.from_buffer_copy(held)
    kv.k, kv.v = pool_k.data_ptr(), pool_v.data_ptr()
    if block_table is not None:
        # (one of no columns has no address; null would be the identity table)
        kv.block_table = block_table.data_ptr() or kv.k
    if kv.dtype == N.IA_FP8_E4M3:
        kv.k_scale, kv.v_scale = ks.data_ptr(), vs.data_ptr()
    return kv, hkv, d


def output(q, out, out_dtype):
    """The caller's ``out`` or a new tensor, ``q``'s shape, contiguous."""
    if out is None:
        return torch.empty(q.shape, device=q.device, dtype=out_dtype or q.dtype)
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {list(q.shape)} tensor")
    if out.dtype not in (_F32, _BF16) or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("out must be float32 or bfloat16, of out_dtype where that is given")
    device_of(q, out)
    return out


def _n_seq(cu_seqlens):
    n = check_ints(cu_seqlens, "cu_seqlens") - 1
    if n < 0:
        raise ValueError("cu_seqlens must have n_seq + 1 entries")
    return n


def _workspace(shape, kv_dtype, max_keys, workspace, device):
    """The partials' buffer of a call that cuts its keys: one size per device, type and head
    size, so that a later call never replaces a buffer that a captured graph uses."""
    need = N.lib().ia_prompt_attention_workspace_size(shape, kv_dtype, max_keys)
    if not need:
        return None
    return workspace_tensor(workspace, ("prompt_scratch", kv_dtype, shape.head_dim), (need,), device=device,
                            dtype=torch.uint8)


def prompt_attention(q, k, v, cu_seqlens, *, scale=None, out=None, out_dtype=None, workspace=None):
    """Causal attention of packed prompts: ``q [tokens, Hq, D]``, ``k, v [tokens, Hkv, D]``
    (any token and head strides of 16-byte multiples with contiguous rows: views of one
    fused projection need no copy), the query heads of a kv head neighbours.  Token i of a
    sequence attends tokens 0..i of it, softmax in float32.  ``k, v`` bf16 or float32 (then
    ``q`` too; over bf16 a float32 ``q`` is rounded to bf16).  Returns ``[tokens, Hq, D]`` of ``out_dtype`` (``q``'s by default); rows of
    no sequence are left as ``out`` had them.  The prompt side of the paged decode calls,
    and what ``_sdpa_prefill_attention_forward`` (CBT/core.py:1180-1200) computes, without
    padding.  Forward only."""
    device_of(q, k, v, cu_seqlens)
    kv, tokens, hkv, d = _packed_rows(k, v)
    shape = _prompt_shape(q, _n_seq(cu_seqlens), hkv, d)
    if shape.n_tokens != tokens:
        raise ValueError("k and v must have q's tokens")
    out = output(q, out, out_dtype)
    if tokens == 0:
        return out
    ws = _workspace(shape, kv.dtype, tokens, workspace, q.device)
    launch(N.lib().ia_prompt_attention, q, shape, q.data_ptr(), kv, cu_seqlens.data_ptr(),
           d ** -0.5 if scale is None else float(scale), out.data_ptr(), _DTYPE_CODE[out.dtype],
           *((None, 0) if ws is None else (ws.data_ptr(), ws.numel())))
    return out


def paged_prompt_attention(q, pool_k, pool_v, block_table, seq_lens, cu_seqlens, *, scale=None, scales=None, out=None,
                           out_dtype=None, workspace=None):
    """Causal attention of each sequence's newest tokens over all of it in the paged pool:
    ``q [tokens, Hq, D]`` packs the last ``cu_seqlens[b + 1] - cu_seqlens[b]`` tokens of
    sequence b, which has ``seq_lens[b]`` tokens in the pool, the new ones among them
    (``append_prompt_kv`` writes them).  A chunk of a long prompt, a prompt behind a cached
    prefix and a single token are the same call; bf16, float32 and fp8 pools
    (``scales=(k_scale, v_scale)``).  Returns ``[tokens, Hq, D]``; rows of no sequence are
    left as ``out`` had them, a row that sees no key is zeros.  Forward only."""
    device_of(q, pool_k, pool_v, block_table, seq_lens, cu_seqlens, *(scales or ()))
    n_seq = _n_seq(cu_seqlens)
    kv, hkv, d = _pool(pool_k, pool_v, block_table, scales, n_seq)
    shape = _prompt_shape(q, n_seq, hkv, d)
    check_ints(seq_lens, "seq_lens", n_seq)
    out = output(q, out, out_dtype)
    if shape.n_tokens == 0:
        return out
    cap = (kv.bt_cols if block_table is not None else kv.n_pages) * kv.page_size
    ws = _workspace(shape, kv.dtype, min(cap, (1 << 31) - 1025), workspace, q.device)
    launch(N.lib().ia_paged_prompt_attention, q, shape, q.data_ptr(), kv, seq_lens.data_ptr(), cu_seqlens.data_ptr(),
           d ** -0.5 if scale is None else float(scale), out.data_ptr(), _DTYPE_CODE[out.dtype],
           *((None, 0) if ws is None else (ws.data_ptr(), ws.numel())))
    return out


def append_prompt_kv(pool_k, pool_v, block_table, seq_lens, k_new, v_new, cu_seqlens, *, new_seq_lens=None):
    """Write the K/V rows of packed prompts (``k_new, v_new [tokens, Hkv, D]`` of the pool's
    dtype, any token and head strides) into the pool: sequence b's rows go to positions
    ``seq_lens[b], seq_lens[b] + 1, ...`` through the block table.  Returns the lengths
    after it, ``[n_seq] int32`` (``new_seq_lens`` when given; never ``seq_lens`` itself, so
    ``update_block_summaries`` can have both).  A position without a page is skipped and the
    length counts up to the first of them.  The many-token form of ``append_kv``: bf16 and
    float32 pools, capturable."""
    device_of(pool_k, pool_v, block_table, seq_lens, k_new, v_new, cu_seqlens, new_seq_lens)
    n_seq = _n_seq(cu_seqlens)
    check_ints(seq_lens, "seq_lens", n_seq)
    if pool_k.dtype not in (_F32, _BF16):
        raise ValueError("append takes bf16 or float32 pools")
    kv, hkv, d = _pool(pool_k, pool_v, block_table, None, n_seq)
    rows, tokens, *heads = _packed_rows(k_new, v_new)
    if heads != [hkv, d] or rows.dtype != kv.dtype:
        raise ValueError("k_new/v_new must be [tokens, Hkv, D] of the pool dtype with contiguous rows")
    if new_seq_lens is None:
        new_seq_lens = torch.empty_like(seq_lens)
    else:
        check_ints(new_seq_lens, "new_seq_lens", n_seq)
        if n_seq and abs(new_seq_lens.data_ptr() - seq_lens.data_ptr()) < 4 * n_seq:
            raise ValueError("new_seq_lens must not overlap seq_lens")
    launch(N.lib().ia_append_prompt_kv, pool_k, kv, rows, cu_seqlens.data_ptr(), seq_lens.data_ptr(),
           new_seq_lens.data_ptr(), n_seq, tokens, hkv, d)
    return new_seq_lens


def shared_prefix_decode(q, pool_k, pool_v, block_table, seq_lens, group_starts, shared_lens, *, scale=None,
                         scales=None, out=None, out_dtype=None, workspace=None):
    """Dense decode of a batch whose sequences share long prefixes: the result of
    ``paged_decode``, each shared prefix's K/V read once for all sequences of its group.

    ``q [batch, Hq, D]``; group g is the neighbouring sequences ``group_starts[g] ..
    group_starts[g + 1] - 1`` (``[n_groups + 1] int32``, on the device), whose first
    ``shared_lens[g]`` tokens (``[n_groups] int32``, any number, no multiple of a page
    needed) are the same; sequences of no group share nothing.  The shared tokens are read
    through the block-table row of the group's first sequence, the rest through each
    sequence's own row, so forked tables (``fork_sequences``) and tables that repeat the
    prefix in pages of their own give the same.  Any group of query heads up to 64; bf16,
    float32 and fp8 pools; at most 32768 sequences and as many groups."""
    device_of(q, pool_k, pool_v, block_table, seq_lens, group_starts, shared_lens, *(scales or ()))
    b = check_ints(seq_lens, "seq_lens")
    kv, hkv, d = _pool(pool_k, pool_v, block_table, scales, b)
    rows = _prompt_shape(q, 0, hkv, d)  # (checks q; a row per sequence)
    hq = rows.n_q_heads
    if rows.n_tokens != b:
        raise ValueError("q must have a row for each sequence")
    n_groups = check_ints(shared_lens, "shared_lens")
    check_ints(group_starts, "group_starts", n_groups + 1)
    out = output(q, out, out_dtype)
    shape_tail = hq, hkv, d, rows.q_token_stride, rows.q_head_stride, rows.q_dtype
    shape = N.DecodeShape(b, *shape_tail)
    # one buffer for every batch and group count up to a power of two: a later, larger call
    # never replaces one that a captured graph uses, and a server whose batch changes keeps few
    cap = 1 << (max(b, n_groups, 64) - 1).bit_length()
    key = ("shared_prefix_scratch", q.get_device(), cap, hkv, hq, d, kv.dtype)
    ws = None if workspace is None else workspace.get(key)
    if ws is None:
        need = N.lib().ia_shared_prefix_workspace_size(N.DecodeShape(cap, *shape_tail), kv.dtype, cap)
        ws = workspace_tensor(workspace, key, (max(need, 1),), device=q.device, dtype=torch.uint8)
    launch(N.lib().ia_shared_prefix_decode, q, shape, q.data_ptr(), kv, seq_lens.data_ptr(), group_starts.data_ptr(),
           shared_lens.data_ptr(), n_groups, d ** -0.5 if scale is None else float(scale), out.data_ptr(),
           _DTYPE_CODE[out.dtype], ws.data_ptr(), ws.numel())
    return out
