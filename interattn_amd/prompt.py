"""Prompt attention: causal attention of packed prompts, over their own K/V or over a
paged pool that holds them.

Packed rows put the sequences of a batch one behind the other with no padding:
``cu_seqlens [n_seq + 1] int32`` on the device holds the first row of each, and the end of
the last.  Pools, block tables and scales are those of ``ops``.  Calls launch on the
current stream of their tensors' device, never synchronise, and keep scratch and output in
the caller's ``workspace`` dict; calls that share one must not overlap.
"""

import torch

from . import _native as N
from .ops import _DTYPE_CODE, _code, _stream, paged_kv, workspace_tensor

_F32, _BF16 = torch.float32, torch.bfloat16


def same_device(ref, **tensors):
    """Every tensor on ``ref``'s GPU (a kernel dereferences them all there)."""
    if not ref.is_cuda:
        raise ValueError("interattn_amd kernels need device (cuda) tensors")
    for name, t in tensors.items():
        if t is not None and t.device != ref.device:
            raise ValueError(f"{name} must be on {ref.device}, got {t.device}")


def check_ints(t, name, length=None):
    """A contiguous int32 vector."""
    if t.dtype != torch.int32 or t.dim() != 1 or (t.shape[0] > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 vector")
    if length is not None and t.shape[0] != length:
        raise ValueError(f"{name} must have {length} entries, got {t.shape[0]}")


def launch(fn, ref, *args):
    """Call an entry point on the current stream of ``ref``'s device, with it current."""
    if torch.cuda.current_device() == ref.get_device():
        N.check(fn(*args, _stream(ref)))
    else:
        with torch.cuda.device(ref.device):
            N.check(fn(*args, _stream(ref)))


def _strides(t):
    """(token, head) strides of packed rows; a dimension of one row has any."""
    s = t.stride()
    return (s[0] if t.shape[0] > 1 else 0), (s[1] if t.shape[1] > 1 else 0)


def _shape(q, cu_seqlens, hkv, d):
    if q.dim() != 3 or (q.shape[2] > 1 and q.stride(2) != 1):
        raise ValueError("q must be [tokens, n_q_heads, D] with contiguous rows")
    if q.dtype not in (_F32, _BF16):
        raise ValueError("q must be float32 or bfloat16")
    if q.shape[2] != d:
        raise ValueError("q and the keys disagree on head_dim")
    if hkv <= 0 or q.shape[1] <= 0 or q.shape[1] % hkv:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads (grouped query attention)")
    check_ints(cu_seqlens, "cu_seqlens")
    if cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must have n_seq + 1 entries")
    return N.PromptShape(cu_seqlens.shape[0] - 1, q.shape[0], q.shape[1], hkv, d, _DTYPE_CODE[q.dtype], *_strides(q))


def output(q, out, out_dtype, workspace, key):
    """The caller's ``out`` or the workspace's, ``q``'s shape, contiguous."""
    if out is None:
        return workspace_tensor(workspace, key, q.shape, device=q.device, dtype=out_dtype or q.dtype)
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {list(q.shape)} tensor")
    if out.dtype not in (_F32, _BF16) or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("out must be float32 or bfloat16, of out_dtype where that is given")
    same_device(q, out=out)
    return out


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
    ``q`` too).  Returns ``[tokens, Hq, D]`` of ``out_dtype`` (``q``'s by default); rows of
    no sequence are left as ``out`` had them.  The prompt side of the paged decode calls,
    and what ``_sdpa_prefill_attention_forward`` (CBT/core.py:1180-1200) computes, without
    padding.  Forward only."""
    same_device(q, k=k, v=v, cu_seqlens=cu_seqlens)
    if k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0]:
        raise ValueError("k and v must be [tokens, n_kv_heads, D] with q's tokens")
    if k.stride(2) != 1 or v.stride(2) != 1 or k.dtype != v.dtype:
        raise ValueError("k and v must share a dtype and have contiguous rows")
    code = _code(k.dtype, "k and v")
    shape = _shape(q, cu_seqlens, int(k.shape[1]), int(k.shape[2]))
    out = output(q, out, out_dtype, workspace, "prompt_output")
    kv = N.PackedKV(k.data_ptr(), v.data_ptr(), code, *_strides(k), *_strides(v))
    ws = _workspace(shape, code, int(q.shape[0]), workspace, q.device)
    if q.shape[0] == 0:
        return out
    launch(N.lib().ia_prompt_attention, q, shape, q.data_ptr(), kv, cu_seqlens.data_ptr(),
           q.shape[2] ** -0.5 if scale is None else float(scale), out.data_ptr(), _DTYPE_CODE[out.dtype],
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
    kv, keep = paged_kv(pool_k, pool_v, block_table, scales)
    same_device(q, pool_k=pool_k, pool_v=pool_v, block_table=block_table, seq_lens=seq_lens, cu_seqlens=cu_seqlens)
    shape = _shape(q, cu_seqlens, int(pool_k.shape[1]), int(pool_k.shape[3]))
    check_ints(seq_lens, "seq_lens", int(shape.n_seq))
    if block_table is not None and block_table.shape[0] != shape.n_seq:
        raise ValueError("block_table rows must match the sequences")
    out = output(q, out, out_dtype, workspace, "prompt_output")
    cap = (kv.bt_cols if block_table is not None else kv.n_pages) * kv.page_size
    ws = _workspace(shape, kv.dtype, min(cap, (1 << 31) - 1025), workspace, q.device)
    if q.shape[0] == 0:
        return out
    launch(N.lib().ia_paged_prompt_attention, q, shape, q.data_ptr(), kv, seq_lens.data_ptr(), cu_seqlens.data_ptr(),
           q.shape[2] ** -0.5 if scale is None else float(scale), out.data_ptr(), _DTYPE_CODE[out.dtype],
           *((None, 0) if ws is None else (ws.data_ptr(), ws.numel())))
    del keep
    return out


def append_prompt_kv(pool_k, pool_v, block_table, seq_lens, k_new, v_new, cu_seqlens, *, new_seq_lens=None):
    """Write the K/V rows of packed prompts (``k_new, v_new [tokens, Hkv, D]`` of the pool's
    dtype, any token and head strides) into the pool: sequence b's rows go to positions
    ``seq_lens[b], seq_lens[b] + 1, ...`` through the block table.  Returns the lengths
    after it, ``[n_seq] int32`` (``new_seq_lens`` when given; never ``seq_lens`` itself, so
    ``update_block_summaries`` can have both).  A position without a page is skipped and the
    length counts up to the first of them.  The many-token form of ``append_kv``: bf16 and
    float32 pools, capturable."""
    kv, keep = paged_kv(pool_k, pool_v, block_table)
    same_device(pool_k, pool_v=pool_v, block_table=block_table, seq_lens=seq_lens, k_new=k_new, v_new=v_new,
                cu_seqlens=cu_seqlens, new_seq_lens=new_seq_lens)
    check_ints(cu_seqlens, "cu_seqlens")
    n_seq = int(cu_seqlens.shape[0]) - 1
    if n_seq < 0:
        raise ValueError("cu_seqlens must have n_seq + 1 entries")
    check_ints(seq_lens, "seq_lens", n_seq)
    hkv, d = int(pool_k.shape[1]), int(pool_k.shape[3])
    for t in (k_new, v_new):
        if t.dim() != 3 or tuple(t.shape[1:]) != (hkv, d) or t.stride(2) != 1 or t.dtype != pool_k.dtype:
            raise ValueError("k_new/v_new must be [tokens, Hkv, D] of the pool dtype with contiguous rows")
    if k_new.shape[0] != v_new.shape[0]:
        raise ValueError("k_new and v_new must have the same tokens")
    if block_table is not None and block_table.shape[0] != n_seq:
        raise ValueError("block_table rows must match the sequences")
    if new_seq_lens is None:
        new_seq_lens = torch.empty_like(seq_lens)
    check_ints(new_seq_lens, "new_seq_lens", n_seq)
    if n_seq and abs(new_seq_lens.data_ptr() - seq_lens.data_ptr()) < 4 * n_seq:
        raise ValueError("new_seq_lens must not overlap seq_lens")
    rows = N.PackedKV(k_new.data_ptr(), v_new.data_ptr(), kv.dtype, *_strides(k_new), *_strides(v_new))
    launch(N.lib().ia_append_prompt_kv, pool_k, kv, rows, cu_seqlens.data_ptr(), seq_lens.data_ptr(),
           new_seq_lens.data_ptr(), n_seq, int(k_new.shape[0]), hkv, d)
    del keep
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
    float32 and fp8 pools."""
    kv, keep = paged_kv(pool_k, pool_v, block_table, scales)
    same_device(q, pool_k=pool_k, pool_v=pool_v, block_table=block_table, seq_lens=seq_lens,
                group_starts=group_starts, shared_lens=shared_lens)
    hkv, d = int(pool_k.shape[1]), int(pool_k.shape[3])
    if q.dim() != 3 or q.stride(2) != 1 or q.dtype not in (_F32, _BF16) or q.shape[2] != d:
        raise ValueError("q must be [batch, n_q_heads, D] float32 or bfloat16 with contiguous rows of the pool's D")
    b, hq, _ = q.shape
    if hkv <= 0 or hq <= 0 or hq % hkv:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads (grouped query attention)")
    check_ints(seq_lens, "seq_lens", b)
    check_ints(shared_lens, "shared_lens")
    n_groups = int(shared_lens.shape[0])
    check_ints(group_starts, "group_starts", n_groups + 1)
    if block_table is not None and block_table.shape[0] != b:
        raise ValueError("block_table rows must match the batch")
    out = output(q, out, out_dtype, workspace, "attention_output")
    shape = N.DecodeShape(b, hq, hkv, d, *_strides(q), _DTYPE_CODE[q.dtype])
    key = ("shared_prefix_scratch", b, n_groups, hkv, hq, d, kv.dtype)
    ws = None if workspace is None else workspace.get(key)
    if ws is None or ws.device != q.device:
        need = N.lib().ia_shared_prefix_workspace_size(shape, kv.dtype, n_groups)
        ws = workspace_tensor(workspace, key, (max(need, 1),), device=q.device, dtype=torch.uint8)
    launch(N.lib().ia_shared_prefix_decode, q, shape, q.data_ptr(), kv, seq_lens.data_ptr(), group_starts.data_ptr(),
           shared_lens.data_ptr(), n_groups, d ** -0.5 if scale is None else float(scale), out.data_ptr(),
           _DTYPE_CODE[out.dtype], ws.data_ptr(), ws.numel())
    del keep
    return out
