"""Rotary positions, and the way into the cache that turns keys as it writes them.

A ``RotaryPlan`` (``rotary_plan``) holds a model's frequencies on the device.  Angles are
formed in the kernels from whole positions in 64-bit fixed point, so there is no table to
build or outgrow and far positions lose nothing.  Rows are packed as in ``prompt``
(``[tokens, heads, D]``, any token and head strides of 16-byte multiples).  Calls launch on the
current stream of their tensors' device, never synchronise and can be captured.  Forward only;
the gradient of a rotation is the call with ``inverse=True``.
"""

import functools
import math

import torch

from . import _native as N
from .ops import _DTYPE_CODE
from .prompt import check_ints, device_of, launch, packed_rows, pool_of, prompt_lengths

_ROW_DTYPES = (torch.float32, torch.bfloat16)
LAYOUTS = ("half", "interleaved")
_TWO_ROWS = N.RotaryRows * 2


# 2 pi in units of 10^-62: with the 53 bits of a float64 pi, the angle of position 2^31 would be
# 150 units of 2^-32 turns off
_TWO_PI = 628318530717958647692528676655900576839433879875021164194988918


def _turns(w):
    """``w`` radians as turns in units of 2^-64: the nearest whole number.  (Whole turns a position,
    which no model has, are first taken off in float64.)"""
    num, den = math.fmod(w, 2 * math.pi).as_integer_ratio()
    num, den = num * (10 ** 62 << 64), den * _TWO_PI
    return (2 * num + den) // (2 * den) % (1 << 64)


class RotaryPlan:
    """Frequencies of a rotation on one device: ``dim`` channels in pairs, ``layout`` ``"half"``
    (channel i with i + dim / 2) or ``"interleaved"`` (2 i with 2 i + 1), ``factor`` the amplitude,
    ``turns [dim / 2] int64`` the turns per position in units of 2^-64."""

    def __init__(self, turns, layout, factor):
        self.turns, self.layout, self.factor = turns, layout, float(factor)
        self.dim = 2 * turns.shape[0]
        self.native = N.Rotary(turns.data_ptr() or None, self.dim, int(layout == "interleaved"), self.factor)


def _known(scaling, *keys):
    extra = set(scaling) - {"rope_type", "type", "rope_theta", *keys}
    if extra:
        raise ValueError(f"scaling has entries that {scaling.get('rope_type')!r} does not know: {sorted(extra)}")
    missing = [k for k in ("factor", "original_max_position_embeddings") if k in keys and scaling.get(k) is None]
    if missing:
        raise ValueError(f"scaling needs {missing}")
    if "factor" in keys and scaling["factor"] <= 0:
        raise ValueError("the scaling factor must be positive")


def rotary_frequencies(dim, *, base=None, scaling=None):
    """``(radians per position of each pair, factor)``, in 64 bits.  ``base`` is 10000 unless
    given, here or as ``scaling``'s ``rope_theta``.  ``scaling`` is a model config's entry:
    ``rope_type`` ``"default"``, ``"linear"`` (``factor``), ``"yarn"`` (``factor``,
    ``original_max_position_embeddings``, optional ``beta_fast``, ``beta_slow``, ``truncate``,
    ``attention_factor``) or ``"llama3"`` (``factor``, ``original_max_position_embeddings``,
    ``low_freq_factor``, ``high_freq_factor``)."""
    if dim < 0 or dim % 2:
        raise ValueError("the rotated channels must be an even number")
    scaling = dict(scaling or {})
    theta = scaling.get("rope_theta")
    if base is not None and theta is not None and base != theta:
        raise ValueError(f"base {base} is not scaling's rope_theta {theta}")
    base = float(base if base is not None else 10000.0 if theta is None else theta)
    if not 0 < base < math.inf:
        raise ValueError("base must be positive")
    w = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        _known(scaling)
        return w, 1.0
    if kind == "linear":
        _known(scaling, "factor")
        return [x / scaling["factor"] for x in w], 1.0
    if kind == "yarn":
        # pairs that turn often in the original context keep their frequency, those that turn
        # less than beta_slow times are stretched, and a ramp over the pairs joins them
        _known(scaling, "factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate",
               "attention_factor")
        s, context = float(scaling["factor"]), scaling["original_max_position_embeddings"]
        if base <= 1:
            raise ValueError("'yarn' needs a base above 1")

        def pair(turns):
            return dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = pair(scaling.get("beta_fast") or 32), pair(scaling.get("beta_slow") or 1)
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, dim - 1)
        width = hi - lo if hi != lo else 1e-3
        ramp = [min(max((i - lo) / width, 0.0), 1.0) for i in range(dim // 2)]
        amplitude = scaling.get("attention_factor")
        if amplitude is None:
            amplitude = 0.1 * math.log(s) + 1.0 if s > 1 else 1.0
        return [x * (1.0 - r) + x / s * r for x, r in zip(w, ramp)], float(amplitude)
    if kind == "llama3":
        _known(scaling, "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor")
        s, context = float(scaling["factor"]), scaling["original_max_position_embeddings"]
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        # turns in the original context: `high` and more stay, `low` and less are stretched
        keep = [min(max((context * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in w]
        return [x * k + x / s * (1.0 - k) for x, k in zip(w, keep)], 1.0
    raise ValueError(f"unknown rope_type {kind!r}: 'default', 'linear', 'yarn' or 'llama3', or pass inv_freq")


def rotary_plan(dim, *, base=None, scaling=None, inv_freq=None, factor=None, layout="half", device="cuda"):
    """A ``RotaryPlan`` of ``dim`` channels: frequencies from ``base`` and ``scaling`` (see
    ``rotary_frequencies``), or ``inv_freq``, radians per position of each pair (numbers or a
    tensor).  ``factor`` multiplies the rotated channels (by default what ``scaling`` asks for).
    Made once per model and kept; copies a few hundred bytes to the device."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if inv_freq is None:
        w, amplitude = rotary_frequencies(dim, base=base, scaling=scaling)
    else:
        if scaling is not None or base is not None:
            raise ValueError("base and scaling make frequencies: inv_freq holds them already")
        w, amplitude = [float(x) for x in inv_freq], 1.0
        if 2 * len(w) != dim:
            raise ValueError("inv_freq must hold a frequency for each of dim / 2 pairs")
    if not all(math.isfinite(x) for x in w) or (factor is not None and not math.isfinite(factor)):
        raise ValueError("frequencies and factor must be finite")
    fixed = [_turns(x) for x in w]
    turns = torch.tensor([x - (1 << 64) if x >> 63 else x for x in fixed], dtype=torch.int64).to(device)
    return RotaryPlan(turns, layout, amplitude if factor is None else factor)


@functools.lru_cache(maxsize=1024)
def _heads(shape, stride, dtype, what):
    """``(heads, D, token stride, head stride)`` of rows ``[tokens, heads, D]``."""
    if len(shape) != 2 or (shape[1] > 1 and stride[2] != 1):
        raise ValueError(f"{what} must be [tokens, heads, D] with contiguous rows")
    if dtype not in _ROW_DTYPES:
        raise ValueError(f"{what} must be float32 or bfloat16")
    return shape[0], shape[1], stride[0], stride[1] if shape[0] > 1 else 0


def _rows(x, out, what):
    """``RotaryRows`` of ``x`` and its output (made where None), and the output."""
    shape = x.shape
    heads, d, tok, head = _heads(shape[1:], x.stride(), x.dtype, what)
    if out is None:
        out = x.new_empty(shape)
        o_tok, o_head = heads * d, d
    else:
        if out.shape != shape or out.dtype != x.dtype:
            raise ValueError(f"{what}_out must have {what}'s shape and dtype")
        _, _, o_tok, o_head = _heads(shape[1:], out.stride(), out.dtype, what + "_out")
    if shape[0] <= 1:
        tok = o_tok = 0  # (any stride means nothing then)
    return N.RotaryRows(x.data_ptr(), out.data_ptr(), tok, head, o_tok, o_head, heads), out


def apply_rotary(q, k, positions, plan, *, inverse=False, q_out=None, k_out=None):
    """Turn packed rows ``q [tokens, Hq, D]`` and ``k [tokens, Hkv, D]`` (or None) to
    ``positions [tokens] int32`` (any, negative ones too): one launch, sums in float32, rounded
    once.  D is a multiple of 16 up to 256; channels past ``plan.dim`` are copied as they are.
    Returns ``(q, k)`` turned: new tensors, or ``q_out`` / ``k_out``, each of which may be its
    input itself and has to lie apart from the inputs and the other output else (views of one
    buffer do where their rows do).  ``inverse``: angles negated (the gradient; a rotation by
    position differences moves cached keys).  Forward only: the outputs carry no gradient back to
    the inputs; a backward pass calls it with the outputs' gradients and ``inverse``."""
    device_of(q, k, positions, plan.turns if plan.dim else None, q_out, k_out)
    shape = q.shape
    tokens = check_ints(positions, "positions", shape[0] if len(shape) else None)
    q_rows, q_out = _rows(q, q_out, "q")
    d = shape[2]
    n = 1
    if k is not None:
        of_k = k.shape
        if len(of_k) != 3 or of_k[0] != tokens or of_k[2] != d or k.dtype != q.dtype:
            raise ValueError("k must have q's tokens, head_dim and dtype")
        k_rows, k_out = _rows(k, k_out, "k")
        rows, n = _TWO_ROWS(q_rows, k_rows), 2
    else:
        if k_out is not None:
            raise ValueError("k_out is given without k")
        rows = _TWO_ROWS(q_rows)
    if tokens:
        launch(N.lib().ia_apply_rotary, q, plan.native, rows, n, _DTYPE_CODE[q.dtype], d, positions.data_ptr(), tokens,
               int(inverse))
    return q_out, k_out


def rotary_append_kv(q, k_new, v_new, plan, pool_k, pool_v, block_table, seq_lens, cu_seqlens=None, *, positions=None,
                     scales=None, q_out=None, new_seq_lens=None):
    """One launch between a layer's projections and its attention: queries turned to their
    positions, keys turned and written with the values into the paged pool.

    ``q [tokens, Hq, D]`` (or None), ``k_new, v_new [tokens, Hkv, D]`` packed; sequence b's rows
    ``cu_seqlens[b] ..`` are the positions ``seq_lens[b], seq_lens[b] + 1, ...`` of the pool, and
    what they are turned to, unless ``positions [tokens] int32`` (not the tensor the lengths are
    written to) says otherwise.  ``plan`` None turns nothing.  ``q_out`` may be ``q`` itself and has
    to lie apart from the inputs else.  Pools are bf16 or float32 as the rows are, or fp8 with ``scales=(k_scale,
    v_scale)`` (two tensors, or views that lie apart), which the call sets: every page gets the least power of two that brings its
    largest finite magnitude down to 448; a page with earlier tokens keeps its scale while that
    is enough, else its codes are rewritten with it (exact, but for what turns subnormal).  A
    value that is not finite becomes NaN and sets no scale.  What else holds scales
    (``sequence_scales``) has to be rebuilt.

    Without ``cu_seqlens`` every sequence has one token (a decode step) and ``seq_lens`` advances
    in place unless ``new_seq_lens`` is given.  Returns ``(q turned, lengths after it)``; a
    position without a page is skipped and the length counts up to the first of them, as in
    ``append_prompt_kv``.  Rows of no sequence are left as ``q_out`` had them (a new tensor's are
    not set).  Forward only."""
    device_of(k_new, pool_k, pool_v, block_table, seq_lens, v_new, cu_seqlens, q, q_out, positions, new_seq_lens,
              plan.turns if plan is not None and plan.dim else None, *(scales or ()))
    n_seq = check_ints(seq_lens, "seq_lens")
    if scales is not None and len(scales) != 2:
        raise ValueError("scales must be (k_scale, v_scale): copies per sequence are gathered again afterwards")
    kv, hkv, d = pool_of(pool_k, pool_v, block_table, scales, n_seq)
    rows, tokens, *heads = packed_rows(k_new, v_new)
    if heads != [hkv, d] or k_new.dtype not in _ROW_DTYPES or (rows.dtype != kv.dtype
                                                               and kv.dtype != N.IA_FP8_E4M3):
        raise ValueError("k_new/v_new must be [tokens, Hkv, D] of the pool dtype (float32 or bfloat16 for fp8 pools) "
                         "with contiguous rows")
    if cu_seqlens is not None:
        check_ints(cu_seqlens, "cu_seqlens", n_seq + 1)
    elif tokens != n_seq:
        raise ValueError("without cu_seqlens every sequence has one token")
    new_seq_lens = prompt_lengths(seq_lens, new_seq_lens, n_seq, in_place=cu_seqlens is None)
    if positions is not None:
        check_ints(positions, "positions", tokens)
    q_rows = None
    if q is not None:
        shape = q.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != d or q.dtype != k_new.dtype:
            raise ValueError("q must be [tokens, Hq, D] with k_new's tokens, head_dim and dtype")
        if shape[1] == 0 or shape[1] % hkv:
            raise ValueError("n_q_heads must be a multiple of n_kv_heads (grouped query attention)")
        q_rows, q_out = _rows(q, q_out, "q")
    elif q_out is not None:
        raise ValueError("q_out is given without q")
    launch(N.lib().ia_rotary_append_kv, k_new, None if plan is None else plan.native, q_rows, rows, kv,
           None if cu_seqlens is None else cu_seqlens.data_ptr(), seq_lens.data_ptr(), new_seq_lens.data_ptr(),
           None if positions is None else positions.data_ptr(), n_seq, tokens, hkv, d)
    return q_out, new_seq_lens
