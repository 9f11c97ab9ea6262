"""A serving step's work on the paged K/V pool that the codes protect.

No reference counterpart: the reference's plugin hooks an engine that brings its
own cache writes and attention (bench_ghostserve_rdp.py:396-481).

  norm_rotate_write   queries and keys normed by head and turned to their
                      positions, keys and values written to their slots
  prefix_attention    attention over the pool for a batch whose requests share
                      a prefix, which is computed once for all of them

Both serve and do not train: there is no backward pass, and tensors that ask for
a gradient are refused (under ``torch.no_grad()`` nothing asks for one).

Pool tensor: [layers, pool_pages, page_tokens, 2 (K,V), kv_heads, head_dim], of
the queries' type or float8_e4m3fn with a scale for K and for V, as in
:mod:`.paged`; slots and page tables as :func:`.paged.step_tables` makes them.
"""
from __future__ import annotations

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3}
_FLOAT_MAX = torch.finfo(torch.float32).max
_COMPUTE = (torch.bfloat16, torch.float16, torch.float32)


def rotary_frequencies(rot: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """theta^(-2i/rot) for the rot/2 pairs of a rotation, in 64 bits (radians a
    position); a program with frequencies of its own passes those instead."""
    if rot < 2 or rot % 2:
        raise ValueError("rot must be even and positive")
    i = torch.arange(rot // 2, dtype=torch.float64)
    return (float(theta) ** (-2.0 * i / rot)).to(device)


def rotary_axes(sections, device="cuda") -> torch.Tensor:
    """axis_of for positions with several axes (time, height, width): the first
    sections[0] pairs turn with axis 0, the next sections[1] with axis 1, ..."""
    if not sections or any(int(n) < 0 for n in sections) or len(sections) > 8:
        raise ValueError("sections are 1 to 8 counts of pairs")
    n = torch.tensor([int(x) for x in sections])
    return torch.repeat_interleave(torch.arange(len(sections), dtype=torch.uint8), n).to(device)


def _layer(pool: torch.Tensor, layer: int) -> tuple[int, int, int, int]:
    """(address of the layer, slots, kv_heads, head_dim) of a pool."""
    shape = pool.shape
    if len(shape) != 6 or shape[3] != 2:
        raise ValueError("pool must be [layers, pool_pages, page_tokens, 2, heads, dim]")
    if not pool.is_contiguous():
        raise ValueError("pool must be a contiguous GPU (HIP) tensor")
    L, pages, pt, _, H, D = shape
    if not 0 <= layer < L:
        raise ValueError(f"layer {layer} not in [0, {L})")
    n = pages * pt
    return pool.data_ptr() + layer * n * 2 * H * D * pool.element_size(), n, H, D


def _scale(t, device, what: str):
    """Address of a scale: a float32 tensor of one value on the GPU, or 0."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != 1 or t.device != device:
        raise ValueError(f"{what} must be one float32 value on the pool's device")
    return t.data_ptr()


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def norm_rotate_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None,
                      freqs: torch.Tensor | None, pool: torch.Tensor, slots: torch.Tensor, *, layer: int = 0,
                      norm: bool = True, q_weight: torch.Tensor | None = None,
                      k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                      axis_of: torch.Tensor | None = None, interleaved: bool = False, factor: float = 1.0,
                      k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                      tokens: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Queries and keys normed by head and rotated; K and V written to the pool.

    ``q`` [tokens, heads, dim], ``k`` and ``v`` [tokens, kv_heads, dim], float32,
    bfloat16 or float16: tensors or views of a packed projection (each head's
    values adjacent, any other strides).  With ``norm`` each head of q and k is
    divided by the root of its mean square (+ ``eps``) and multiplied by the
    weight [dim].  Then its first 2 len(``freqs``) values are turned: pair i by the
    angle positions * freqs[i], pairs (i, i + len) or, ``interleaved``, (2i, 2i+1),
    cos and sin times ``factor``.  ``positions``: int32 [tokens], or [axes, tokens]
    with ``axis_of`` (uint8 [len(freqs)], see :func:`rotary_axes`) naming each
    pair's axis.  ``freqs``: float64, or None: no rotation.

    Token t's K and V go to slot ``slots[t]`` (int32, page * page_tokens + place;
    negative or past the pool: none) of the pool's ``layer``, in the queries' type
    or, float8_e4m3fn, as value / scale.  The slots of a call must be distinct.
    ``tokens`` (int32 [1] on the GPU, e.g. ``cu_new[-1:]``): tokens from that
    number on are left as they were, here and in the result.

    Returns the queries (``out``: contiguous like q, or q itself)."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError("q must be [tokens, heads, dim], k and v [tokens, kv_heads, dim]")
    dev, dt = q.device, q.dtype
    if dt not in _COMPUTE or k.dtype != dt or v.dtype != dt:
        raise ValueError("q, k and v must be of one type: float32, bfloat16 or float16")
    _lib.require_no_grad(q, k, v, q_weight, k_weight, pool, out, what="norm_rotate_write")
    _lib.require_same_device(dev, k, v, positions, freqs, pool, slots, q_weight, k_weight, axis_of, tokens, out,
                             what="norm_rotate_write tensor")
    N, Hq, D = qs
    base, n_slots, Hk, Dp = _layer(pool, layer)
    if Hk != ks[1] or Dp != D:
        raise ValueError(f"pool holds {Hk} heads of {Dp}, k has {ks[1]} of {D}")
    pool_dt = pool.dtype
    if pool_dt != dt and pool_dt != torch.float8_e4m3fn:
        raise ValueError("pool must be of q's type or float8_e4m3fn")
    (q0, q1, q2), (k0, k1, k2), (v0, v1, v2) = q.stride(), k.stride(), v.stride()
    if D > 1 and N and not q2 == k2 == v2 == 1:
        raise ValueError("a head's values must be adjacent")
    if slots.dtype != torch.int32 or slots.shape != (N,) or not slots.is_contiguous():
        raise ValueError(f"slots must be contiguous int32 [{N}]")
    half = 0 if freqs is None else freqs.shape[0]
    axes, axis_stride = 1, N
    if half:
        if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous() or 2 * half > D:
            raise ValueError("freqs must be contiguous float64 with at most dim/2 values")
        if positions is None or positions.dtype != torch.int32 or positions.dim() not in (1, 2) \
                or positions.shape[-1] != N or (N > 1 and positions.stride(-1) != 1):
            raise ValueError(f"positions must be int32 [{N}] or [axes, {N}], adjacent by token")
        if positions.dim() == 2:
            axes = positions.shape[0]
            if axes > 1:
                axis_stride = positions.stride(0)
                if axis_of is None:
                    raise ValueError("positions with several axes need axis_of")
        if axis_of is not None and (axis_of.dtype != torch.uint8 or axis_of.shape != (half,)
                                    or not axis_of.is_contiguous()):
            raise ValueError(f"axis_of must be contiguous uint8 [{half}]")
    for w in (q_weight, k_weight):
        if w is not None and (not norm or w.dtype != dt or w.shape != (D,) or not w.is_contiguous()):
            raise ValueError(f"weights belong to the norm and must be contiguous [{D}] of q's type")
    if tokens is not None and (tokens.dtype != torch.int32 or tokens.numel() != 1):
        raise ValueError("tokens must be one int32 value")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        o0, o1 = Hq * D, D
    elif out.shape != qs or out.dtype != dt or not (out.is_contiguous() or out is q):
        raise ValueError("out must be contiguous and like q, or q itself")
    else:
        o0, o1, _ = out.stride()
    if not (abs(eps) <= _FLOAT_MAX and abs(factor) <= _FLOAT_MAX):
        raise ValueError("eps and factor must be finite 32-bit numbers")
    s = _lib.pack(
        _lib.NORM_ROTATE_FORMAT, N, Hq, Hk, D, _DTYPES[dt], q.data_ptr(), k.data_ptr(), v.data_ptr(), q0, q1, k0, k1,
        v0, v1, out.data_ptr(), o0, o1, bool(norm), eps, _ptr(q_weight), _ptr(k_weight), 2 * half, bool(interleaved),
        axes, _ptr(positions), axis_stride, _ptr(axis_of), _ptr(freqs), factor, base, _DTYPES[pool_dt], n_slots,
        slots.data_ptr(), _scale(k_scale, dev, "k_scale"), _scale(v_scale, dev, "v_scale"), _ptr(tokens))
    _lib.call_on(dev, "kvec_norm_rotate_write", s, _lib.stream_handle(dev))
    return out


def prefix_attention(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     prefix: int = 0, *, layer: int = 0, cu_q: torch.Tensor | None = None,
                     max_q: int | None = None, max_len: int | None = None,
                     prefix_pages: torch.Tensor | None = None, scale: float | None = None,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's queries over the pool's ``layer``.

    ``q`` [tokens, heads, dim] (bfloat16 or float16; each head's values adjacent):
    the requests' new tokens one after another, request b's from ``cu_q[b]`` to
    ``cu_q[b+1]`` - 1, or without ``cu_q`` one token a request.  Request b holds
    ``seq_lens[b]`` tokens, its new ones included (their K and V are in the pool
    already, see :func:`norm_rotate_write`), on the pages of its row of
    ``page_table``; each query sees the positions up to its own.  Query heads
    share K/V heads in order.  dim: a multiple of 8 (fp8 pool: 16) up to 256.

    The first ``prefix`` positions are the same for all requests; they are read
    from ``prefix_pages`` (default: the first row of ``page_table``, which has to hold
    them even if its request is idle) once for all queries.  ``prefix`` need not be
    whole pages.  0 is ordinary paged attention.

    Keys on pages outside the pool are left out; a query that sees no key (an idle
    row: ``seq_lens`` 0) gives zeros.  Rows before ``cu_q[0]`` and from ``cu_q[-1]``
    on are left as they were.

    ``max_q``: the most tokens of a request; a request's tokens past it are left as
    they were.  The kind of blocks is chosen by it, once for the call: without it every
    request is taken for one of all tokens, which for 64 decoding requests behind 8192
    shared keys takes nearly six times as long, and a step of few long and many short requests
    is faster as two calls.  ``max_len``: about the longest of ``seq_lens`` (default:
    what a table row can hold), by which the work is split.  ``scale``: default
    1/sqrt(dim).  ``k_scale``, ``v_scale``: an fp8 pool's, as in
    :func:`norm_rotate_write`.  Nothing is read back to the host, so the call can be
    captured in a graph.

    Scores, maxima, sums and outputs are 32-bit; the softmax's weights are rounded to
    the queries' type before they multiply V."""
    shape, tab = q.shape, page_table.shape
    if len(shape) != 3:
        raise ValueError("q must be [tokens, heads, dim]")
    dev, dt, i32 = q.device, q.dtype, torch.int32
    if dt != torch.bfloat16 and dt != torch.float16:
        raise ValueError("q must be bfloat16 or float16")
    if len(tab) != 2 or page_table.dtype != i32 or seq_lens.dtype != i32:
        raise ValueError("page_table must be int32 [batch, pages_per_seq], seq_lens int32")
    N, Hq, D = shape
    B, width = tab
    if seq_lens.shape != (B,) or (cu_q is not None and (cu_q.shape != (B + 1,) or cu_q.dtype != i32)):
        raise ValueError(f"seq_lens must be [{B}] and cu_q int32 [{B + 1}]")
    if cu_q is None and N != B:
        raise ValueError("without cu_q there is one query token a request")
    _lib.require_no_grad(q, pool, out, what="prefix_attention")
    _lib.require_same_device(dev, pool, page_table, seq_lens, cu_q, prefix_pages, out, what="prefix_attention tensor")
    base, _, Hk, Dp = _layer(pool, layer)
    if Dp != D or Hq % Hk:
        raise ValueError(f"q has {Hq} heads of {D}, the pool {Hk} of {Dp}")
    pool_dt = pool.dtype
    if pool_dt != dt and pool_dt != torch.float8_e4m3fn:
        raise ValueError("pool must be of q's type or float8_e4m3fn")
    for t in (page_table, seq_lens, cu_q, prefix_pages):
        if t is not None and not t.is_contiguous():
            raise ValueError("page_table, seq_lens, cu_q and prefix_pages must be contiguous")
    q0, q1, q2 = q.stride()
    if N and D > 1 and q2 != 1:
        raise ValueError("a head's values must be adjacent")
    pages, pt, prefix = pool.shape[1], pool.shape[2], int(prefix)
    if prefix_pages is None:
        front = page_table
    else:
        front = prefix_pages
        if front.dtype != i32 or front.numel() * pt < prefix:
            raise ValueError("prefix_pages must be int32 and hold the prefix")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != dt or not out.is_contiguous():
        raise ValueError("out must be contiguous and like q")
    max_q = max(N, 1) if max_q is None else min(int(max_q), max(N, 1))
    max_len = min(int(max_len or 0), width * pt)
    scale = D ** -0.5 if scale is None else float(scale)
    if max_q < 0 or max_len < 0 or not 0.0 <= scale <= _FLOAT_MAX:
        raise ValueError("max_q, max_len and scale must not be negative, and scale finite")
    if max_q == 0 and cu_q is not None:           # every request is idle
        return out
    s = _lib.pack(
        _lib.ATTENTION_FORMAT, N, B, Hq, Hk, D, _DTYPES[dt], q.data_ptr(), q0, q1, out.data_ptr(), Hq * D, D, base,
        _DTYPES[pool_dt], pages, pt, page_table.data_ptr(), width, seq_lens.data_ptr(), _ptr(cu_q), max_q, max_len,
        prefix, front.data_ptr(), scale, _scale(k_scale, dev, "k_scale"), _scale(v_scale, dev, "v_scale"))
    need = _lib.lib().kvec_prefix_attention_workspace(s)
    ws = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _lib.call_on(dev, "kvec_prefix_attention", s, _ptr(ws), max(need, 0), _lib.stream_handle(dev))
    return out
