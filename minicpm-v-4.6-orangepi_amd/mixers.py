"""Token mixers that stand between a decoder layer's quantised projections, over
the C-ABI in include/mcv_mixers.h: the gated delta rule of the linear-attention
layers, several-axis rotary positions, and one-token attention over a paged
key-value cache for the full-attention layers.

Activations and caches are fp16, gates and states fp32.  q, k and v may be
columns of one projection's output: rows and heads have strides, the elements
of one head are contiguous.
"""
from __future__ import annotations

from . import _GEMM_COUNTER_BYTES, McvError, _check, _stream, _torch, gemm_workspace, lib

_NULL = 0


def _heads(who: str, name: str, t, rows: int | None = None, heads: int | None = None):
    """(pointer, row stride, head stride) of fp16 [rows][heads][D]."""
    s = t.stride()
    if t.dtype != _torch().float16 or len(s) != 3 or s[2] != 1 or (rows is not None and t.shape[0] != rows) or \
            (heads is not None and t.shape[1] != heads):
        raise McvError(f"{who}: {name} must be fp16 [{'rows' if rows is None else rows}, "
                       f"{'heads' if heads is None else heads}, D] with contiguous heads, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr(), s[0], s[1]


def _workspace(nbytes: int, device, stream):
    """gemm_workspace's buffer of the next power of two: few sizes, whatever the calls'.  Other calls
    on the stream use it too, so its first _GEMM_COUNTER_BYTES are counters and stay zero."""
    return gemm_workspace(1 << (nbytes - 1).bit_length(), device, stream)


def _same_device(who: str, t, *others) -> None:
    for o in others:
        if o is not None and o.device != t.device:
            raise McvError(f"{who}: tensors on {t.device} and {o.device}")


def _delta(who, q, k, v, g, beta, state, cu, B, scale, normalize, state_index, out, state_out, stream):
    torch = _torch()
    T, Hk, Dk = q.shape
    Hv, Dv = v.shape[1], v.shape[2]
    if k.shape != q.shape:
        raise McvError(f"{who}: q {tuple(q.shape)} and k {tuple(k.shape)} must have one shape")
    qa, ka, va = _heads(who, "q", q), _heads(who, "k", k), _heads(who, "v", v, T)
    gates = []
    for name, t in (("g", g), ("beta", beta)):
        s = t.stride()
        if t.dtype != torch.float32 or t.shape != (T, Hv) or s[1] != 1:
            raise McvError(f"{who}: {name} must be fp32 [{T}, {Hv}] with contiguous rows")
        gates += (t.data_ptr(), s[0])
    n_states = B
    if state_index is not None:
        if state_index.dtype != torch.int32 or state_index.shape != (B,) or not state_index.is_contiguous():
            raise McvError(f"{who}: state_index must be contiguous int32 [{B}]")
        pool = state_out if state_out is not None else state
        if pool is None:
            raise McvError(f"{who}: state_index needs a state or state_out to index")
        n_states = pool.shape[0]
        if state_out is None:
            state_out = state                    # a pool is updated in place
    if state_out is None:
        state_out = torch.empty((B, Hv, Dk, Dv), dtype=torch.float32, device=q.device)
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (n_states, Hv, Dk, Dv) or not t.is_contiguous()):
            raise McvError(f"{who}: {name} must be contiguous fp32 [{n_states}, {Hv}, {Dk}, {Dv}]")
    if out is None:
        out = torch.empty((T, Hv, Dv), dtype=torch.float16, device=q.device)
    elif out.dtype != torch.float16 or out.shape != (T, Hv, Dv) or not out.is_contiguous():
        raise McvError(f"{who}: out must be contiguous fp16 [{T}, {Hv}, {Dv}]")
    _same_device(who, q, k, v, g, beta, state, state_out, state_index, cu, out)
    L = lib()
    nbytes = L.mcv_delta_rule_workspace_bytes(B, T, Hk, Hv, Dk, Dv)
    ws = _workspace(_GEMM_COUNTER_BYTES + nbytes, q.device, stream) if nbytes else None      # behind the counters
    rc = L.mcv_delta_rule(*qa, *ka, *va, *gates, state.data_ptr() if state is not None else _NULL, state_out.data_ptr(),
                          state_index.data_ptr() if state_index is not None else _NULL, n_states,
                          cu.data_ptr() if cu is not None else _NULL, B, T, Hk, Hv, Dk, Dv,
                          Dk ** -0.5 if scale is None else scale, 1 if normalize else 0, out.data_ptr(),
                          ws.data_ptr() + _GEMM_COUNTER_BYTES if nbytes else _NULL, nbytes, _stream(stream))
    if rc:
        _check(rc, who)
    return out, state_out


def gated_delta_rule(q, k, v, g, beta, state=None, *, cu_seqlens=None, scale=None, normalize=False, state_index=None,
                     out=None, state_out=None, stream=None):
    """The gated delta rule over whole sequences: q, k fp16 [T, Hk, Dk], v fp16 [T, Hv,
    Dv], g (the decay's logarithm) and beta fp32 [T, Hv], state fp32 [B, Hv, Dk, Dv]
    (None: zeros).  Per token, with S the state of its sequence and value head:
    S <- exp(g) S;  S <- S + k (beta (v - S^T k))^T;  out = scale S^T q.

    cu_seqlens int32 [B + 1] on the device: sequence b is tokens cu[b] .. cu[b + 1] - 1
    (none: its state is copied); None: one sequence.  normalize divides q and k by
    sqrt(|.|^2 + 1e-6).  state_index int32 [B] picks each sequence's row of a pool
    of states, updated in place unless state_out is given.  Returns (out fp16
    [T, Hv, Dv], state_out); state_out may be `state`."""
    if q.dim() != 3 or v.dim() != 3:
        raise McvError("gated_delta_rule: q, k and v must be [T, heads, D]")
    B = 1
    if cu_seqlens is not None:
        if cu_seqlens.dtype != _torch().int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or \
                not cu_seqlens.is_contiguous():
            raise McvError("gated_delta_rule: cu_seqlens must be contiguous int32 [B + 1]")
        B = cu_seqlens.numel() - 1
    return _delta("gated_delta_rule", q, k, v, g, beta, state, cu_seqlens, B, scale, normalize, state_index, out,
                  state_out, stream)


def gated_delta_rule_step(q, k, v, g, beta, state, *, scale=None, normalize=False, state_index=None, out=None,
                          state_out=None, stream=None):
    """gated_delta_rule of one token for each of B sequences: q, k fp16 [B, Hk, Dk], v fp16
    [B, Hv, Dv], g and beta fp32 [B, Hv]; the state is updated in place unless state_out is given."""
    if q.dim() != 3 or v.dim() != 3:
        raise McvError("gated_delta_rule_step: q, k and v must be [B, heads, D]")
    return _delta("gated_delta_rule_step", q, k, v, g, beta, state, None, q.shape[0], scale, normalize, state_index, out,
                  state if state_out is None else state_out, stream)


def _cache(who, k_cache, v_cache, Hkv, D):
    """Pointer and strides of both caches, fp16 [pages][page_size][Hkv][D]."""
    got = []
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        s = t.stride()
        if t.dtype != _torch().float16 or len(s) != 4 or t.shape[2] != Hkv or t.shape[3] != D or s[3] != 1 or \
                t.shape != k_cache.shape:
            raise McvError(f"{who}: {name} must be fp16 [pages, page_size, {Hkv}, {D}] with contiguous heads, both caches "
                           f"of one shape, got {t.dtype} {tuple(t.shape)}")
        got.append((t.data_ptr(), s[0], s[1], s[2]))
    return got


def paged_attention_decode(q, k_cache, v_cache, block_table, seq_lens, *, scale=None, max_seq_len=None, out=None,
                           stream=None):
    """Attention of one new token per sequence over a paged cache: q fp16 [B, Hq, D], caches
    fp16 [pages, page_size, Hkv, D] (page, token and head strides: a permuted view of
    another order will do), block_table int32 [B, width], seq_lens int32 [B] (the new
    token's own key among them).  Query head h reads cache head h // (Hq / Hkv).

    Token t lies in row t % page_size of page block_table[b, t // page_size]; a page
    number outside the cache is left out like a masked token, and a sequence of
    length 0 gives zeros.  max_seq_len, at most width * page_size (the default),
    bounds the lengths and sets how the work is split; pass the longest length
    known.  Returns out fp16 [B, Hq, D]."""
    who = "paged_attention_decode"
    torch = _torch()
    if q.dim() != 3 or k_cache.dim() != 4:
        raise McvError(f"{who}: q must be [B, Hq, D] and the caches [pages, page_size, Hkv, D]")
    B, Hq, D = q.shape
    pages, page_size, Hkv, _ = k_cache.shape
    qa = _heads(who, "q", q)
    ka, va = _cache(who, k_cache, v_cache, Hkv, D)
    ts = block_table.stride()
    if block_table.dtype != torch.int32 or len(ts) != 2 or block_table.shape[0] != B or \
            (ts[1] != 1 and block_table.shape[1] != 1):
        raise McvError(f"{who}: block_table must be int32 [{B}, width] with contiguous rows")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,) or not seq_lens.is_contiguous():
        raise McvError(f"{who}: seq_lens must be contiguous int32 [{B}]")
    width = block_table.shape[1]
    most = width * page_size if max_seq_len is None else int(max_seq_len)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float16, device=q.device)
    elif out.dtype != torch.float16 or out.shape != (B, Hq, D) or not out.is_contiguous():
        raise McvError(f"{who}: out must be contiguous fp16 [{B}, {Hq}, {D}]")
    _same_device(who, q, k_cache, v_cache, block_table, seq_lens, out)
    L = lib()
    nbytes = L.mcv_paged_attention_workspace_bytes(B, Hq, Hkv, D, most)
    ws = _workspace(nbytes, q.device, stream) if nbytes else None
    rc = L.mcv_paged_attention(*qa, *ka, *va, pages, page_size, block_table.data_ptr(), ts[0], width, seq_lens.data_ptr(),
                               most, B, Hq, Hkv, D, D ** -0.5 if scale is None else scale, out.data_ptr(),
                               ws.data_ptr() if nbytes else _NULL, nbytes, _stream(stream))
    if rc:
        _check(rc, who)
    return out


def rotary_axes_table(rot: int, theta: float, sections, interleaved: bool = True, device="cuda"):
    """(freq fp64 [rot / 2], axis int32 [rot / 2]) for rotary_axes: freq[i] = theta^(-2 i / rot);
    `sections` gives each axis its number of frequencies (their sum rot / 2).  interleaved:
    axis a > 0 has the frequencies a, a + n, a + 2 n ... (n axes) below n sections[a], the first axis
    the rest; else the axes' frequencies follow one another."""
    torch = _torch()
    half, n = rot // 2, len(sections)
    if rot % 2 or sum(sections) != half or min(sections) < 0:
        raise McvError(f"rotary_axes_table: sections {tuple(sections)} must add up to rot / 2 = {rot / 2:g}")
    axis = [0] * half
    if interleaved:
        for a in range(1, n):
            own = range(a, n * sections[a], n)
            if len(own) and own[-1] >= half:
                raise McvError(f"rotary_axes_table: axis {a} does not find {sections[a]} frequencies in turn")
            for i in own:
                axis[i] = a
    else:
        axis = [a for a, m in enumerate(sections) for _ in range(m)]
    freq = [float(theta) ** (-2.0 * i / rot) for i in range(half)]
    return (torch.tensor(freq, dtype=torch.float64, device=device), torch.tensor(axis, dtype=torch.int32, device=device))


def _rotary_args(who, q, k, positions, freq, axis, q_out):
    torch = _torch()
    if q.dim() != 3 or k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise McvError(f"{who}: q and k must be [T, heads, D], got {tuple(q.shape)} and {tuple(k.shape)}")
    T, Hq, D = q.shape
    if positions.dtype != torch.int64 or positions.dim() != 2 or positions.shape[1] != T:
        raise McvError(f"{who}: positions must be int64 [axes, {T}]")
    half = freq.numel()
    if freq.dtype != torch.float64 or not freq.is_contiguous() or axis.dtype != torch.int32 or axis.numel() != half or \
            not axis.is_contiguous():
        raise McvError(f"{who}: freq must be contiguous fp64 [rot / 2] and axis contiguous int32 of its length")
    if q_out is None:
        q_out = torch.empty((T, Hq, D), dtype=torch.float16, device=q.device)
    elif q_out.shape != q.shape:
        raise McvError(f"{who}: q_out must be {tuple(q.shape)}")
    _same_device(who, q, k, positions, freq, axis, q_out)
    ps = positions.stride()
    where = (positions.data_ptr(), ps[0], ps[1], positions.shape[0], freq.data_ptr(), axis.data_ptr(), T, Hq, k.shape[1], D,
             2 * half)
    return where, q_out


def rotary_axes(q, k, positions, freq, axis, *, q_out=None, k_out=None, stream=None):
    """Rotary positions with several axes: the pair (x[i], x[i + rot / 2]) of the first rot =
    2 freq.numel() elements of every head turns by positions[axis[i], t] freq[i] (in 64
    bits), the rest is copied.  q fp16 [T, Hq, D], k fp16 [T, Hkv, D], positions int64
    [axes, T], freq and axis as rotary_axes_table gives them.  Returns (q_out, k_out);
    q_out = q and k_out = k work in place."""
    who = "rotary_axes"
    where, q_out = _rotary_args(who, q, k, positions, freq, axis, q_out)
    T = where[6]
    if k_out is None:
        k_out = _torch().empty(k.shape, dtype=_torch().float16, device=k.device)
    elif k_out.shape != k.shape:
        raise McvError(f"{who}: k_out must be {tuple(k.shape)}")
    _same_device(who, q, k_out)
    if T:
        rc = lib().mcv_rotary_axes(*_heads(who, "q", q), *_heads(who, "k", k), *where, *_heads(who, "q_out", q_out),
                                   *_heads(who, "k_out", k_out), _stream(stream))
        if rc:
            _check(rc, who)
    return q_out, k_out


def rotary_axes_cached(q, k, v, positions, freq, axis, k_cache, v_cache, slots, *, q_out=None, stream=None):
    """rotary_axes whose rotated k goes, with v fp16 [T, Hkv, D], into the paged caches fp16
    [pages, page_size, Hkv, D]: token t to row slots[t] % page_size of page slots[t] //
    page_size (int64 [T]; a slot outside the cache, such as -1 for a padded token, is
    written nowhere; no two tokens may share one).  Returns q_out."""
    who = "rotary_axes_cached"
    torch = _torch()
    where, q_out = _rotary_args(who, q, k, positions, freq, axis, q_out)
    T, Hkv, D = where[6], where[8], where[9]
    if k_cache.dim() != 4 or v.shape != k.shape:
        raise McvError(f"{who}: v must be {tuple(k.shape)} and the caches [pages, page_size, {Hkv}, {D}]")
    if slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
        raise McvError(f"{who}: slots must be contiguous int64 [{T}]")
    ka, va = _cache(who, k_cache, v_cache, Hkv, D)
    _same_device(who, q, v, k_cache, v_cache, slots)
    if T:
        rc = lib().mcv_rotary_axes_cached(*_heads(who, "q", q), *_heads(who, "k", k), *_heads(who, "v", v), *where,
                                          *_heads(who, "q_out", q_out), *ka, *va, k_cache.shape[0], k_cache.shape[1],
                                          slots.data_ptr(), _stream(stream))
        if rc:
            _check(rc, who)
    return q_out
