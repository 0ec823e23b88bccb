"""Token mixers that stand between a decoder layer's quantised projections, over
the C-ABI in include/mcv_mixers.h: the gated delta rule of the linear-attention
layers, several-axis rotary positions, and attention of one new token or of chunks of
them over a paged key-value cache for the full-attention layers, whose pages are dealt
out and taken back on the device.

Activations and caches are fp16, gates and states fp32.  q, k and v may be
columns of one projection's output: rows and heads have strides, the elements
of one head are contiguous.  A call with stream= runs there, and what it allocates is that
stream's, as under torch.cuda.stream(stream).
"""
from __future__ import annotations

import importlib.util

from . import _GEMM_WS, GEMM_WORKSPACE_BYTES, PKG_DIR, McvError, _made_on, _new_workspace, _stream, _torch, gemm_workspace, lib

# A call's checks and its launch are native (binding/mixers_ext.cpp): the kernels of one
# decoded token take 3 to 5 us, and a call written here with ctypes took 9 to 12.  MI355X,
# one token: delta rule 10.8 us a call, now 4.2; rotary with the cache 12.7, now 4.2.
_BINDING = None


def binding():
    """The loaded native binding; raises McvError if it has not been built."""
    global _BINDING
    if _BINDING is None:
        path = PKG_DIR / "lib" / "_mcv_mixers.so"
        if not path.exists():
            raise McvError(f"HIP library not built: {path} is missing (run __graft_entry__.build())")
        _torch()                                                 # its libraries first
        lib()
        spec = importlib.util.spec_from_file_location("_mcv_mixers", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        most = lib().mcv_paged_attention_workspace_bytes(512, 16, 1, 256, 1 << 20)      # of any call
        mod.bind(McvError, _empty_on, gemm_workspace, _GEMM_WS, GEMM_WORKSPACE_BYTES, most, delta_workspace, _DELTA_WS, *DELTA_WORKSPACE_BYTES,
                 chunk_workspace, _CHUNK_WS, CHUNK_WORKSPACE_BYTES)
        _BINDING = mod
    return _BINDING


def _empty_on(shape, kind: int, device, stream):
    """An output (0 fp16, 1 fp32, 2 int8, 3 int64) of a call on a stream that is not the current one: its memory, so that it is not handed
    out anew while that stream still writes to it, nor written while the current stream still uses what it was."""
    torch = _torch()
    dtype = (torch.float16, torch.float32, torch.int8, torch.int64)[kind]
    make = lambda: torch.empty(shape, dtype=dtype, device=device)     # noqa: E731
    return _made_on(make, torch.device(device), _stream(stream), stream)


# The delta rule's workspace comes in two sizes, for some 800 tokens of 16 heads of 128 and for all that a pass takes of
# any length, so that a stream holds one of each at most.  Its two launches read what the first has written, and calls
# that let other threads run launch on the GEMM's: it has buffers of its own.
DELTA_WORKSPACE_BYTES = (16 << 20, 192 << 20)
_DELTA_WS: dict = {}            # (device, stream, bytes) -> workspace
_DELTA_WS_CAPTURE: dict = {}    # the same -> (capture id, workspace of that graph)


def delta_workspace(nbytes: int, device, stream=None):
    """The workspace of gated_delta_rule for calls on one stream, of any content; kept, and recorded by
    graphs, as gemm_workspace's is."""
    torch = _torch()
    dev = torch.device(device)
    handle = _stream(stream)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), handle,
           next((size for size in DELTA_WORKSPACE_BYTES if nbytes <= size), nbytes))
    ws = _DELTA_WS.get(key)
    if ws is not None:
        return ws
    return _new_workspace(_DELTA_WS, _DELTA_WS_CAPTURE, key, 0, 0, dev, handle, stream)


# The chunks' parts of a long cache meet in a workspace that is as large for any call as for the largest, so that a stream
# holds one; its counters start and end at zero.
CHUNK_WORKSPACE_BYTES = 144 << 20
_CHUNK_COUNTER_BYTES = 8192
_CHUNK_WS: dict = {}            # (device, stream, bytes) -> workspace
_CHUNK_WS_CAPTURE: dict = {}    # the same -> (capture id, workspace of that graph)


def chunk_workspace(nbytes: int, device, stream=None):
    """The workspace of paged_attention_chunk for calls on one stream; kept, and recorded by graphs, as
    gemm_workspace's is."""
    torch = _torch()
    dev = torch.device(device)
    handle = _stream(stream)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), handle, max(nbytes, CHUNK_WORKSPACE_BYTES))
    ws = _CHUNK_WS.get(key)
    if ws is not None:
        return ws
    return _new_workspace(_CHUNK_WS, _CHUNK_WS_CAPTURE, key, _CHUNK_COUNTER_BYTES, _CHUNK_COUNTER_BYTES, dev, handle, stream)


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
    return (_BINDING or binding()).delta("gated_delta_rule", q, k, v, g, beta, state, cu_seqlens, False, scale, normalize,
                                         state_index, out, state_out, stream)


def gated_delta_rule_step(q, k, v, g, beta, state, *, scale=None, normalize=False, state_index=None, out=None,
                          state_out=None, stream=None):
    """gated_delta_rule of one token for each of B sequences: q, k fp16 [B, Hk, Dk], v fp16
    [B, Hv, Dv], g and beta fp32 [B, Hv]; the state is updated in place unless state_out is given.
    B may be 0."""
    return (_BINDING or binding()).delta("gated_delta_rule_step", q, k, v, g, beta, state, None, True, scale, normalize,
                                         state_index, out, state if state_out is None else state_out, stream)


def paged_attention_decode(q, k_cache, v_cache, block_table, seq_lens, *, scale=None, max_seq_len=None, out=None,
                           stream=None):
    """Attention of one new token per sequence over a paged cache: q fp16 [B, Hq, D], caches
    fp16 [pages, page_size, Hkv, D] (page, token and head strides: a permuted view of
    another order will do), block_table int32 [B, width], seq_lens int32 [B] (the new
    token's own key among them).  Query head h reads cache head h // (Hq / Hkv).

    Token t lies in row t % page_size of page block_table[b, t // page_size]; a page
    number outside the cache is left out like a masked token, and a sequence of
    length 0 gives zeros (and a batch of none an empty result).  max_seq_len, at most width * page_size (the default),
    bounds the lengths.  Returns out fp16 [B, Hq, D]."""
    return (_BINDING or binding()).paged(q, k_cache, v_cache, block_table, seq_lens, scale, max_seq_len, out, stream)


def paged_attention_chunk(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens=None, *, scale=None, max_seq_len=None,
                          out=None, positions=None, stream=None):
    """Attention of chunks of new tokens over a paged cache that holds them already (rotary_axes_cached): q fp16 [T, Hq, D],
    sequence b's rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (int32 [B + 1] on the device; None: T / B rows each) its last
    tokens.  Each sees the tokens of its sequence up to and with itself.  Caches, block_table, seq_lens int32 [B] (the new
    tokens among them) and max_seq_len as for paged_attention_decode.

    positions int64 [T], paged_append's: each sequence's new tokens are at positions[cu_seqlens[b]] and on, in place of the
    last ones of seq_lens[b].  So tokens that had room in an append without room for all see what they should; those that
    had none see all of their sequence.

    Prompts, their chunks and single tokens may share a call.  A row that sees nothing gives zeros, a row of no sequence is
    left as it is, and so is all of `out` that no row writes.  `out` may be a contiguous q.  The softmax's
    weights are rounded to fp16 (paged_attention_decode keeps them in two parts).  Returns out fp16 [T, Hq, D]."""
    return (_BINDING or binding()).chunk(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, scale, max_seq_len, out, positions, stream)


def paged_append(block_table, seq_lens, cu_seqlens=None, page_size=16, *, tokens=None, free_pages=None, free_count=None,
                 seq_lens_out=None, free_count_out=None, slots=None, positions=None, stream=None):
    """Room in a paged cache for new tokens: sequence b, of seq_lens[b] tokens, gets the rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1 of a packed batch of `tokens` rows (None: the rows of `slots`; without cu_seqlens else one each) as
    its next.

    Pages that a sequence lacks are taken from the top of the stack free_pages int32 [n], free_count int32 [1] and written
    into block_table int32 [B, width]; without free_pages the table is complete.  Returns (slots int64 [tokens], where
    rotary_axes_cached writes each token, -1 for a row of no sequence or a token without room; positions int64 [tokens];
    seq_lens_out).  seq_lens and free_count are updated in place unless seq_lens_out and free_count_out are given; a
    count below zero says how many pages were lacking, and lengths then end where the room does."""
    return (_BINDING or binding()).append(block_table, seq_lens, cu_seqlens, page_size, tokens, free_pages, free_count, seq_lens_out,
                                          free_count_out, slots, positions, stream)


def paged_truncate(block_table, seq_lens, keep, page_size, free_pages, free_count, *, seq_lens_out=None, free_count_out=None,
                   stream=None):
    """The reverse of paged_append: sequence b keeps its first keep[b] tokens (int32 [B]; None: no sequence keeps any), and its
    pages behind them go on top of the free list.  seq_lens and free_count are updated in place unless seq_lens_out and
    free_count_out are given.  Returns seq_lens_out."""
    return (_BINDING or binding()).truncate(block_table, seq_lens, keep, page_size, free_pages, free_count, seq_lens_out,
                                            free_count_out, stream)


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


def rotary_axes(q, k, positions, freq, axis, *, q_out=None, k_out=None, stream=None):
    """Rotary positions with several axes: the pair (x[i], x[i + rot / 2]) of the first rot =
    2 freq.numel() elements of every head turns by positions[axis[i], t] freq[i] (in 64
    bits), the rest is copied.  q fp16 [T, Hq, D], k fp16 [T, Hkv, D], positions int64
    [axes, T], freq and axis as rotary_axes_table gives them.  Returns (q_out, k_out);
    q_out = q and k_out = k work in place."""
    return (_BINDING or binding()).rotary(q, k, positions, freq, axis, q_out, k_out, stream)


def rotary_axes_cached(q, k, v, positions, freq, axis, k_cache, v_cache, slots, *, q_out=None, stream=None):
    """rotary_axes whose rotated k goes, with v fp16 [T, Hkv, D], into the paged caches fp16
    [pages, page_size, Hkv, D]: token t to row slots[t] % page_size of page slots[t] //
    page_size (int64 [T]; a slot outside the cache, such as -1 for a padded token, is
    written nowhere; no two tokens may share one).  Returns q_out."""
    return (_BINDING or binding()).rotary_cached(q, k, positions, freq, axis, q_out, v, k_cache, v_cache, slots, stream)
