"""What a serving step needs around the compressed cache: its block tables and slots from the lengths
of its requests, rotary positions, and layers whose pages keep 16-bit keys and values.

The pages of such layers are ``key_cache`` and ``value_cache`` ``(num_blocks, block_size, H_kv, D)`` of
any strides between rows (two tensors, or views of one), fp16 or bf16; block tables, slots and sequence
lengths are those of the compressed pages (the reference's vLLM backend has the compressed form only:
src/flashquant/vllm/impl.py:220-263, 362-395).  As everywhere in this package there is no CPU branch.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N
from .kernels import _DENSE, _contig, _host, _workspace

_HEAD = 32768  # bytes at the start of a decode workspace that are zero between calls
_LAYOUTS = {"half": 0, "interleaved": 1}
_INTS = (torch.int32, torch.int64)
_MOST = 2 ** 31 - 1  # (ctypes keeps the low bits of a larger int)


def _layout(name: str) -> int:
    try:
        return _LAYOUTS[name]
    except (KeyError, TypeError):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {name!r}") from None


# --------------------------------------------------------------------------------------
# block tables and slots
# --------------------------------------------------------------------------------------

class PagedStepPlan(NamedTuple):
    """What ``plan_paged_step`` returns; the names are those of the other entry points' arguments."""
    seq_lens: torch.Tensor       # (R,) int32: context and new tokens
    cu_seqlens_q: torch.Tensor   # (R + 1,) int32
    slot_mapping: torch.Tensor   # (max_tokens,) int64, -1 behind the last token
    positions: torch.Tensor      # (max_tokens,) int64, -1 behind the last token
    served: torch.Tensor         # (R,) bool
    free_count: torch.Tensor     # (1,) int32


def _pool_args(block_table, free_blocks, free_count, free_count_out):
    N.require_cuda(block_table, free_blocks, free_count, free_count_out)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or \
            (block_table.shape[1] > 1 and block_table.stride(1) != 1) or \
            (block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table must be int32 (num_requests, width) with adjacent entries")
    if free_blocks.dtype != torch.int32 or free_blocks.dim() != 1 or not free_blocks.is_contiguous():
        raise ValueError("free_blocks must be a contiguous int32 vector")
    for t in (free_count, free_count_out):
        if t is not None and (t.dtype != torch.int32 or t.numel() != 1):
            raise ValueError("free_count must hold one int32")
    for t in (free_blocks, free_count, free_count_out):
        if t is not None and t.device != block_table.device:
            raise ValueError("all tensors must be on one device")


def _lens(t, n, device, name):
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in _INTS:
        raise ValueError(f"{name} must hold one int32 or int64 per row of block_table")
    if t.dtype == torch.int64:  # what does not fit stays too long, or negative
        t = t.clamp(-1, _MOST)
    return _contig(t.to(device=device, dtype=torch.int32))


def plan_paged_step(context_lens, query_lens, block_table, free_blocks, free_count, block_size: int,
                    max_tokens: int, *, free_count_out: Optional[torch.Tensor] = None) -> PagedStepPlan:
    """Block tables, slots and positions of a step from the lengths of its requests, in one launch.

    ``context_lens`` ``(R,)`` tokens of a request that are cached, ``query_lens`` its new ones;
    ``block_table`` ``(R, width)`` int32 holds the pages of the former, those of the latter are written
    behind them.  They come off the top of the stack ``free_blocks[:free_count]``, requests in order.
    ``max_tokens`` is the length of ``slot_mapping`` and ``positions``; entries behind the last token
    are -1, which the appends skip (a padded step).  ``free_count_out`` may be ``free_count``.

    A request is served if the pages and slots of all requests up to and including it can be had, or if
    it has no new tokens; from the first that is not, only those without new tokens are.  A negative
    length, or more pages than a row holds, is not served and takes nothing.  At most 4096 requests.

    The tokens' rows are compact, request ``i``'s from ``cu_seqlens_q[i]`` on: the decodes, which take a row of
    ``q`` per row of ``block_table``, are given ``q[cu_seqlens_q[:-1]]`` (cut to ``max_tokens - 1``), unless every
    request is known to be served with one token.
    """
    r = _host().plan_paged_step(context_lens, query_lens, block_table, free_blocks, free_count, block_size,
                                max_tokens, free_count_out)
    if r is not None:
        return PagedStepPlan._make(r) if type(r) is tuple else N.check(r)
    N.require_cuda(context_lens, query_lens)
    _pool_args(block_table, free_blocks, free_count, free_count_out)
    dev, (n, width) = block_table.device, block_table.shape
    if max_tokens < 0 or not 1 <= block_size <= _MOST:
        raise ValueError("max_tokens must not be negative, block_size positive and below 2^31")
    context, query = (_lens(t, n, dev, m) for t, m in ((context_lens, "context_lens"), (query_lens, "query_lens")))
    i32 = dict(dtype=torch.int32, device=dev)
    plan = PagedStepPlan(torch.empty(n, **i32), torch.empty(n + 1, **i32),
                         torch.empty(max_tokens, dtype=torch.int64, device=dev),
                         torch.empty(max_tokens, dtype=torch.int64, device=dev),
                         torch.empty(n, dtype=torch.bool, device=dev),
                         torch.empty(1, **i32) if free_count_out is None else free_count_out)
    with torch.cuda.device(dev):
        N.check(N.load().fq_plan_paged_step(
            N.ptr(context), N.ptr(query), n, N.ptr(block_table), max(block_table.stride(0), width), width,
            int(block_size), N.ptr(free_blocks), free_blocks.numel(), N.ptr(free_count), int(max_tokens),
            N.ptr(plan.seq_lens), N.ptr(plan.cu_seqlens_q), N.ptr(plan.slot_mapping), N.ptr(plan.positions),
            N.ptr(plan.served), N.ptr(plan.free_count), N.stream_ptr(dev)))
    return plan


def release_pages(finished, context_lens, block_table, free_blocks, free_count, block_size: int, *,
                  free_count_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Puts the pages of the requests with ``finished`` ``(R,)`` bool on the stack ``free_blocks`` (in
    place), in order, and returns its new height ``(1,)`` int32 (``free_count_out``, which may be
    ``free_count``).  The rows of ``block_table`` are left as they are: the caller's next lengths for
    them start at zero."""
    r = _host().release_pages(finished, context_lens, block_table, free_blocks, free_count, block_size,
                              free_count_out)
    if r is not None:
        return r if type(r) is not int else N.check(r)
    N.require_cuda(finished, context_lens)
    _pool_args(block_table, free_blocks, free_count, free_count_out)
    dev, (n, width) = block_table.device, block_table.shape
    if finished.dim() != 1 or finished.shape[0] != n or finished.dtype != torch.bool:
        raise ValueError("finished must hold one bool per row of block_table")
    if not 1 <= block_size <= _MOST:
        raise ValueError("block_size must be positive and below 2^31")
    context, finished = _lens(context_lens, n, dev, "context_lens"), _contig(finished.to(dev))
    out = torch.empty(1, dtype=torch.int32, device=dev) if free_count_out is None else free_count_out
    with torch.cuda.device(dev):
        N.check(N.load().fq_release_pages(
            N.ptr(finished), N.ptr(context), n, N.ptr(block_table), max(block_table.stride(0), width), width,
            int(block_size), N.ptr(free_blocks), free_blocks.numel(), N.ptr(free_count), N.ptr(out),
            N.stream_ptr(dev)))
    return out


# --------------------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------------------

def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 8192, low: float = 1.0, high: Optional[float] = None,
                       device=None) -> Tuple[torch.Tensor, float]:
    """``(frequencies, scale)`` for the rotary entry points: ``rotary_dim / 2`` angles per position in
    fp64, ``base ** (-2j / rotary_dim)``, and what rotated values are multiplied with.

    ``scaling`` for contexts ``factor`` times ``original_length``:
      None          as they are
      "linear"      all divided by ``factor``
      "ntk"         another base, ``base * factor ** (rotary_dim / (rotary_dim - 2))``: the slowest is
                    divided by ``factor``, the fastest kept
      "wavelength"  kept where ``original_length`` holds ``high`` (4) or more turns, divided where it holds
                    ``low`` or fewer, blended by the number of turns between
      "yarn"        the same blended linearly over the index, between those that make ``high`` (32) and ``low``
                    turns, the latter at most ``rotary_dim - 1``: it may lie behind the last frequency, which is
                    then not fully divided; values are multiplied by ``0.1 ln factor + 1``
    """
    if high is None:
        high = 32.0 if scaling == "yarn" else 4.0
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (base > 1.0 and factor >= 1.0 and original_length > 0 and 0 < low < high):
        raise ValueError("base above 1, factor at least 1, original_length positive and 0 < low < high are needed")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("'ntk' needs more than one frequency")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    j = torch.arange(half, dtype=torch.float64)
    freq = torch.exp(j * (-2.0 * math.log(base) / rotary_dim))
    scale = 1.0
    if scaling in ("linear", "wavelength", "yarn"):
        turns = original_length * freq / (2.0 * math.pi)
        if scaling == "linear":
            keep = torch.zeros_like(freq)
        elif scaling == "wavelength":
            keep = ((turns - low) / (high - low)).clamp(0, 1)
        else:
            def index(n):  # of the frequency that makes n turns
                return half * math.log(original_length / (n * 2.0 * math.pi)) / math.log(base)
            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rotary_dim - 1)
            keep = 1.0 - ((j - first) / max(last - first, 1e-3)).clamp(0, 1)
            scale = 0.1 * math.log(factor) + 1.0
        freq = freq * keep + freq / factor * (1.0 - keep)
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return freq.to(device) if device is not None else freq, scale


def _rows(t, name, tokens=None, dtype=None):
    """``t`` (tokens, heads, D) with adjacent values of a head, copied only if it has none."""
    if t.dim() != 3 or (tokens is not None and t.shape[0] != tokens) or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be (tokens, heads, head_dim) of the type and number of tokens of the others")
    return t if t.shape[2] <= 1 or t.stride(2) == 1 else t.contiguous()


def _own_rows(t) -> bool:
    """No two rows (of the last dimension) of ``t`` share memory."""
    if t.numel() == 0:
        return True
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return False
    extent = t.shape[-1]
    for s, n in sorted((s, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        if s < extent:
            return False
        extent += s * (n - 1)
    return True


def _rotary_args(head_dim, tokens, positions, frequencies, dev):
    if positions.dim() != 1 or positions.shape[0] != tokens or positions.dtype not in _INTS:
        raise ValueError("positions must hold one int32 or int64 per token")
    if frequencies.dim() != 1 or 2 * frequencies.shape[0] > head_dim:
        raise ValueError("frequencies must be a vector of at most head_dim / 2")
    if positions.device != dev:
        raise ValueError("all tensors must be on one device")
    return _contig(positions), _contig(frequencies.to(device=dev, dtype=torch.float64))


def _out_rows(t, like, name):
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device or not _own_rows(t):
        raise ValueError(f"{name} must have the shape, type and device of its input, and rows of its own")
    return t


def _strides(*values):
    return (C.c_int64 * len(values))(*values)


def rotary_embed(q, k, positions, frequencies, *, layout: str = "half", scale: float = 1.0, inverse: bool = False,
                 out=None):
    """Rotary positions of ``q`` ``(tokens, H_q, D)`` and ``k`` ``(tokens, H_kv, D)`` (or None), in fp32,
    fp16 or bf16: pair ``j`` of every head is turned by ``positions[i] * frequencies[j]`` and multiplied by
    ``scale``; values behind the ``2 * len(frequencies)`` first of a head are kept.  Returns ``(q, k)``.

    ``layout``: pairs are ``(x[j], x[j + len(frequencies)])`` ("half") or ``(x[2j], x[2j + 1])``
    ("interleaved").  ``inverse``: by the negative angle, which takes a key back to position zero, or a
    gradient to the input.  ``out``: ``(q_out, k_out)``, which may be ``(q, k)``; tokens with a negative
    position are not written.  Angles are taken in 64 bits, any position may be given.
    """
    code = _layout(layout)
    r = _host().rotary_embed(q, k, positions, frequencies, code, scale, inverse, out)
    if r is not None:
        return r if type(r) is not int else N.check(r)
    N.require_cuda(q, k, positions)
    dtype = N.dtype_code(q.dtype)
    q = _rows(q, "q")
    n, hq, d = q.shape
    dev = q.device
    if k is not None:
        if k.device != dev:
            raise ValueError("all tensors must be on one device")
        k = _rows(k, "k", n, q.dtype)
        if k.shape[2] != d:
            raise ValueError("q and k must have one head_dim")
    pos, freq = _rotary_args(d, n, positions, frequencies, dev)
    q_out, k_out = (None, None) if out is None else out
    if k is None and k_out is not None:
        raise ValueError("k_out without k")
    q_out = _out_rows(q_out, q, "q_out")
    k_out = None if k is None else _out_rows(k_out, k, "k_out")
    ks, ko = ((0, 0), (0, 0)) if k is None else (k.stride()[:2], k_out.stride()[:2])
    with torch.cuda.device(dev):
        N.check(N.load().fq_rotary_embed(
            N.ptr(q), N.ptr(k), dtype, n, hq, 0 if k is None else k.shape[1], d, 2 * freq.shape[0],
            _strides(*q.stride()[:2], *ks, *q_out.stride()[:2], *ko), N.ptr(pos), int(pos.dtype == torch.int64),
            N.ptr(freq), code, float(scale), int(bool(inverse)), N.ptr(q_out), N.ptr(k_out), N.stream_ptr(dev)))
    return q_out, k_out


def _cache(t, name, like):
    if t.dim() != 4 or t.dtype != like.dtype or t.device != like.device or not _own_rows(t):
        raise ValueError(f"{name} must be (num_blocks, block_size, H_kv, D) of the type of the others, "
                         "rows of adjacent values that are its own")
    return t


def rotary_append_dense(q, key, value, key_cache, value_cache, slot_mapping, positions=None, frequencies=None, *,
                        layout: str = "half", scale: float = 1.0, q_out: Optional[torch.Tensor] = None):
    """Writes ``key`` and ``value`` ``(tokens, H_kv, D)`` of new tokens to the rows ``slot_mapping`` of 16-bit
    pages, with rotary positions on ``key`` and ``q`` ``(tokens, H_q, D)`` as ``rotary_embed``, in one
    launch.  Returns the rotated ``q`` (``q_out``, which may be ``q``); None if ``q`` is None.

    Without ``positions`` and ``frequencies`` nothing is rotated (and ``q`` must be None).  A slot is
    ``block * block_size + token``, as in ``tq4_compress_append``; negative ones, and those beyond the pages, are
    skipped, the others are distinct.  A token with a negative position has its values stored, not its queries
    and keys.
    """
    code = _layout(layout)
    r = _host().rotary_append_dense(q, key, value, key_cache, value_cache, slot_mapping, positions, frequencies,
                                    code, scale, q_out)
    if r is not None:
        return r if type(r) is not int else N.check(r)
    N.require_cuda(q, key, value, key_cache, value_cache, slot_mapping, positions)
    if key.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {key.dtype}; pages are float16 or bfloat16")
    key = _rows(key, "key")
    n, h, d = key.shape
    value = _rows(value, "value", n, key.dtype)
    dev = key.device
    _cache(key_cache, "key_cache", key)
    _cache(value_cache, "value_cache", key)
    blocks, bs = key_cache.shape[:2]
    if value.shape != key.shape or tuple(key_cache.shape) != (blocks, bs, h, d) or value_cache.shape != key_cache.shape:
        raise ValueError("key and value, and both caches, must have the same heads and head_dim")
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != n or slot_mapping.dtype not in _INTS:
        raise ValueError("slot_mapping must hold one int32 or int64 per token")
    if any(t.device != dev for t in (value, slot_mapping)):
        raise ValueError("all tensors must be on one device")
    if (positions is None) != (frequencies is None) or (positions is None and q is not None):
        raise ValueError("positions and frequencies go together, and q needs them")
    pos = freq = None
    if positions is not None:
        pos, freq = _rotary_args(d, n, positions, frequencies, dev)
    hq = 0
    qs = qo = (0, 0)
    if q is not None:
        if q.device != dev:
            raise ValueError("all tensors must be on one device")
        q = _rows(q, "q", n, key.dtype)
        if q.shape[2] != d:
            raise ValueError("q and key must have one head_dim")
        q_out = _out_rows(q_out, q, "q_out")
        hq, qs, qo = q.shape[1], q.stride()[:2], q_out.stride()[:2]
    elif q_out is not None:
        raise ValueError("q_out without q")
    slots = _contig(slot_mapping)
    with torch.cuda.device(dev):
        N.check(N.load().fq_rotary_append_dense(
            N.ptr(q), N.ptr(key), N.ptr(value), N.dtype_code(key.dtype), n, hq, h, d,
            0 if freq is None else 2 * freq.shape[0],
            _strides(*qs, *key.stride()[:2], *value.stride()[:2], *qo, *key_cache.stride()[:3],
                     *value_cache.stride()[:3]),
            N.ptr(pos), int(pos is not None and pos.dtype == torch.int64), N.ptr(freq), code, float(scale),
            N.ptr(q_out), N.ptr(key_cache), N.ptr(value_cache), max(bs, 1), blocks * bs, N.ptr(slots),
            int(slots.dtype == torch.int64), N.stream_ptr(dev)))
    return q_out


# --------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------

def dense_workspace(device, num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> torch.Tensor:
    """The cached workspace of the current stream for ``split_k_paged_decode_dense`` (word 0: status)."""
    need = N.load().fq_dense_paged_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim)
    return _workspace(torch.device(device), _DENSE, need)


def _call_workspace(device, need: int) -> torch.Tensor:
    """The workspace of a call that is being recorded: its own, so that two recorded graphs never share
    counters; its head is zeroed by every replay."""
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    ws[:_HEAD].zero_()
    return ws


def split_k_paged_decode_dense(q, key_cache, value_cache, block_table, seq_lens, sm_scale: Optional[float] = None, *,
                               window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                               workspace: Optional[torch.Tensor] = None):
    """Decode attention of one query token per sequence over 16-bit pages: ``split_k_paged_decode`` for the
    layers whose cache is not compressed.

    ``q`` ``(num_seqs, H_q, D)``, the caches ``(num_blocks, block_size, H_kv, D)`` of its type (fp16 or
    bf16), ``block_table`` ``(num_seqs, width)`` and ``seq_lens`` int32.  ``window``: each sequence sees its
    last ``window`` tokens (0: all).  ``return_lse``: also the fp32 ``(num_seqs, H_q)`` logarithms of the sums
    of ``exp(sm_scale q k)``.  ``out``: contiguous, at a multiple of 8 bytes.  A sequence without tokens gives zeros
    (and -inf).

    head_dim 64, 96, 128 or 256; block_size a multiple of 16; rows of the caches start at multiples of 16
    bytes; up to 2048 sequences.  Keys and values of visible tokens must be finite; what other rows hold does
    not matter.  A page id out of range is skipped, a length beyond the block table cut, both noted in word 0
    of the workspace (``workspace_status``), the stream's ``dense_workspace`` unless one is given.  ``workspace``: as many
    uint8, the first 32 KiB zero before the first use; one per concurrent call.  A call that is recorded in a graph
    without one has memory of its own, whose status nobody sees: replays that are to be looked at are given one (one per
    graph where graphs run side by side).
    """
    if workspace is None:
        r = _host().dense_decode(q, key_cache, value_cache, block_table, seq_lens, sm_scale, window, out, return_lse)
        if r is not None:
            return r if type(r) is not int else N.check(r)
    N.require_cuda(q, key_cache, value_cache, block_table, seq_lens, out, workspace)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {q.dtype}; pages are float16 or bfloat16")
    if q.dim() != 3:
        raise ValueError("q must be (num_seqs, H_q, D)")
    n, hq, d = q.shape
    dev = q.device
    for t, m in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        if t.dim() != 4 or t.dtype != q.dtype or t.shape[3] != d or (d > 1 and t.stride(3) != 1):
            raise ValueError(f"{m} must be (num_blocks, block_size, H_kv, D) of q's type, rows of adjacent values")
    if value_cache.shape != key_cache.shape:
        raise ValueError("key_cache and value_cache must have the same shape")
    blocks, bs, hkv, _ = key_cache.shape
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block_table and seq_lens must be int32")
    if block_table.dim() != 2 or block_table.shape[0] != n or tuple(seq_lens.shape) != (n,):
        raise ValueError("block_table must be (num_seqs, width), seq_lens (num_seqs,)")
    if any(t is not None and t.device != dev for t in (key_cache, value_cache, block_table, seq_lens, out, workspace)):
        raise ValueError("all tensors must be on one device")
    if window < 0:
        raise ValueError("window must not be negative")
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous uint8 tensor")  # (its numel is taken for its bytes)
    if q.stride(2) != 1 or q.stride(0) % 2 or q.stride(1) % 2 or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    seq_lens = _contig(seq_lens)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty(n, hq, d, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    lse = torch.empty(n, hq, dtype=torch.float32, device=dev) if return_lse else None
    lib = N.load()
    with torch.cuda.device(dev):
        if workspace is None:
            need = lib.fq_dense_paged_decode_workspace_bytes(n, hq, hkv, d)
            workspace = _call_workspace(dev, max(need, _HEAD)) if torch.cuda.is_current_stream_capturing() else \
                dense_workspace(dev, n, hq, hkv, d)
        N.check(lib.fq_dense_paged_decode(
            N.ptr(q), N.dtype_code(q.dtype), q.stride(0), q.stride(1), N.ptr(key_cache), *key_cache.stride()[:3],
            N.ptr(value_cache), *value_cache.stride()[:3], N.ptr(block_table), block_table.stride(0),
            block_table.shape[1], N.ptr(seq_lens), n, hq, hkv, d, bs, blocks, float(sm_scale),
            min(int(window), _MOST), N.ptr(out),
            N.ptr(lse), N.ptr(workspace), workspace.numel(), N.stream_ptr(dev)))
    return (out, lse) if return_lse else out
