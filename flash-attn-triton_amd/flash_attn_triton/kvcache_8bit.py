"""Serving over a paged KV cache held in 8 bits.

Three operators, in the order a serving step calls them:

* ``paged_kvcache_slots`` gives the next tokens of a batch of requests their
  pages and slots, on the GPU from the requests' lengths;
* ``kvcache_append_8bit`` quantizes new K / V rows into those slots;
* ``flash_attn_with_kvcache_8bit`` is ``flash_attn_with_kvcache`` over the
  8-bit cache, for batched or packed queries.

The cache: ``k_cache`` and ``v_cache`` are (num_pages, page_size, nheads_k,
headdim) of ``torch.float8_e4m3fn`` or ``torch.float8_e5m2``, each with a scale
per block of tokens and head, ``k_scale`` / ``v_scale`` (num_pages, page_size //
block, nheads_k) of ``torch.float8_e8m0fnu``: a value is its number times the
block's scale, which is a power of two.  ``block`` is whatever the scale's shape
says: a power of two of at least 16 that divides page_size.  headdim is 64, 128
or 256.  Any strides do whose rows are 16-byte aligned; the caches are used in
place, never copied.

Each operator takes ``validate``.  With True (the default) device arrays are
checked as ``flash_attn_with_kvcache`` checks them, which costs one wait of the
host per call and is refused while a stream is being captured.  With False
nothing is read back, so the call is asynchronous and can be captured into a
graph; the kernels stay within the tensors whatever the arrays hold (what is
skipped or clamped is said at each operator).

The operators are for inference: inputs that require gradients are refused
while gradients are enabled.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _native
from ._checks import Deferred
from .flash_attn_interface import _normalize_alibi
from .triton_kernel.attention_kernel import _kernel_ready, _needs_grad

_STORES = (torch.float8_e4m3fn, torch.float8_e5m2)
_INTS = (torch.int32, torch.int64)
_HEAD_DIMS = (64, 128, 256)


class _Here:
    """The context of a call whose tensors are on the current device."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(device):
    """``torch.cuda.device(device)`` where it is not the current one (entering it
    takes 1.3 us of the host's time, a tenth of a small call)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _int32(t):
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _lengths(name, t, batch, device):
    """Checks ``t``: one integer per sequence (any number of them: None) on ``device``."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _INTS or t.ndim != 1:
        raise ValueError(f"{name} must be a one-dimensional int32 or int64 tensor")
    if batch is not None and t.shape[0] != batch:
        raise ValueError(f"{name} must contain one value per sequence")
    if t.device != device:
        raise ValueError(f"{name} must be on the same CUDA device")


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    """The checks of the cache's own tensors; returns the tokens of a scale block."""
    shape, sshape = k_cache.shape, k_scale.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be rank-4 tensors of the same shape")
    if k_cache.dtype not in _STORES or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be float8_e4m3fn or both float8_e5m2")
    pages, page, heads, dim = shape
    if k_scale.dtype != torch.float8_e8m0fnu or v_scale.dtype != torch.float8_e8m0fnu:
        raise ValueError("k_scale and v_scale must be float8_e8m0fnu tensors")
    if len(sshape) != 3 or v_scale.shape != sshape or sshape[0] != pages or sshape[2] != heads:
        raise ValueError("k_scale and v_scale must have shape (num_pages, page_size // block, nheads_k)")
    blocks = sshape[1]
    block = page // blocks if blocks else 0
    if block < 16 or block & (block - 1) or block * blocks != page:
        raise ValueError("a scale block must be a power of two of at least 16 tokens that divides page_size")
    if dim not in _HEAD_DIMS:
        raise ValueError("head dimension must be one of 64, 128, or 256")
    if not k_cache.is_cuda:
        raise ValueError("All cache tensors must be CUDA tensors")
    dev = k_cache.device
    if v_cache.device != dev or k_scale.device != dev or v_scale.device != dev:
        raise ValueError("caches and scales must be on the same CUDA device")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1
            or (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2] | k_cache.data_ptr() | v_cache.data_ptr()) % 16):
        raise ValueError("cache rows must be contiguous and 16-byte aligned")
    return block


@functools.lru_cache(maxsize=64)
def _apart(shape, *strides):
    """Whether no two elements of a tensor of ``shape`` share memory, for each of ``strides``."""
    if 0 in shape:
        return True
    for stride in strides:
        end = 0   # offset of the last element of the dimensions so far
        for st, n in sorted((st, n) for st, n in zip(stride, shape) if n > 1):
            if st <= end:
                return False
            end += st * (n - 1)
    return True


def _check_targets(k_cache, v_cache, k_scale, v_scale):
    """What is written must not overlap itself: workgroups would write it at once."""
    if k_cache.numel() and (k_cache.data_ptr() == v_cache.data_ptr() or k_scale.data_ptr() == v_scale.data_ptr()):
        raise ValueError("K and V must not share a cache or scales")
    if not (_apart(k_cache.shape, k_cache.stride(), v_cache.stride())
            and _apart(k_scale.shape, k_scale.stride(), v_scale.stride())):
        raise ValueError("elements of the cache or its scales share memory")


def _check_no_grad(name, *tensors):
    if _needs_grad(*tensors):
        raise ValueError(f"{name} has no backward pass: call it under torch.no_grad()")


def _check_capture(validate):
    if validate and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("validate=True waits for the device, which a capturing stream cannot do: "
                           "pass validate=False")


def paged_kvcache_slots(block_table, cache_seqlens, new_seqlens, free_pages, page_size, max_tokens,
                        free_start=None, validate=True):
    """Pages and slots of the next tokens of a batch of requests.

    Arguments:
        block_table: (batch, max_num_pages) int32, written in place: each
            request's new pages, behind those it has.
        cache_seqlens: (batch,) tokens cached per request.
        new_seqlens: (batch,) tokens that each request gets.
        free_pages: (n,) int32 numbers of free pages, taken in order.
        page_size: int. Tokens per page.
        max_tokens: int. Rows of the packed outputs, at least the sum of
            new_seqlens.
        free_start: (1,) int32, index of free_pages to take pages from (None:
            0); what a call returns goes into the next one.
        validate: check the lengths and the room in the packed rows and
            the block table (see the module's documentation).  With False,
            negative lengths count as 0.
    Return:
        (slot_mapping, positions, cu_seqlens, seqlens, free_start): int64
        (max_tokens,) slots, page * page_size + index in the page, -1 in rows
        past the last request; int32 (max_tokens,) positions in the sequence;
        int32 (batch + 1,) offsets of each request's packed rows; int32 (batch,)
        lengths with the new tokens; int32 (1,).

    Pages go to the requests in order.  Where the free ones do not reach, a
    request that needs any gets none: its slots are -1 (an append skips them),
    its length and its row of the table stay as they were.  That is no error:
    a scheduler compares the returned lengths with the ones it asked for, and
    comes with a new list.  Until then nobody overtakes a refused request: the
    returned index counts the pages needed up to the last request served,
    with those of refused requests in between, and may lie past the list.
    """
    if not isinstance(block_table, torch.Tensor) or block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError("block_table must be an int32 tensor of shape (batch, max_num_pages)")
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor")
    batch, cols = block_table.shape
    dev = block_table.device
    if cols and block_table.stride(1) != 1 or batch > 1 and block_table.stride(0) < cols:
        raise ValueError("block_table must have contiguous rows that do not overlap")
    _lengths("cache_seqlens", cache_seqlens, batch, dev)
    _lengths("new_seqlens", new_seqlens, batch, dev)
    if free_pages.ndim != 1 or free_pages.dtype != torch.int32 or free_pages.device != dev:
        raise ValueError("free_pages must be a one-dimensional int32 tensor on the same CUDA device")
    if free_start is not None and (free_start.numel() != 1 or free_start.dtype != torch.int32
                                   or free_start.device != dev):
        raise ValueError("free_start must be one int32 on the same CUDA device")
    page_size, max_tokens = int(page_size), int(max_tokens)
    if page_size < 1:
        raise ValueError("page_size must be positive")
    if max_tokens < 0:
        raise ValueError("max_tokens must be non-negative")
    _check_capture(validate)
    with _on(dev):
        if validate:
            chk = Deferred()
            bad = ValueError("cache_seqlens must contain valid lengths for every request")
            chk.check_range(cache_seqlens, 0, cols * page_size, bad)
            chk.check_range(new_seqlens, 0, None, ValueError("new_seqlens must be non-negative"))
            chk.check_range(new_seqlens, None, cols * page_size,
                            ValueError("new tokens do not fit in the block table"), plus=cache_seqlens)
            if batch:
                total = chk.value(new_seqlens.sum())
            if free_start is not None:
                chk.check_range(free_start, 0, None, ValueError("free_start must be non-negative"))
            values = chk.flush()
            if batch and values[total] > max_tokens:
                raise ValueError("max_tokens must cover the new tokens of every request")
        # One allocation for the int32 outputs.
        slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        positions, cu, seqlens, end = torch.empty(
            max_tokens + 2 * batch + 2, dtype=torch.int32, device=dev).split_with_sizes(
                (max_tokens, batch + 1, batch, 1))
        _native.kvcache_slots(block_table, _int32(cache_seqlens), _int32(new_seqlens), free_pages.contiguous(),
                              free_start, page_size, slots, positions, cu, seqlens, end)
    return slots, positions, cu, seqlens, end


def kvcache_append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, slot_mapping, validate=True):
    """Quantize new K / V rows into the 8-bit cache, in place.

    Arguments:
        k, v: (tokens, nheads_k, headdim), fp16, bf16 or fp32.
        k_cache, v_cache, k_scale, v_scale: the cache (see the module's
            documentation), written in place; no two elements may share
            memory.
        slot_mapping: (tokens,) int64, each row's slot, page * page_size + index
            in the page, as ``paged_kvcache_slots`` gives it; a row with -1
            is skipped.
        validate: check that slots lie in the cache and that no two runs share a
            block.  With False, a slot outside the cache is skipped, and blocks
            that two runs share get values of either.

    Consecutive rows with consecutive slots of one block form a run, and a block
    must be in one run only: a sequence's new tokens in order, one after the
    other.  A block holds the slots below its run.  A run that begins a block
    sets its scale, the least that holds the run's finite numbers; another
    one raises the scale where its numbers need that, and the rows that the
    block holds are then rounded to the new scale.  Numbers are rounded to
    nearest even; one that is not finite is stored as NaN.
    """
    if k.ndim != 3 or v.ndim != 3 or k.shape != v.shape:
        raise ValueError("k and v must have shape (tokens, nheads_k, headdim)")
    if k.dtype not in (torch.float16, torch.bfloat16, torch.float32) or v.dtype != k.dtype:
        raise ValueError("k and v must both be FP16, BF16 or FP32 tensors")
    block = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if k.shape[1:] != k_cache.shape[2:]:
        raise ValueError("new k/v tensors are incompatible with the cache")
    dev = k_cache.device
    if k.device != dev or v.device != dev:
        raise ValueError("k, v and the caches must be on the same CUDA device")
    if slot_mapping.shape != k.shape[:1] or slot_mapping.dtype != torch.int64 or slot_mapping.device != dev:
        raise ValueError("slot_mapping must hold one int64 slot per row on the same CUDA device")
    _check_no_grad("kvcache_append_8bit", k, v)
    _check_capture(validate)
    _check_targets(k_cache, v_cache, k_scale, v_scale)
    with _on(dev):
        slot_mapping = slot_mapping.contiguous()
        if validate and k.shape[0]:
            chk = Deferred()
            chk.check_range(slot_mapping, -1, k_cache.shape[0] * k_cache.shape[1] - 1,
                            ValueError("slot_mapping contains a slot outside the cache"))
            # The blocks of the runs, skipped rows apart, must all differ.
            of = slot_mapping // block
            begins = slot_mapping >= 0
            begins[1:] &= (slot_mapping[1:] != slot_mapping[:-1] + 1) | (of[1:] != of[:-1])
            runs = torch.where(begins, of, -1 - torch.arange(of.shape[0], device=dev)).sort().values
            chk.check((runs[1:] == runs[:-1]).any(),
                      ValueError("slot_mapping has two runs of rows in one scale block"))
            chk.flush()
        _native.kvcache8_append(_kernel_ready(k), _kernel_ready(v), k_cache, v_cache, k_scale, v_scale,
                                slot_mapping)


def flash_attn_with_kvcache_8bit(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens=None, block_table=None,
                                 cu_seqlens_q=None, max_seqlen_q=None, max_seqlen_k=None, softmax_scale=None,
                                 causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None,
                                 validate=True):
    """Attention against the 8-bit KV cache (``flash_attn_with_kvcache``'s form).

    Arguments:
        q: (batch, seqlen_q, nheads, headdim), or packed (total_q, nheads,
            headdim) with cu_seqlens_q; fp16 or bf16.
        k_cache, v_cache, k_scale, v_scale: the cache (see the module's
            documentation).
        cache_seqlens: (batch,) visible keys per sequence, the new tokens' own
            among them (None: all slots).
        block_table: (batch, max_num_pages) int32 pages of each sequence (None:
            page b is sequence b's cache).
        cu_seqlens_q: (batch + 1,) int32, sequence b's queries are rows
            cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 of q.
        max_seqlen_q: int, the most queries of a sequence (packed only).
        max_seqlen_k: int, a bound on cache_seqlens that the work is split by
            (None: the slots that block_table or a page has).
        softmax_scale, causal, window_size, alibi_slopes: as in
            ``flash_attn_with_kvcache``: with ``causal``, query i of n sits at
            position i + L - n.  softcap: as in ``flash_attn_func``.
        validate: check lengths, pages and offsets.  With False, lengths are
            clamped to max_seqlen_k, a page outside the cache reads as zeros, and
            a sequence whose offsets leave q or that has more than max_seqlen_q
            queries gets none or the first of them.
    Return:
        like q.  Rows without a visible key are 0, and so are rows of packed q
        behind the last sequence.

    A cached value counts as q's type holds it: exact in bf16; with fp16 queries
    values must be below 65504, as in an fp16 cache.
    """
    packed = cu_seqlens_q is not None
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q must be an FP16 or BF16 tensor")
    if q.ndim != (3 if packed else 4):
        raise ValueError("q must have shape (batch, seqlen_q, nheads, headdim), or (total_q, nheads, headdim) "
                         "with cu_seqlens_q")
    _check_cache(k_cache, v_cache, k_scale, v_scale)
    pages, page, heads_k, dim = k_cache.shape
    dev = q.device
    if dev != k_cache.device:
        raise ValueError("q and KV caches must be on the same CUDA device")
    if q.shape[-1] != dim:
        raise ValueError("q and KV cache dimensions are incompatible")
    heads = q.shape[-2]
    if heads_k == 0 or heads % heads_k != 0:
        raise ValueError("The number of query heads must be divisible by KV heads")
    if softcap < 0.0:
        raise ValueError("softcap must be non-negative")
    if packed:
        _lengths("cu_seqlens_q", cu_seqlens_q, None, dev)
        if cu_seqlens_q.shape[0] < 1:
            raise ValueError("cu_seqlens_q must contain a batch boundary")
        if max_seqlen_q is None:
            raise ValueError("max_seqlen_q must be given with cu_seqlens_q")
        batch, max_q = cu_seqlens_q.shape[0] - 1, int(max_seqlen_q)
        if max_q < 0:
            raise ValueError("max sequence lengths must be non-negative")
        max_q = min(max_q, q.shape[0])
    else:
        if max_seqlen_q is not None:
            raise ValueError("max_seqlen_q is for packed queries (cu_seqlens_q)")
        batch, max_q = q.shape[:2]
    if block_table is not None:
        if block_table.ndim != 2 or block_table.shape[0] != batch:
            raise ValueError("block_table must have shape (batch, max_num_pages)")
        if block_table.dtype not in _INTS or block_table.device != dev:
            raise ValueError("block_table must contain integer page indices on the same CUDA device")
        capacity = block_table.shape[1] * page
    else:
        if pages < batch:
            raise ValueError("a cache without block_table must have a page per sequence")
        capacity = page
    if cache_seqlens is not None:
        _lengths("cache_seqlens", cache_seqlens, batch, dev)
    max_k = capacity
    if max_seqlen_k is not None:
        if max_seqlen_k < 0:
            raise ValueError("max sequence lengths must be non-negative")
        max_k = min(int(max_seqlen_k), capacity)
    _check_no_grad("flash_attn_with_kvcache_8bit", q)
    _check_capture(validate)
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    with _on(dev):
        alibi = _normalize_alibi(alibi_slopes, batch, heads, dev)
        # (packed: rows behind the last sequence are 0)
        out = torch.zeros(q.shape, dtype=q.dtype, device=dev) if packed else torch.empty(
            q.shape, dtype=q.dtype, device=dev)

        def launch():
            if batch == 0 or q.numel() == 0:
                return
            table = block_table
            if table is not None and (table.dtype != torch.int32 or table.shape[1] and table.stride(1) != 1):
                table = table.to(torch.int32).contiguous()
            _native.fwd_kvcache8(
                _kernel_ready(q), out, k_cache, v_cache, k_scale, v_scale,
                None if cache_seqlens is None else _int32(cache_seqlens), table,
                _int32(cu_seqlens_q) if packed else None, batch, max_q, max_k, scale, causal,
                int(window_size[0]), int(window_size[1]), float(softcap), alibi)

        if not validate:
            launch()
            return out
        # The kernels stay within the tensors whatever the arrays hold, so the
        # launch goes out before the host waits for the checks.
        chk = Deferred()
        if block_table is not None:
            chk.check_range(block_table, 0, pages - 1,
                            ValueError("block_table contains an invalid physical page index"))
        if cache_seqlens is not None:
            chk.check_range(cache_seqlens, 0, max_k,
                            ValueError("cache_seqlens must contain valid lengths for every batch item"))
        if packed:
            chk.check_range(cu_seqlens_q[:1], 0, 0, ValueError("cu_seqlens_q must start at zero"))
            chk.check_range(cu_seqlens_q, 0, None,
                            ValueError("cu_seqlens_q must be monotonically non-decreasing"), diff=True)
            chk.check_range(cu_seqlens_q[-1:], None, q.shape[0],
                            ValueError("cu_seqlens_q exceeds the packed queries"))
            chk.check_range(cu_seqlens_q, None, max_q,
                            ValueError("max_seqlen_q must cover every packed sequence"), diff=True)
        chk.flush(launch)
    return out


__all__ = ["paged_kvcache_slots", "kvcache_append_8bit", "flash_attn_with_kvcache_8bit"]
