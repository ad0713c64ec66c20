"""The paged KV cache of the attention pass (CUDA, sm_100a): block tables and
slot maps from request lengths, the cache write, and attention over the blocks.

A step of a batch is three calls:

    m = extend_block_tables(block_table, cached, fresh, free_blocks, block_size, num_tokens)
    store_kv(k, v, k_cache, v_cache, m["slot_mapping"])
    out = paged_attention(q, k_cache, v_cache, block_table, m["cu_seqlens_q"], m["seq_lens"], max_seqlen_q)

They take the place of what the reference's attention backend does around its
library attention calls (vllm_gr/v1/attention/backends/beam_attn.py:629-755):
the cache write, the paged attention of plain requests, and, for the
beam-consecutive tokens of mega requests, prefix pass, suffix gather, suffix
pass and merge in one call (`beam_tail` / `beam_steps`).

Tensors stay on the GPU; calls run on the current stream of the tensors' device,
do not synchronise and can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_I32, _I64 = torch.int32, torch.int64


# the current stream's handle by device index, without a Stream object around it
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _plain_empty(size, stride, dtype):
    return torch.empty_strided(size, stride, dtype=dtype, device="cuda")


def _pick_empty():
    """torch.empty_strided on the current device without the argument parser (0.75 us instead
    of 1.3 to 2.3 us a tensor, a quarter of a small call), where this torch has it.  It is not
    a public entry, so it is taken only if it answers as expected."""
    try:
        fast = torch._C._dynamo.guards._empty_strided_cuda
        t = fast((2, 3), (3, 1), _I32)
        if t.is_cuda and t.device.index == torch.cuda.current_device() and t.dtype == _I32 and \
                tuple(t.shape) == (2, 3) and t.stride() == (3, 1):
            return fast
    except (AttributeError, TypeError, RuntimeError):
        pass
    return _plain_empty


def _empty(size, stride, dtype):
    """The first allocation, which replaces this function by the one picked."""
    global _empty
    _empty = _pick_empty()
    return _empty(size, stride, dtype)


def _on(index, fn, *args):
    """fn(*args) with device `index` current."""
    if index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _check(rc, name):
    if rc != _lib.GR_OK:
        raise RuntimeError(f"{name} failed: {_lib.STATUS_NAMES.get(rc, rc)}")


def _check_ints(name, t, device, dtype, shape=None):
    """An index tensor as the library reads it."""
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_table(block_table, device, num_seqs):
    if block_table.dtype != _I32 or block_table.device != device or block_table.dim() != 2:
        raise ValueError(f"block_table must be a 2-D int32 tensor on {device}")
    if block_table.shape[0] != num_seqs:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {num_seqs} requests")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table rows must have unit stride")
    if num_seqs > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table rows must not overlap")


def _check_caches(k_cache, v_cache):
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache / v_cache must be [num_blocks, block_size, num_kv_heads, head_dim]")
    if k_cache.dtype != v_cache.dtype or k_cache.shape != v_cache.shape or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must have the same dtype, shape and device")


def _check_sizes(*sizes):
    """The library's descriptors hold these in 32 bits."""
    if max(sizes) > 0x7FFFFFFF:
        raise ValueError(f"sizes must be below 2^31, not {max(sizes)}")


def _err(err, device):
    if err is None:
        return None
    if err.dtype != _I32 or err.device != device:
        raise ValueError(f"err must be an int32 tensor on {device}")
    return err.data_ptr()


class _Descs:
    """Descriptors of calls by everything but their tensors' addresses (shapes, strides,
    types, devices, options): a call like an earlier one skips the checks and the struct,
    which take longer on the host than the smallest steps on the device."""

    def __init__(self):
        self.known = {}

    def get(self, key, make, *args):
        d = self.known.get(key)
        if d is None:
            d = make(*args)
            if len(self.known) >= 1024:
                self.known.clear()
            self.known[key] = d
        return d


_table_descs, _store_descs, _attn_descs = _Descs(), _Descs(), _Descs()


def _table_desc(block_table, cached_lens, new_lens, free_blocks, block_size, num_tokens):
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor")
    device, n = block_table.device, num_tokens
    if cached_lens.dim() != 1:
        raise ValueError("cached_lens must be 1-D")
    R = cached_lens.shape[0]
    if block_size < 1 or n < 0 or n > 0x7FFFFFFF or free_blocks.dim() != 1:
        raise ValueError("block_size must be positive, num_tokens between 0 and 2^31 - 1, free_blocks 1-D")
    _check_table(block_table, device, R)
    _check_ints("cached_lens", cached_lens, device, _I32, (R,))
    _check_ints("new_lens", new_lens, device, _I32, (R,))
    _check_ints("free_blocks", free_blocks, device, _I32)
    _check_sizes(R, free_blocks.numel(), block_size, block_table.shape[1])
    d = _lib.BlockTableDesc(R, n, free_blocks.numel(), block_size, block_table.shape[1], 0, block_table.stride(0))
    return d, device.index


def extend_block_tables(block_table, cached_lens, new_lens, free_blocks, block_size: int, num_tokens: int, *, err=None):
    """Grows the requests' block tables for a step's new tokens and maps the tokens to cache slots.

    block_table: int32 [R, max_blocks], rows of unit stride, updated in place: request r,
    with cached_lens[r] tokens in the cache, gets ceil((cached + new) / block_size) -
    ceil(cached / block_size) blocks from the front of free_blocks (int32), the requests
    in order; other entries stay as they are.  cached_lens, new_lens: int32 [R].
    num_tokens: the step's token count, at least the sum of new_lens; entries behind that
    sum (a padded batch) get slot -1 and position 0.

    Returns a dict: cu_seqlens_q int32 [R + 1], seq_lens int32 [R] (cached + new),
    slot_mapping int64 [num_tokens], positions int64 [num_tokens], blocks_used int32 [1]
    (the blocks the step needs: what the caller removes from its free list).  A block that
    the free list or a row has no room for gives slot -1 and GR_DEVERR_NO_BLOCK in `err`
    (optional int32 device tensor), bad lengths GR_DEVERR_BAD_RECORD."""
    block_size, num_tokens = int(block_size), int(num_tokens)
    key = (block_table.shape, block_table.stride(), block_table.device, block_table.dtype, cached_lens.shape,
           cached_lens.stride(), cached_lens.dtype, cached_lens.device, new_lens.shape, new_lens.stride(), new_lens.dtype,
           new_lens.device, free_blocks.shape, free_blocks.stride(), free_blocks.dtype, free_blocks.device, block_size,
           num_tokens)
    d, index = _table_descs.get(key, _table_desc, block_table, cached_lens, new_lens, free_blocks, block_size, num_tokens)
    return _on(index, _extend, d, index, block_table, cached_lens, new_lens, free_blocks,
               _err(err, block_table.device))


def _extend(d, index, block_table, cached_lens, new_lens, free_blocks, err):
    R, n = d.num_seqs, d.num_tokens
    cu, lens, used = _empty((R + 1,), (1,), _I32), _empty((R,), (1,), _I32), _empty((1,), (1,), _I32)
    slots, positions = _empty((n,), (1,), _I64), _empty((n,), (1,), _I64)
    _check(_lib.load().gr_extend_block_tables(
        d, block_table.data_ptr(), cached_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(), cu.data_ptr(),
        lens.data_ptr(), slots.data_ptr(), positions.data_ptr(), used.data_ptr(), err, _stream(index)),
        "gr_extend_block_tables")
    return {"cu_seqlens_q": cu, "seq_lens": lens, "slot_mapping": slots, "positions": positions, "blocks_used": used}


def _store_desc(k, v, k_cache, v_cache, slot_mapping):
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be a CUDA tensor")
    device = k_cache.device
    _check_caches(k_cache, v_cache)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != k_cache.shape[2:]:
        raise ValueError("k and v must be [num_tokens, num_kv_heads, head_dim] with the cache's heads and head_dim")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype or k.device != device or v.device != device:
        raise ValueError("k and v must have the cache's dtype and device")
    if k_cache.element_size() not in (1, 2, 4):
        raise ValueError(f"unsupported KV element size {k_cache.element_size()}")
    T = k.shape[0]
    _check_ints("slot_mapping", slot_mapping, device, _I64, (T,))
    if k.numel() and not k_cache.numel():
        raise ValueError("the cache has no blocks")
    nb, bs, heads, dim = k_cache.shape
    _check_sizes(bs, heads, dim)
    d = _lib.KvStoreDesc(T, nb, bs, heads, dim, k_cache.element_size(), *k.stride(), *v.stride(), *k_cache.stride(),
                         *v_cache.stride())
    return d, device.index, k.numel() > 0


def store_kv(k, v, k_cache, v_cache, slot_mapping, *, err=None) -> None:
    """Writes the rows k[t], v[t] ([T, num_kv_heads, head_dim]) into the cache slots
    slot_mapping[t] (int64 [T], or int32, which is widened; slot = block * block_size +
    offset).  Slots < 0 are skipped; slots behind the cache are skipped and set
    GR_DEVERR_BAD_SLOT in `err`.  The slots of one call must differ, and k and v must not lie in
    the caches.  Any strides (rows of whole 16-byte vectors in the row and in the cache are
    copied as such, others by the element, some four times slower); 1-, 2- and 4-byte elements; rows
    are copied as they are, so k and the cache have one dtype.  The inverse of
    extract_suffix_kv."""
    if slot_mapping.dtype == _I32:
        slot_mapping = slot_mapping.to(_I64)
    key = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, k_cache.shape, k_cache.stride(),
           k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device,
           slot_mapping.shape, slot_mapping.stride(), slot_mapping.dtype, slot_mapping.device)
    d, index, any_rows = _store_descs.get(key, _store_desc, k, v, k_cache, v_cache, slot_mapping)
    err = _err(err, k_cache.device)
    if any_rows:
        _check(_on(index, _lib.load().gr_store_kv, d, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                   slot_mapping.data_ptr(), err, _stream(index)), "gr_store_kv")


def _attn_desc(q, k_cache, v_cache, block_table, cu_seqlens_q, seq_lens, max_seqlen_q, scale, causal, beam_tail,
               beam_steps, out):
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor")
    device = q.device
    _check_caches(k_cache, v_cache)
    if q.dtype not in _DTYPES or k_cache.dtype != q.dtype:
        raise ValueError(f"q and the caches must both be bf16 or f16, not {q.dtype} and {k_cache.dtype}")
    if q.dim() != 3 or q.shape[2] != k_cache.shape[3] or k_cache.device != device:
        raise ValueError("q must be [num_tokens, num_heads, head_dim] with the cache's head_dim and device")
    T, H, D = q.shape
    nb, bs, HK, _ = k_cache.shape
    if H == 0 or HK == 0 or D == 0 or bs == 0 or H % HK:
        raise ValueError(f"num_heads={H} must be a multiple of num_kv_heads={HK}, sizes positive")
    if D > 1 and (q.stride(2) != 1 or k_cache.stride(3) != 1 or v_cache.stride(3) != 1):
        raise ValueError("q and the caches need unit stride in head_dim")
    if seq_lens.dim() != 1:
        raise ValueError("seq_lens must be 1-D")
    R = seq_lens.shape[0]
    _check_ints("seq_lens", seq_lens, device, _I32)
    _check_ints("cu_seqlens_q", cu_seqlens_q, device, _I32, (R + 1,))
    _check_table(block_table, device, R)
    if (beam_tail is None) != (beam_steps is None):
        raise ValueError("beam_tail and beam_steps go together")
    if beam_tail is not None:
        if not causal:
            raise ValueError("beams need causal attention")
        _check_ints("beam_tail", beam_tail, device, _I32, (R,))
        _check_ints("beam_steps", beam_steps, device, _I32, (R,))
    scale = D ** -0.5 if scale is None else scale
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != device or
                            (D > 1 and out.stride(2) != 1)):
        raise ValueError("out must have q's shape, dtype and device and unit stride in head_dim")
    _check_sizes(R, T, H, D, bs, block_table.shape[1])
    out_tok, out_head = (H * D, D) if out is None else out.stride()[:2]
    d = _lib.PagedAttnDesc(R, T, H, HK, D, bs, block_table.shape[1], _DTYPES[q.dtype], int(causal),
                           max_seqlen_q, scale, 0, nb, block_table.stride(0), q.stride(0), q.stride(1),
                           *k_cache.stride()[:3], *v_cache.stride()[:3], out_tok, out_head)
    size = ctypes.c_size_t(0)
    _lib.check(_lib.load().gr_paged_attention_workspace_size(d, size), "gr_paged_attention_workspace_size")
    return d, size.value, device.index, bool(T and R), ((T, H, D), (H * D, D, 1)), ((T, H), (H, 1))


def _kind(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def paged_attention(q, k_cache, v_cache, block_table, cu_seqlens_q, seq_lens, max_seqlen_q: int, *, scale=None,
                    causal: bool = True, beam_tail=None, beam_steps=None, out=None, return_lse: bool = False, err=None):
    """Attention of a step's query tokens over the requests' cache blocks.

    q: [T, num_heads, head_dim], bf16 or f16; caches [num_blocks, block_size, num_kv_heads,
    head_dim] of the same dtype; block_table int32 [R, max_blocks]; cu_seqlens_q int32 [R + 1]
    query offsets; seq_lens int32 [R] keys per request, the new tokens' own (already
    written by store_kv) included; max_seqlen_q: the longest query, a host number that only
    picks the kernel.  Query token i of request r sits at position seq_lens[r] - n_r + i and
    sees the keys up to there (causal) or all of them.  Whole prompts, chunks and single
    tokens mix freely.

    beam_tail, beam_steps (int32 [R], both or neither; causal only) mark beam-consecutive
    requests: where beam_steps[r] > 0, query tokens from beam_tail[r] on belong to beams of
    beam_steps[r] tokens each, and a beam's tokens see the shared prefix, the tail before the
    beams and their own beam only.

    Returns out ([T, num_heads, head_dim], q's dtype; pass `out` to write into a tensor of
    yours), with return_lse also the fp32 [T, num_heads] natural log-sum-exp of the scaled
    scores.  A token without keys gets 0 and -inf; rows of tokens that belong to no request
    are left as they were (unspecified in a new `out`).  `out` must not overlap the inputs;
    gradients are not computed.  scale defaults to head_dim ** -0.5.
    V has to be finite at positions below seq_lens; what blocks hold behind does not matter.

    Scores, sums and accumulators are fp32.  The softmax's weights are rounded once to q's
    dtype before they multiply V (each off by at most half a step: 2^-8 in bf16, 2^-11 in f16,
    relative; their sum takes them unrounded), and out is rounded once.

    head_dim: a multiple of 8 up to 256; block_size: a multiple of 8; num_heads /
    num_kv_heads up to 128; unit stride in head_dim, other strides multiples of 8 elements,
    16-byte aligned tensors.  Block ids outside the cache read as zero rows and set
    GR_DEVERR_BAD_SLOT in `err` (optional int32 device tensor); lengths outside the table's
    row or the tokens are clamped and set GR_DEVERR_BAD_RECORD.  A wait inside the kernel that
    runs out (2 to 32 seconds, by what it waits for) sets GR_DEVERR_TIMEOUT and leaves the
    outputs incomplete, of which nothing tells without `err`; a captured call that has set it
    must be captured anew."""
    # a longer bound than any query tile picks the same kernel
    max_seqlen_q, causal = min(int(max_seqlen_q), 129), bool(causal)
    scale = None if scale is None else float(scale)
    key = (q.shape, q.stride(), q.dtype, q.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
           v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device, block_table.shape, block_table.stride(),
           block_table.dtype, block_table.device, cu_seqlens_q.shape, cu_seqlens_q.stride(), cu_seqlens_q.dtype,
           cu_seqlens_q.device, seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, max_seqlen_q, scale,
           causal, _kind(beam_tail), _kind(beam_steps), _kind(out))
    desc = _attn_descs.get(key, _attn_desc, q, k_cache, v_cache, block_table, cu_seqlens_q, seq_lens, max_seqlen_q, scale,
                           causal, beam_tail, beam_steps, out)
    return _on(desc[2], _attend, desc, q, k_cache, v_cache, block_table, cu_seqlens_q, seq_lens, beam_tail, beam_steps, out,
               return_lse, _err(err, q.device))


def _attend(desc, q, k_cache, v_cache, block_table, cu_seqlens_q, seq_lens, beam_tail, beam_steps, out, return_lse, err):
    d, size, index, any_rows, out_as, lse_as = desc
    if out is None:
        out = _empty(*out_as, q.dtype)
    lse = _empty(*lse_as, torch.float32) if return_lse else None
    if any_rows:
        # from the caching allocator per call: stream ordered, and a captured graph keeps its own
        ws = _empty((size,), (1,), torch.uint8)
        io = _lib.PagedAttnIO(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
                              cu_seqlens_q.data_ptr(), seq_lens.data_ptr(),
                              None if beam_tail is None else beam_tail.data_ptr(),
                              None if beam_steps is None else beam_steps.data_ptr(), out.data_ptr(),
                              None if lse is None else lse.data_ptr(), err)
        _check(_lib.load().gr_paged_attention(d, io, ws.data_ptr(), size, _stream(index)), "gr_paged_attention")
    return (out, lse) if return_lse else out
