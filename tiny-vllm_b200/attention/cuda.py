"""Python entry points of the attention kernels and of the paged key-value cache that they read.

What the reference's attention layer gets from libraries (``nanovllm/layers/attention.py:10-89``): keys and values
of new tokens are stored into pages, whole prompts attend causally, and each new token attends over its sequence's
pages.  One backend, no CPU path: what the kernels cannot take raises ``RuntimeError``.  All of it is for
inference: nothing here has a gradient.

With ``G = heads / kv_heads`` and a sequence of ``n`` queries and ``m`` keys, the queries being the last ``n`` of its
``m`` positions, row ``i`` of head ``h`` is

    o[i, h] = sum_j p[i, h, j] v[j, h // G],    p = softmax_j(scale * q[i, h] . k[j, h // G])

over ``j <= i + m - n`` (``causal``) or all ``j < m``; zeros where that leaves no key, or only scores of -infinity.
Sums and softmax statistics are fp32; the softmax weights are rounded to the tensors' type for the second product, as
is the result.  What keys and values hold that a row does not see does not matter, NaN and infinities included.  Scores
``scale * q . k`` are fp32 and may be of any size up to 2^127.  Two things that no healthy model has make prompts slow,
a hundred times for the rows concerned: scores beyond 700,000, and values that are not finite up to 255 positions
behind a row that does not see them.

``float16`` or ``bfloat16``; ``dim`` a multiple of 8 up to 128; up to 128 query heads per key head; pages of a
multiple of 16 positions.  Heads, tokens and pages may stand apart (strides of a multiple of 8 elements).  Calls run on
the current stream of the tensors' device, can be captured, and follow the contents of lengths, tables and slots at
every replay.  A page number outside of the cache counts as a page of zeros and a slot outside of it is skipped;
both set the device status word, which ``_lib.check_device()`` turns into an error.
"""
from __future__ import annotations

import torch

from .. import _lib

_DTYPES = (torch.float16, torch.bfloat16)


def _native():
    return _lib._native or _lib.native()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: a dense last dimension, the others on 16-byte boundaries."""
    dense = (t.stride(-1) == 1 or t.shape[-1] == 1) and t.data_ptr() % 16 == 0
    if dense and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride())):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _require_cuda(*tensors: torch.Tensor | None) -> None:
    if not all(t.is_cuda for t in tensors if t is not None):
        raise RuntimeError(
            "b200q kernels need CUDA tensors on a B200; there is no CPU implementation of this path")


def _require_one_gpu(what: str, *tensors: torch.Tensor | None) -> None:
    if len({t.device for t in tensors if t is not None}) > 1:
        raise RuntimeError(f"{what} does not support the provided tensors (all of them must be on one GPU)")


def _check_ints(what: str, name: str, t: torch.Tensor, dim: int) -> None:
    if t.dtype != torch.int32 or t.dim() != dim:
        raise RuntimeError(f"{what}: {name} must be a {dim}-D int32 tensor")


def _check_cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype, kv_heads: int | None,
                 dim: int) -> None:
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise RuntimeError(f"{what} expects two [pages, page size, kv heads, dim] caches of {dtype}")
    if k_cache.shape[3] != dim or kv_heads not in (None, k_cache.shape[2]):
        raise RuntimeError(f"{what}: caches of {k_cache.shape[2]} heads of {k_cache.shape[3]} do not fit the tensors")
    if k_cache.numel() == 0:
        raise RuntimeError(f"{what}: the caches hold no page")
    for t in (k_cache, v_cache):    # a cache is not copied to suit the kernels
        if _aligned(t) is not t:
            raise RuntimeError(f"{what}: a cache's last dimension must be dense and the others on 16-byte boundaries")


def _check_queries(what: str, q: torch.Tensor, k: torch.Tensor) -> None:
    if q.dim() != 3 or q.dtype not in _DTYPES:
        raise RuntimeError(f"{what} expects float16/bfloat16 queries [tokens, heads, dim]")
    heads, dim, kv_heads = q.shape[1], q.shape[2], k.shape[-2]
    if kv_heads == 0 or heads == 0 or heads % kv_heads != 0:
        raise RuntimeError(f"{what}: {heads} query heads are not a multiple of {kv_heads} key heads")
    if dim == 0 or dim % 8 != 0 or dim > 128 or heads // kv_heads > 128:
        _lib.check(_lib.ERR_UNSUPPORTED_SHAPE, what, f"heads={heads}/{kv_heads} dim={dim}")


def _check_out(what: str, q: torch.Tensor, out: torch.Tensor | None) -> None:
    if out is None:
        return
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() \
            or out.data_ptr() % 16 != 0:
        raise RuntimeError(f"{what}: out must be a contiguous {list(q.shape)} {q.dtype} tensor on {q.device}")


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    def end(t: torch.Tensor) -> int:
        return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _finish(what: str, out, *tensors):
    if out is None:
        _require_one_gpu(what, *tensors)
        _lib.check(_lib.ERR_BAD_SHAPE, what, " ".join(str(list(t.shape)) for t in tensors if t is not None))
    return out


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, *,
                      scale: float | None = None, causal: bool = True, block_tables: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of sequences packed one after another: rows ``cu_seqlens_q[b]`` to ``cu_seqlens_q[b + 1]`` of ``q``
    are the queries of sequence ``b``.

    ``q``: ``[tokens, heads, dim]``.  Without ``block_tables``, ``k`` and ``v`` are ``[key tokens, kv heads, dim]``,
    packed by ``cu_seqlens_k``.  With ``block_tables`` (int32 ``[sequences, pages of the longest]``) they are a layer's
    caches ``[pages, page size, kv heads, dim]``, and position ``j`` of sequence ``b`` stands in page
    ``block_tables[b, j // page size]`` (a prompt whose beginning is cached, a chunk of a long one); of
    ``cu_seqlens_k`` only the differences count.  Both ``cu_seqlens`` are int32 ``[sequences + 1]`` on the GPU.
    ``max_seqlen_k`` bounds the keys of a sequence and only helps to divide the work: the result does not depend on it
    beyond rounding.  ``max_seqlen_q`` belongs to the call as engines make it and is not used.  ``scale`` is positive
    and defaults to ``dim ** -0.5``.

    Returns ``[tokens, heads, dim]`` (``out``, where that is given, contiguous; it may be the memory of ``q``).  Rows
    behind the last sequence are not written.
    """
    if scale is None:
        scale = max(q.shape[-1], 1) ** -0.5
    o = _native().attention(q, k, v, cu_seqlens_q, cu_seqlens_k, None, block_tables, max_seqlen_q, max_seqlen_k, scale,
                            causal, out)
    if o is not None:
        return o
    what = "prefill_attention"
    _require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, block_tables)
    if block_tables is None and (k.dim() != 3 or k.shape != v.shape or k.dtype != q.dtype or v.dtype != q.dtype
                                 or k.shape[-1] != q.shape[-1]):
        raise RuntimeError(f"{what} expects k and v [key tokens, kv heads, dim] of the queries' type and dim")
    if block_tables is not None:
        _check_cache(what, k, v, q.dtype, None, q.shape[-1])
        _check_ints(what, "block_tables", block_tables, 2)
    _check_queries(what, q, k)
    _check_ints(what, "cu_seqlens_q", cu_seqlens_q, 1)
    _check_ints(what, "cu_seqlens_k", cu_seqlens_k, 1)
    sequences = cu_seqlens_q.numel() - 1
    if sequences < 0 or cu_seqlens_k.numel() != sequences + 1:
        raise RuntimeError(f"{what}: cu_seqlens_q and cu_seqlens_k must have one entry per sequence and one more")
    if block_tables is not None and (block_tables.shape[0] != sequences or (sequences and block_tables.shape[1] == 0)):
        raise RuntimeError(f"{what}: block_tables must have a row of pages for each of the {sequences} sequences")
    if max_seqlen_q < 0 or max_seqlen_k < 0:
        raise RuntimeError(f"{what}: max_seqlen_q and max_seqlen_k must not be negative")
    _check_out(what, q, out)
    if q.numel() == 0 or sequences == 0:
        return torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    if block_tables is None:
        k, v = _aligned(k), _aligned(v)
    else:
        block_tables = block_tables.contiguous()
    q = _aligned(q)
    if out is not None and _share_memory(q, out):
        q = q.clone(memory_format=torch.contiguous_format)      # the kernel may read queries again behind their results
    o = _native().attention(q, k, v, cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous(), None, block_tables,
                            max_seqlen_q, max_seqlen_k, scale, causal, out)
    return _finish(what, o, q, k, v, cu_seqlens_q, cu_seqlens_k, block_tables)


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, context_lens: torch.Tensor,
                     block_tables: torch.Tensor, *, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages.

    ``q``: ``[sequences, heads, dim]``; caches ``[pages, page size, kv heads, dim]``; ``context_lens``: int32
    ``[sequences]``, the positions that each token sees, its own among them (0, as in the padding of a captured batch:
    zeros); ``block_tables``: int32 ``[sequences, pages of the longest]``, of which entries behind a sequence's
    last page are not read.  Lengths are cut to what a row of the tables holds.  ``scale`` is positive and defaults
    to ``dim ** -0.5``.  Returns ``[sequences, heads, dim]`` (``out``, where that is given, contiguous).

    A long context is divided over the GPU and joined in a fixed order: the same call gives the same bits.
    """
    if scale is None:
        scale = max(q.shape[-1], 1) ** -0.5
    o = _native().attention(q, k_cache, v_cache, None, None, context_lens, block_tables, 1, 0, scale, True, out)
    if o is not None:
        return o
    what = "decode_attention"
    _require_cuda(q, k_cache, v_cache, context_lens, block_tables)
    _check_cache(what, k_cache, v_cache, q.dtype, None, q.shape[-1])
    _check_queries(what, q, k_cache)
    _check_ints(what, "context_lens", context_lens, 1)
    _check_ints(what, "block_tables", block_tables, 2)
    sequences = q.shape[0]
    if context_lens.numel() != sequences or block_tables.shape[0] != sequences \
            or (sequences and block_tables.shape[1] == 0):
        raise RuntimeError(f"{what}: context_lens and block_tables must have an entry for each of the {sequences} queries")
    _check_out(what, q, out)
    if q.numel() == 0:
        return torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    q = _aligned(q)
    if out is not None and _share_memory(q, out) and not (q.data_ptr() == out.data_ptr() and q.is_contiguous()):
        q = q.clone(memory_format=torch.contiguous_format)
    o = _native().attention(q, k_cache, v_cache, None, None, context_lens.contiguous(),
                            block_tables.contiguous(), 1, 0, scale, True, out)
    return _finish(what, o, q, k_cache, v_cache, context_lens, block_tables)


def store_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slot_mapping: torch.Tensor) -> None:
    """Writes new tokens' keys and values into a layer's caches.

    ``k``, ``v``: ``[tokens, kv heads, dim]``; caches ``[pages, page size, kv heads, dim]``; ``slot_mapping``: int32
    ``[tokens]``, page times page size plus position.  A negative slot is skipped (padding).  Slots of a call are
    distinct: which of two tokens with one slot stays is not defined.
    """
    if _native().kv_store(k, v, k_cache, v_cache, slot_mapping) is not None:
        return
    what = "store_kv"
    _require_cuda(k, v, k_cache, v_cache, slot_mapping)
    if k.dim() != 3 or k.shape != v.shape or k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise RuntimeError(f"{what} expects float16/bfloat16 k and v [tokens, kv heads, dim]")
    _check_cache(what, k_cache, v_cache, k.dtype, k.shape[1], k.shape[2])
    _check_ints(what, "slot_mapping", slot_mapping, 1)
    if slot_mapping.numel() != k.shape[0]:
        raise RuntimeError(f"{what}: slot_mapping must have one entry per token")
    if k.shape[2] % 8 != 0:
        _lib.check(_lib.ERR_UNSUPPORTED_SHAPE, what, f"dim={k.shape[2]}")
    if k.numel() == 0:
        return
    done = _native().kv_store(_aligned(k), _aligned(v), k_cache, v_cache, slot_mapping.contiguous())
    _finish(what, done, k, v, k_cache, v_cache, slot_mapping)


def copy_pages(kv_cache: torch.Tensor, src: list[int], dst: list[int]) -> None:
    """Copies pages of a cache: page ``src[i]`` to page ``dst[i]``, in every layer, keys and values, in one launch
    per 480 pages.

    ``kv_cache``: ``[..., pages, page size, kv heads, dim]`` (the whole cache ``[2, layers, pages, ...]``, or one
    layer's part of it), any element type.  ``src`` and ``dst`` are host lists, as a block manager has them: a fork
    copies a sequence's last, partly filled page; compaction moves pages from the end of the cache into free ones, after
    which the manager rewrites its tables and takes the old pages as free.  A page may go to several places.  Each
    destination stands once and is no source of the same call; anything else raises ``ValueError`` and copies
    nothing.  A captured call keeps its pairs.
    """
    what = "copy_pages"
    if not isinstance(src, (list, tuple)) or not isinstance(dst, (list, tuple)) \
            or not all(isinstance(i, int) and not isinstance(i, bool) for i in (*src, *dst)):
        raise ValueError(f"{what} expects lists of page numbers on the host")
    if len(src) != len(dst):
        raise ValueError(f"{what}: {len(src)} sources and {len(dst)} destinations")
    if kv_cache.dim() < 4:
        raise RuntimeError(f"{what} expects a cache [..., pages, page size, kv heads, dim]")
    pages, targets = kv_cache.shape[-4], set(dst)
    if not all(0 <= i < pages for i in (*src, *dst)):
        raise ValueError(f"{what}: a page is not one of the cache's {pages}")
    if len(targets) != len(dst) or targets.intersection(src):
        raise ValueError(f"{what}: a destination stands twice or is a source as well")
    _require_cuda(kv_cache)
    if not src or kv_cache.numel() == 0:
        return
    if _native().copy_pages(kv_cache, src, dst) is None:
        raise RuntimeError(f"{what}: the cache's pages must be dense and its layers evenly spaced")
