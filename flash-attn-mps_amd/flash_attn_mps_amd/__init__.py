"""FlashAttention inference for PyTorch-ROCm on AMD Instinct MI355X (gfx950).

A drop-in for the public API of flash_attn_mps (flash_attn_mps/__init__.py:3-29):
the FlashAttention-2 functions, ``store_kvcache`` and ``merge_attn_states``,
with the same names, signatures and tensor contracts, computed by hand-written
gfx950 HIP kernels in ``libfa_gfx950.so``.  The vLLM contract lives in
``flash_attn_mps_amd.vllm``.
"""

from .interface import (
    flash_attn_func,
    flash_attn_kvpacked_func,
    flash_attn_qkvpacked_func,
    flash_attn_varlen_func,
    flash_attn_varlen_kvpacked_func,
    flash_attn_varlen_qkvpacked_func,
    flash_attn_with_kvcache,
)
from .vllm import merge_attn_states

__version__ = "0.2.0"


def store_kvcache(key, value, k_cache, v_cache, slot_mapping, *, k_scale=None, v_scale=None):
    """Write key/value [T, Hkv, D] rows to cache slots (slot // P, slot % P); slots < 0 are skipped."""
    from ._cache import store_kvcache as _store
    _store(key, value, k_cache, v_cache, slot_mapping, k_scale=k_scale, v_scale=v_scale)


def rotary_embedding(q, k, rotary_cos, rotary_sin, positions, *, pair_axes=None, rotary_interleaved=True):
    """Rotary embedding of packed rows q [T, Hq, D] and k [T, Hk, D] (or None): fresh (q, k).

    ``positions`` is [T], or [axes, T] for up to 4 axes (time, height, width),
    int32 or int64; with several, ``pair_axes`` gives the axis of each rotated
    pair, for instance ``[0] * 16 + [1] * 24 + [2] * 24``.  Pair i turns by row
    ``positions[pair_axes[i], t]`` of ``rotary_cos`` / ``rotary_sin`` [positions,
    rotary_dim / 2]: dims (2i, 2i + 1) interleaved, else (i, i + rotary_dim / 2);
    dims past rotary_dim are copied.  A position outside the tables gives NaN.
    """
    from ._cache import rotary_embedding as _rotary
    return _rotary(q, k, rotary_cos, rotary_sin, positions, pair_axes=pair_axes, interleaved=rotary_interleaved)


def append_paged_kvcache(k, v, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, *, q=None, rotary_cos=None,
                         rotary_sin=None, positions=None, pair_axes=None, rotary_interleaved=True, k_scale=None,
                         v_scale=None):
    """Append packed rows k [T, Hkv, Dk] / v [T, Hkv, Dv] to a paged cache, in one launch
    with the rotary embedding of k on the way and of q; returns q rotated (None without q).

    The metadata is that of the attention call that follows: request b owns rows
    ``cu_seqlens_q[b]`` .. ``cu_seqlens_q[b + 1]``, the last of its ``seqused_k[b]``
    positions (lengths after the append), in the pages ``block_table[b]`` of caches
    [pages, page_size, Hkv, D].  Positions and pages outside the table or the
    cache are skipped.  Rows behind the last request are not written; their q
    is copied, or turned where ``positions`` are given.  Two requests must not
    write to one page.

    Rotary arguments as in ``rotary_embedding``; without ``positions`` each row turns
    by its cache position.  Keys round once, to the cache's type: the rows' type
    or E4M3, with ``k_scale`` / ``v_scale``

    * None, a value or one per head: E4M3(x / scale), as ``store_kvcache``;
    * float8_e8m0fnu [pages, page_size / block, Hkv]: one power of two per block of
      tokens and head, written by the append.  A block takes the smallest one >=
      2^-100 under which its largest finite new magnitude is at most 448; if it
      holds earlier rows of its request, the larger of that and its old one, and
      those rows are coded again.  ``vllm.flash_attn_varlen_func`` reads such a
      cache; let it start as zeros (NaN codes where no row looks cost time).
    """
    from ._cache import append_paged_kvcache as _append
    return _append(k, v, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, q=q, cos=rotary_cos, sin=rotary_sin,
                   positions=positions, pair_axes=pair_axes, interleaved=rotary_interleaved, k_scale=k_scale,
                   v_scale=v_scale)


__all__ = [
    "flash_attn_func", "flash_attn_kvpacked_func", "flash_attn_qkvpacked_func",
    "flash_attn_varlen_func", "flash_attn_varlen_kvpacked_func",
    "flash_attn_varlen_qkvpacked_func", "flash_attn_with_kvcache", "store_kvcache",
    "merge_attn_states", "rotary_embedding", "append_paged_kvcache",
]
