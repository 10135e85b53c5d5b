"""KV-cache writes and rotary embedding on gfx950: host side of
fa_store_kvcache / fa_append_kvcache / fa_rotary (counterpart of
flash_attn_mps/_cache.py:55-155).

* store_kvcache scatters token rows to physical slots (page = slot // P,
  row = slot % P); negative or out-of-range slots are skipped by the kernel.
* append_kvcache writes new rows at ``lengths[b] + j`` of a dense cache row
  or through a page table; the lengths themselves are not touched.
* rotary_append is a generation step's rotary embedding and append in one
  launch.
* rotary_embedding turns packed rows by positions on one to four axes, and
  append_paged_kvcache writes packed rows of requests to a paged cache with that
  rotation on the way; its E4M3 caches may hold a power of two per block of
  tokens and head (E8M0) in place of a scale per head.
* An FP8 (E4M3FN) cache stores E4M3(x / scale) with scale a scalar or one
  value per KV head; 16-bit and fp32 caches of the input's dtype get the
  input's bits.
"""
import ctypes
import operator
from functools import lru_cache

import torch

from . import _lib
from ._problem import _check, on_gpu, reject_training

_INPUT_TYPES = (torch.float16, torch.bfloat16, torch.float32)
BLOCK_SCALE = torch.float8_e8m0fnu


def is_block_scale(scale):
    """Whether `scale` is the scales of a block-scaled cache: E8M0 [pages, blocks, heads], a power of two per block
    and head.  (E8M0 tensors of fewer dims are values like any others: one, or one per head.)"""
    return torch.is_tensor(scale) and scale.dtype == BLOCK_SCALE and scale.ndim > 2


def block_of(cache, scale, name):
    """Tokens per scale of a paged E4M3 cache [pages, P, H, D] whose scales [pages, P / block, H] are `scale`."""
    if cache.ndim != 4 or cache.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{name} goes with a paged float8_e4m3fn cache")
    pages, size, heads = cache.shape[:3]
    if scale.ndim != 3 or scale.shape[0] != pages or scale.shape[2] != heads or not scale.shape[1] \
            or size % scale.shape[1]:
        raise ValueError(f"{name} {tuple(scale.shape)} must be [{pages}, blocks dividing {size}, {heads}]")
    if scale.device != cache.device:
        raise ValueError(f"{name} is on {scale.device}; expected the cache's device {cache.device}")
    return size // scale.shape[1]


def _require_gpu(**tensors):
    for name, t in tensors.items():
        if t is not None and not on_gpu(t):
            raise ValueError(f"{name} is on {t.device}; cache operations run on a ROCm GPU")


_ONES = {}


def _one(device):
    """A resident fp32 1.0 per device: the FP8 scale when the caller gives none.
    Copied from the host, so that no other stream can find it unwritten; one made
    while a graph is captured is written by its replays, and stays that call's own."""
    one = _ONES.get(device)
    if one is None:
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            return torch.ones(1, dtype=torch.float32, device=device)
        one = torch.ones(1, dtype=torch.float32, device="cpu").to(device)
        if type(one) is torch.Tensor:   # (not a tracer's stand-in)
            _ONES[device] = one
    return one


def _per_head_scale(scale, heads, device):
    """(fp32 tensor, stride): stride 0 shares one scale, 1 reads one per head."""
    if is_block_scale(scale):
        raise TypeError("scales per block (float8_e8m0fnu) go with append_paged_kvcache")
    t = _one(device) if scale is None else torch.as_tensor(scale, dtype=torch.float32, device=device)
    if t.numel() == 1:
        return t.reshape(1), 0
    if t.numel() == heads:
        return t.reshape(heads).contiguous(), 1
    raise ValueError(f"an FP8 scale is one value or one per KV head ({heads}); got {t.numel()} values")


def _per_request(value, count, device, name):
    """An int32 [count] device tensor from an int, a 1-element or a [count] tensor."""
    t = torch.as_tensor(0 if value is None else value, dtype=torch.int32, device=device)
    if t.numel() == 1:
        t = t.reshape(1).expand(count)
    if t.numel() != count:
        raise ValueError(f"{name}: expected 1 or {count} values, got {t.numel()}")
    return t.contiguous()


def _write_desc(x, cache, scale, x_strides, keep):
    """fa_store_desc for writing `x` rows into `cache` (checks the dtype pair)."""
    if x.dtype not in _INPUT_TYPES:
        raise TypeError(f"cache inputs are float16, bfloat16 or float32; got {x.dtype}")
    fp8 = cache.dtype == torch.float8_e4m3fn
    if not fp8 and cache.dtype != x.dtype:
        raise TypeError(f"a {cache.dtype} cache cannot take {x.dtype} rows (use the same dtype or float8_e4m3fn)")
    d = _lib.StoreDesc()
    d.x, d.cache = x.data_ptr(), cache.data_ptr()
    d.x_dtype, d.cache_dtype = _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[cache.dtype]
    d.heads, d.dim = x.shape[-2], x.shape[-1]
    d.x_stride[:] = x_strides
    d.cache_stride[:] = cache.stride()
    if fp8:
        s, stride = _per_head_scale(scale, x.shape[-2], x.device)
        keep.append(s)
        d.scale, d.scale_stride = s.data_ptr(), stride
    return d


def _check_cache_shape(x, cache, row_dims):
    """cache [pages, page_size, heads, dim] matching the (heads, dim) of x."""
    if cache.ndim != 4 or cache.shape[2:] != x.shape[row_dims:]:
        raise ValueError(f"cache {tuple(cache.shape)} must be [pages, page_size, {x.shape[-2]}, {x.shape[-1]}]")


def store_kvcache(k, v, k_cache, v_cache, slot_mapping, *, k_scale=None, v_scale=None):
    """Write k/v [T, Hkv, D] to the cache slots slot_mapping [T] (int32/int64)."""
    _require_gpu(k=k, v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=slot_mapping)
    if k.ndim != 3 or v.ndim != 3 or k.shape[:2] != v.shape[:2]:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, heads, dim] "
                         "with the same tokens and heads")
    if (slot_mapping.ndim != 1 or slot_mapping.numel() != k.shape[0]
            or slot_mapping.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"slot_mapping must be int32/int64 with one entry per token ({k.shape[0]})")
    _check_cache_shape(k, k_cache, 1)
    _check_cache_shape(v, v_cache, 1)
    if k_cache.shape[:2] != v_cache.shape[:2]:
        raise ValueError("the K and V caches must have the same pages and page size")
    writes = [(x, c, s) for x, c, s in ((k, k_cache, k_scale), (v, v_cache, v_scale)) if x.numel()]
    if not writes:
        return
    keep = []
    args = _lib.StoreArgs()
    for i, (x, c, s) in enumerate(writes):
        args.kv[i] = _write_desc(x, c, s, x.stride(), keep)
    args.slots = slot_mapping.data_ptr()
    args.slot_dtype = _lib.I64 if slot_mapping.dtype == torch.int64 else _lib.I32
    args.slot_stride = slot_mapping.stride(0)
    args.tokens, args.page_size, args.num_pages = k.shape[0], k_cache.shape[1], k_cache.shape[0]
    _lib.call("fa_store_kvcache", args, k.device)


def append_kvcache(k, v, k_cache, v_cache, cache_seqlens, *, cache_batch_idx=None,
                   cache_leftpad=None, block_table=None, k_scale=None, v_scale=None):
    """Write k/v [B, Snew, Hkv, D] at position cache_seqlens[b] + j of request b.

    Dense caches [rows, capacity, Hkv, D] take row ``cache_batch_idx[b]``
    (default b); with ``block_table`` [rows, pages] the position goes through
    the table.  cache_leftpad does not move the write: FA2 lengths already
    count the padding (flash_attn_mps/_cache.py:99-127).
    """
    keep = []
    args = _append_args(k, v, k_cache, v_cache, cache_seqlens, cache_batch_idx, cache_leftpad, block_table, k_scale,
                        v_scale, keep)
    if args is not None:
        _lib.call("fa_append_kvcache", args, k.device)


def _append_args(k, v, k_cache, v_cache, cache_seqlens, cache_batch_idx, cache_leftpad, block_table, k_scale, v_scale,
                 keep):
    """The checked fa_append_args of an append (None: nothing to write)."""
    _require_gpu(k=k, v=v, k_cache=k_cache, v_cache=v_cache, block_table=block_table)
    if k.ndim != 4 or v.ndim != 4 or k.shape[:3] != v.shape[:3]:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [batch, new_tokens, heads, dim] "
                         "with the same batch, tokens and heads")
    batch = k.shape[0]
    lengths = _per_request(cache_seqlens, batch, k.device, "cache_seqlens")
    rows = None
    if block_table is None and cache_batch_idx is not None:
        rows = _per_request(cache_batch_idx, batch, k.device, "cache_batch_idx")
    if cache_leftpad is not None:
        _per_request(cache_leftpad, batch, k.device, "cache_leftpad")
    if block_table is not None and block_table.ndim != 2:
        raise ValueError(f"block_table must be [rows, pages]; got {tuple(block_table.shape)}")
    table = None if block_table is None else block_table.to(torch.int32).contiguous()
    _check_cache_shape(k, k_cache, 2)
    _check_cache_shape(v, v_cache, 2)
    # Positions are bounded by the K cache's extents in both writes.
    if v_cache.shape[0] < k_cache.shape[0] or v_cache.shape[1] < k_cache.shape[1]:
        raise ValueError(f"the V cache {tuple(v_cache.shape)} is smaller than the K cache {tuple(k_cache.shape)}")
    writes = [(x, c, s) for x, c, s in ((k, k_cache, k_scale), (v, v_cache, v_scale)) if x.numel()]
    if not writes:
        return None
    keep += [lengths, rows, table]
    args = _lib.AppendArgs()
    for i, (x, c, s) in enumerate(writes):
        args.kv[i] = _write_desc(x, c, s, x.stride()[1:], keep)
        args.x_batch_stride[i] = x.stride(0)
    args.lengths = lengths.data_ptr()
    args.batch_index = _lib.ptr(rows)
    args.block_table = _lib.ptr(table)
    args.batch, args.new_tokens = batch, k.shape[1]
    args.page_size, args.num_blocks = k_cache.shape[1], k_cache.shape[0]
    args.table_rows, args.table_cols = (0, 0) if table is None else tuple(table.shape)
    return args


def rotary_append(q, k, v, k_cache, v_cache, lengths, cos, sin, *, cache_batch_idx=None, cache_leftpad=None,
                  block_table=None, rotary_interleaved=True, causal=False, window_size=(-1, -1)):
    """rotary() of q and k (cos / sin None: neither) and append_kvcache() of
    (k, v), in one launch where q, k and v share a type and nothing is empty.

    Returns (q rotated, the lengths after the append less cache_leftpad)."""
    one_launch = (q.dtype == k.dtype == v.dtype and q.dtype in _INPUT_TYPES and q.ndim == 4 and k.ndim == 4
                  and q.numel() and k.numel() and v.numel() and lengths.numel() == k.shape[0]
                  and (cos is None or (cos.numel() and cos.dtype in _INPUT_TYPES and sin.dtype == cos.dtype
                                       and cos.device == sin.device == q.device))
                  and (cache_leftpad is None or (cache_leftpad.dtype == torch.int32 and cache_leftpad.device == q.device
                                                 and cache_leftpad.shape == k.shape[:1])))
    if not one_launch:
        if cos is not None:
            q, k = rotary(q, k, cos, sin, lengths, rotary_interleaved=rotary_interleaved, causal=causal,
                          window_size=window_size)
        append_kvcache(k, v, k_cache, v_cache, lengths, cache_batch_idx=cache_batch_idx, cache_leftpad=cache_leftpad,
                       block_table=block_table)
        lengths = lengths + k.shape[1]
        return q, lengths if cache_leftpad is None else lengths - cache_leftpad
    if cos is not None:
        _check_rotary(q, k, cos, sin)
    keep = []
    append = _append_args(k, v, k_cache, v_cache, lengths, cache_batch_idx, cache_leftpad, block_table, None, None, keep)
    a = _lib.StepArgs()
    a.size, a.kv = ctypes.sizeof(_lib.StepArgs), append
    after = torch.empty(k.shape[0], dtype=torch.int32, device=k.device)
    a.lengths_out = after.data_ptr()
    if cache_leftpad is not None:
        a.leftpad, a.leftpad_stride = cache_leftpad.data_ptr(), cache_leftpad.stride(0)
    if cos is not None:
        rotated = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        a.q, a.q_out = q.data_ptr(), rotated.data_ptr()
        a.q_seq, a.q_heads, a.q_dim = q.shape[1:]
        a.q_stride[:] = q.stride()
        a.cos_table, a.sin_table, a.trig_dtype = cos.data_ptr(), sin.data_ptr(), _lib.DTYPE_CODE[cos.dtype]
        a.cos_stride[:], a.sin_stride[:] = cos.stride(), sin.stride()
        a.half_rot, a.table_rows = cos.shape[1], cos.shape[0]
        a.interleaved = int(bool(rotary_interleaved))
        a.q_advance = int(bool(causal) or tuple(window_size) != (-1, -1))
        q = rotated
    _lib.call("fa_rotary_append", a, k.device)
    return q, after


def _check_rotary(q, k, cos, sin):
    _require_gpu(q=q, k=k, cos=cos, sin=sin)
    if q.ndim != 4 or (k is not None and (k.ndim != 4 or k.shape[0] != q.shape[0])):
        raise ValueError("q and k must be [batch, tokens, heads, dim] with one batch")
    if cos.ndim != 2 or sin.shape != cos.shape or 2 * cos.shape[1] > q.shape[-1]:
        raise ValueError(f"cos/sin must be [positions, rotary_dim / 2] with rotary_dim <= {q.shape[-1]}; "
                         f"got {tuple(cos.shape)} / {tuple(sin.shape)}")
    for x in (q, k):
        if x is None:
            continue
        if x.dtype not in _INPUT_TYPES:
            raise TypeError(f"rotary embedding takes float16, bfloat16 or float32; got {x.dtype}")
        if 2 * cos.shape[1] > x.shape[-1]:
            raise ValueError(f"rotary_dim {2 * cos.shape[1]} exceeds the head dim {x.shape[-1]}")


def rotary(q, k, cos, sin, cache_seqlens, *, rotary_interleaved=True, causal=False, window_size=(-1, -1)):
    """Rotary embedding of q [B, Sq, Hq, D] and new k [B, Snew, Hkv, D] (fresh tensors).

    cos/sin are [positions, rotary_dim / 2]; the first rotary_dim dims rotate
    as interleaved pairs (2i, 2i+1) or as halves (i, i + rotary_dim / 2).  New
    key j sits at cache_seqlens[b] + j; queries advance with j only for causal
    or local attention, else all sit at cache_seqlens[b]
    (flash_attn_mps/_cache.py:130-155).  A position past the table rotates to NaN.
    """
    _check_rotary(q, k, cos, sin)
    cos32, sin32 = cos.float().contiguous(), sin.float().contiguous()
    lengths = _per_request(cache_seqlens, q.shape[0], q.device, "cache_seqlens")
    query_moves = bool(causal) or tuple(window_size) != (-1, -1)
    rotated = []
    for x, advance in ((q, query_moves), (k, True)):
        if x is None:
            rotated.append(None)
            continue
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.numel():
            a = _lib.RotaryArgs()
            a.x, a.out = x.data_ptr(), y.data_ptr()
            a.cos_table, a.sin_table, a.lengths = cos32.data_ptr(), sin32.data_ptr(), lengths.data_ptr()
            a.dtype = _lib.DTYPE_CODE[x.dtype]
            a.interleaved, a.advance = int(bool(rotary_interleaved)), int(advance)
            a.batch, a.seq, a.heads, a.dim = x.shape
            a.half_rot, a.table_rows = cos.shape[1], cos.shape[0]
            a.x_stride[:] = x.stride()
            _lib.call("fa_rotary", a, x.device)
        rotated.append(y)
    return tuple(rotated)


@lru_cache(maxsize=64)
def _pair_axis_words(pair_axes, half, axes):
    """The axis of each rotated pair, two bits a pair in eight 64-bit words."""
    if pair_axes is None:
        if axes > 1:
            raise ValueError(f"positions on {axes} axes need pair_axes, the axis of each of the {half} rotated pairs")
        return (0,) * 8
    try:
        pair_axes = [operator.index(a) for a in pair_axes]
    except TypeError:
        pair_axes = []
    if len(pair_axes) != half or any(not 0 <= a < axes for a in pair_axes):
        raise ValueError(f"pair_axes must hold one axis in 0..{axes - 1} for each of the {half} rotated pairs")
    words = [0] * 8
    for i, a in enumerate(pair_axes):
        words[i >> 5] |= a << (2 * (i & 31))
    return tuple(words)


_NO_ROTATION = (0,) * 23


def _rotation(cos, sin, positions, pair_axes, interleaved, tokens, dims, device):
    """The fa_rotation fields of a checked rotation of rows with head dims `dims`."""
    if cos.ndim != 2 or sin.shape != cos.shape or sin.dtype != cos.dtype:
        raise ValueError(f"rotary_cos {tuple(cos.shape)} and rotary_sin {tuple(sin.shape)} must be one "
                         "[positions, rotary_dim / 2] and one type")
    if cos.dtype not in _INPUT_TYPES:
        raise TypeError(f"rotary tables are float16, bfloat16 or float32; got {cos.dtype}")
    if cos.device != device or sin.device != device:
        raise ValueError(f"rotary tables on {cos.device} / {sin.device}; expected {device}")
    rows, half = cos.shape
    if half < 1 or rows < 1:
        raise ValueError(f"rotary tables {tuple(cos.shape)} hold no position or no pair")
    if 2 * half > min(dims):
        raise ValueError(f"rotary_dim {2 * half} exceeds the head dim {min(dims)}")
    axes, at = 1, (0, 0, 1, 0, 0)
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64; got {positions.dtype}")
        if positions.device != device:
            raise ValueError(f"positions is on {positions.device}; expected {device}")
        shape = positions.shape
        if len(shape) not in (1, 2) or shape[-1] != tokens or (len(shape) == 2 and not 1 <= shape[0] <= 4):
            raise ValueError(f"positions {tuple(shape)} must be [{tokens}] or [axes, {tokens}] with 1 to 4 axes")
        axes = shape[0] if len(shape) == 2 else 1
        at = (positions.data_ptr(), _lib.I64 if positions.dtype == torch.int64 else _lib.I32, axes,
              positions.stride(0) if len(shape) == 2 else 0, positions.stride(-1))
    if pair_axes is not None and type(pair_axes) is not tuple:
        if torch.is_tensor(pair_axes):
            raise TypeError("pair_axes is a sequence of ints on the host")
        pair_axes = tuple(pair_axes)
    return (cos.data_ptr(), sin.data_ptr(), _lib.DTYPE_CODE[cos.dtype], int(bool(interleaved)), half, rows,
            *cos.stride(), *sin.stride(), *at, *_pair_axis_words(pair_axes, half, axes))


def _check_rows(**rows):
    """Packed rows [tokens, heads, dim] on one GPU, of one input type and token count."""
    first = None
    for name, x in rows.items():
        if x is None:
            continue
        if not on_gpu(x):
            raise ValueError(f"{name} is on {x.device}; cache operations run on a ROCm GPU")
        if x.ndim != 3 or not 1 <= x.shape[2] <= 512 or x.shape[1] < 1:
            raise ValueError(f"{name} {tuple(x.shape)} must be [tokens, heads, dim] with dim in 1..512")
        if x.dtype not in _INPUT_TYPES:
            raise TypeError(f"{name} is {x.dtype}; rows are float16, bfloat16 or float32")
        if first is None:
            first = x
        elif x.shape[0] != first.shape[0] or x.device != first.device:
            raise ValueError(f"{name} {tuple(x.shape)} on {x.device} does not go with {tuple(first.shape)} on {first.device}")
        elif x.dtype != first.dtype:
            raise TypeError(f"{name} is {x.dtype}; the rows of one call share one type, here {first.dtype}")
    return first


_NO_ROWS = (0,) * 7


def _rows(x, out):
    """The fa_rows fields of rows x written to contiguous `out`."""
    return x.data_ptr(), out.data_ptr(), x.shape[1], x.shape[2], *x.stride()


def rotary_embedding(q, k, cos, sin, positions, *, pair_axes=None, interleaved=True):
    """q [T, Hq, D] and k [T, Hk, D] (None: q alone) turned, as fresh tensors."""
    reject_training(tensors=(q, k, cos, sin))
    _check_rows(q=q, k=k)
    tokens, device = q.shape[0], q.device
    if positions is None:
        raise ValueError("rotary_embedding needs the rows' positions")
    rot = _rotation(cos, sin, positions, pair_axes, interleaved, tokens,
                    [q.shape[2]] if k is None else [q.shape[2], k.shape[2]], device)
    out_q = torch.empty(q.shape, dtype=q.dtype, device=device)
    out_k = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=device)
    if tokens:
        a = _lib.pack_rotary_rows(*_rows(q, out_q), *(_NO_ROWS if k is None else _rows(k, out_k)), tokens,
                                  _lib.DTYPE_CODE[q.dtype], 0, *rot)
        _lib.call("fa_rotary_rows", a, device)
    return out_q, out_k


def append_paged_kvcache(k, v, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, *, q=None, cos=None, sin=None,
                         positions=None, pair_axes=None, interleaved=True, k_scale=None, v_scale=None):
    """The rows of each request, its last seqused_k[b] positions, into its pages (see the package's function)."""
    reject_training(tensors=(k, v, k_cache, v_cache, q, cos, sin))
    _check_rows(k=k, v=v, q=q)
    tokens, heads, dim_k = k.shape
    device, dtype, shape = k.device, k.dtype, k_cache.shape
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    if v.shape[1] != heads:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have the same heads")
    for name, x, cache in (("k_cache", k, k_cache), ("v_cache", v, v_cache)):
        if cache.device != device:
            raise ValueError(f"{name} is on {cache.device}; expected {device}")
        _check_cache_shape(x, cache, 1)
        if cache.dtype != dtype and cache.dtype != torch.float8_e4m3fn:
            raise TypeError(f"a {cache.dtype} cache cannot take {dtype} rows (use the same dtype or float8_e4m3fn)")
    pages, size = shape[0], shape[1]
    if v_cache.shape[:2] != shape[:2] or v_cache.dtype != k_cache.dtype or size < 1:
        raise ValueError("the K and V caches must have the same pages, page size and type")
    for t in (cu_seqlens_q, seqused_k, block_table):
        if not torch.is_tensor(t):
            raise ValueError("cu_seqlens_q, seqused_k and block_table are int32 tensors [B + 1], [B] and [B, pages]")
    batch = seqused_k.numel()
    _check(seqused_k, "seqused_k", (batch,), (torch.int32,), device)
    _check(cu_seqlens_q, "cu_seqlens_q", (batch + 1,), (torch.int32,), device)
    _check(block_table, "block_table", (batch, None), (torch.int32,), device)
    blocks = is_block_scale(k_scale)
    if blocks != is_block_scale(v_scale):
        raise ValueError("k_scale and v_scale are both scales per block (float8_e8m0fnu) or neither")
    block, block_ptrs, block_strides, head_scale = 0, (0, 0), (0,) * 6, ((0, 0), (0, 0))
    if blocks:
        block = block_of(k_cache, k_scale, "k_scale")
        if block_of(v_cache, v_scale, "v_scale") != block:
            raise ValueError("the K and V scales must have the same tokens per block")
        block_ptrs, block_strides = (k_scale.data_ptr(), v_scale.data_ptr()), (*k_scale.stride(), *v_scale.stride())
    elif fp8:
        keep = [_per_head_scale(s, heads, device) for s in (k_scale, v_scale)]
        head_scale = [(s.data_ptr(), stride) for s, stride in keep]
    if (cos is None) != (sin is None):
        raise ValueError("rotary_cos and rotary_sin come together")
    if cos is None:
        if q is not None or positions is not None or pair_axes is not None:
            raise ValueError("q, positions and pair_axes go with rotary_cos and rotary_sin")
        rot = _NO_ROTATION
    else:
        rot = _rotation(cos, sin, positions, pair_axes, interleaved, tokens,
                        [k.shape[2]] if q is None else [k.shape[2], q.shape[2]], device)
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=device)
    if tokens:
        x_code, c_code = _lib.DTYPE_CODE[dtype], _lib.DTYPE_CODE[k_cache.dtype]
        (k_s, k_st), (v_s, v_st) = head_scale
        a = _lib.pack_append(
            k.data_ptr(), k_cache.data_ptr(), k_s, x_code, c_code, heads, dim_k, *k.stride(), *k_cache.stride(), k_st,
            v.data_ptr(), v_cache.data_ptr(), v_s, x_code, c_code, heads, v.shape[2], *v.stride(), *v_cache.stride(), v_st,
            *block_ptrs, *block_strides, block, *(_NO_ROWS if q is None else _rows(q, out)), *rot,
            cu_seqlens_q.data_ptr(), *cu_seqlens_q.stride(), seqused_k.data_ptr(), *seqused_k.stride(),
            block_table.data_ptr(), *block_table.stride(), tokens, batch, size, pages, block_table.shape[1])
        _lib.call("fa_paged_append", a, device)
    return out
