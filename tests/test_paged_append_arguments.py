"""Host-side contract of rotary_embedding and append_paged_kvcache, and of the C
entries under them, without a GPU: what is refused, with which error, before
anything is launched; and the definition that the GPU tests hold them to."""
import ctypes

import pytest
import torch

import flash_attn_mps_amd as fa
from block_cache import CODE, SCALE, append, encode, exponent, random_cache, scale_values
from flash_attn_mps_amd import _cache, _lib


@pytest.fixture
def launches(monkeypatch):
    """Host tensors taken for GPU ones; the launches that the calls would make."""
    made = []
    monkeypatch.setattr(_cache, "on_gpu", lambda t: True)
    monkeypatch.setattr(_lib, "call", lambda name, args, device: made.append((name, args)))
    return made


def rotary(**change):
    args = dict(q=torch.zeros(6, 4, 64, dtype=torch.float16), k=torch.zeros(6, 2, 64, dtype=torch.float16),
                rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 32), positions=torch.zeros(6, dtype=torch.int64))
    args.update(change)
    return fa.rotary_embedding(**args)


def paged(block=True, **change):
    rows = torch.zeros(6, 2, 64, dtype=torch.float16)
    cache = torch.zeros(5, 32, 2, 64).to(CODE) if block else torch.zeros(5, 32, 2, 64, dtype=torch.float16)
    scale = torch.zeros(5, 2, 2, dtype=torch.uint8).view(SCALE) if block else None
    args = dict(k=rows, v=rows, k_cache=cache, v_cache=cache.clone(), cu_seqlens_q=torch.tensor([0, 2, 6], dtype=torch.int32),
                seqused_k=torch.tensor([5, 6], dtype=torch.int32), block_table=torch.zeros(2, 2, dtype=torch.int32),
                q=torch.zeros(6, 4, 64, dtype=torch.float16), rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 32),
                k_scale=scale, v_scale=None if scale is None else scale.clone())
    args.update(change)
    return fa.append_paged_kvcache(**args)


def test_accepted_calls_launch_once(launches):
    q, k = rotary()
    assert q.shape == (6, 4, 64) and k.shape == (6, 2, 64)
    rotary(k=None, positions=torch.zeros(3, 6, dtype=torch.int32), pair_axes=[0, 1, 2, 0] * 8)
    assert paged().shape == (6, 4, 64) and paged(block=False).shape == (6, 4, 64)
    assert paged(q=None, rotary_cos=None, rotary_sin=None) is None
    paged(k_scale=0.5, v_scale=torch.ones(2))
    assert [name for name, _ in launches] == ["fa_rotary_rows"] * 2 + ["fa_paged_append"] * 4
    words = launches[1][1].rot.pair_axis
    assert [words[0] >> 2 * i & 3 for i in range(32)] == [0, 1, 2, 0] * 8 and launches[1][1].rot.axes == 3
    assert launches[2][1].block == 16 and launches[3][1].block == 0


ROWS = torch.zeros(6, 2, 64, dtype=torch.float16)


@pytest.mark.parametrize("change,error,match", [
    (dict(positions=None), ValueError, "positions"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), ValueError, "positions"),
    (dict(positions=torch.zeros(5, 6, dtype=torch.int64)), ValueError, "positions"),
    (dict(positions=torch.zeros(6)), ValueError, "int32 or int64"),
    (dict(positions=torch.zeros(2, 6, dtype=torch.int64)), ValueError, "pair_axes"),
    (dict(positions=torch.zeros(2, 6, dtype=torch.int64), pair_axes=[0, 2] * 16), ValueError, "pair_axes"),
    (dict(pair_axes=[0] * 31), ValueError, "pair_axes"),
    (dict(pair_axes=[True] * 32), ValueError, "pair_axes"),
    (dict(pair_axes=torch.zeros(32)), TypeError, "host"),
    (dict(pair_axes=[0.5] * 32), ValueError, "pair_axes"),
    (dict(rotary_cos=torch.zeros(9, 0), rotary_sin=torch.zeros(9, 0)), ValueError, "no position or no pair"),
    (dict(rotary_cos=torch.zeros(0, 32), rotary_sin=torch.zeros(0, 32)), ValueError, "no position or no pair"),
    (dict(rotary_sin=torch.zeros(9, 31)), ValueError, "rotary_sin"),
    (dict(rotary_cos=torch.zeros(9, 33), rotary_sin=torch.zeros(9, 33)), ValueError, "head dim"),
    (dict(rotary_cos=torch.zeros(9, 32, dtype=torch.float64), rotary_sin=torch.zeros(9, 32, dtype=torch.float64)), TypeError, "tables"),
    (dict(k=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), TypeError, "one type"),
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), ValueError, "does not go with"),
    (dict(q=torch.zeros(6, 4, 64, dtype=torch.float64)), TypeError, "float16"),
    (dict(q=torch.zeros(6, 4, 513)), ValueError, "dim"),
    (dict(q=torch.zeros(6, 64, dtype=torch.float16)), ValueError, "tokens, heads, dim"),
    (dict(q=torch.zeros(6, 4, 64, requires_grad=True)), NotImplementedError, "grad"),
])
def test_rotary_refusals(launches, change, error, match):
    with pytest.raises(error, match=match):
        rotary(**change)
    assert not launches


@pytest.mark.parametrize("change,error,match", [
    (dict(v=torch.zeros(6, 3, 64, dtype=torch.float16)), ValueError, "same heads"),
    (dict(v=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), TypeError, "one type"),
    (dict(k_cache=torch.zeros(5, 32, 2, 32).to(CODE)), ValueError, "cache"),
    (dict(k_cache=torch.zeros(5, 32, 2, 64), v_cache=torch.zeros(5, 32, 2, 64)), TypeError, "cannot take"),
    (dict(v_cache=torch.zeros(4, 32, 2, 64).to(CODE)), ValueError, "same pages"),
    (dict(v_scale=None), ValueError, "neither"),
    (dict(v_scale=torch.zeros(5, 4, 2, dtype=torch.uint8).view(SCALE)), ValueError, "tokens per block"),
    (dict(k_scale=torch.zeros(5, 3, 2, dtype=torch.uint8).view(SCALE)), ValueError, "blocks dividing"),
    (dict(k_scale=torch.zeros(4, 2, 2, dtype=torch.uint8).view(SCALE)), ValueError, "blocks dividing"),
    (dict(k_scale=torch.zeros(5, 0, 2, dtype=torch.uint8).view(SCALE)), ValueError, "blocks dividing"),
    (dict(block=False, k_scale=torch.zeros(5, 2, 2, dtype=torch.uint8).view(SCALE),
          v_scale=torch.zeros(5, 2, 2, dtype=torch.uint8).view(SCALE)), TypeError, "float8_e4m3fn"),
    (dict(cu_seqlens_q=torch.tensor([0, 6], dtype=torch.int32)), ValueError, "cu_seqlens_q"),
    (dict(seqused_k=torch.tensor([5, 6])), ValueError, "seqused_k"),
    (dict(seqused_k=[5, 6]), ValueError, "int32 tensors"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "block_table"),
    (dict(rotary_sin=None), ValueError, "come together"),
    (dict(rotary_cos=None, rotary_sin=None), ValueError, "go with"),
    (dict(q=torch.zeros(6, 4, 32, dtype=torch.float16)), ValueError, "head dim"),
    (dict(positions=torch.zeros(3, 6, dtype=torch.int64)), ValueError, "pair_axes"),
    (dict(k_scale=torch.ones(3), v_scale=torch.ones(3)), ValueError, "one per KV head"),
    (dict(v=torch.zeros(6, 2, 64, dtype=torch.float16, requires_grad=True)), NotImplementedError, "grad"),
])
def test_append_refusals(launches, change, error, match):
    with pytest.raises(error, match=match):
        paged(**change)
    assert not launches


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        rotary()
    with pytest.raises(ValueError, match="GPU"):
        paged()


def test_slot_writes_refuse_block_scales():
    scale = torch.zeros(1, 1, 2, dtype=torch.uint8).view(SCALE)
    with pytest.raises(TypeError, match="append_paged_kvcache"):
        _cache._per_head_scale(scale, 2, torch.device("cpu"))


@pytest.mark.parametrize("name,struct", [("fa_rotary_rows", _lib.RotaryRowsArgs), ("fa_paged_append", _lib.PagedAppendArgs),
                                         ("fa_block_attn_fwd", _lib.BlockAttnArgs)])
def test_c_entries_refuse_null_and_mismatched_arguments(name, struct):
    fn = getattr(_lib.load(), name)
    assert fn(None, None) == 1
    args = struct()
    assert fn(ctypes.byref(args), None) == 1                 # size 0
    args.size = ctypes.sizeof(struct)
    if hasattr(args, "tokens"):
        args.tokens = 1
    else:
        args.attn.num_splits = 1
    assert fn(ctypes.byref(args), None) == 1                 # null tensors
    assert _lib.load().fa_last_error().decode().startswith(name)


def _c_append():
    a = _lib.PagedAppendArgs()
    a.size, a.tokens, a.batch, a.page_size, a.num_pages, a.table_cols = ctypes.sizeof(a), 1, 1, 16, 1, 1
    a.cu_seqlens_q = a.seqused_k = a.block_table = 64
    for d in a.kv:
        d.x = d.cache = d.scale = 64
        d.x_dtype, d.cache_dtype, d.heads, d.dim = _lib.F16, _lib.E4M3, 1, 64
    return a


@pytest.mark.parametrize("spoil,match", [
    (lambda a: setattr(a, "block", 5), "pages they divide"),
    (lambda a: setattr(a, "block", 32), "pages they divide"),
    (lambda a: setattr(a, "block", 16), "null block scales"),
    (lambda a: setattr(a.kv[1], "dim", 513), "heads or dims"),
    (lambda a: setattr(a.kv[1], "heads", 2), "heads or dims"),
    (lambda a: setattr(a.kv[0], "scale", None), "needs a scale"),
    (lambda a: setattr(a.kv[1], "cache_dtype", _lib.F16), "share dtypes"),
    (lambda a: setattr(a.rot, "cos_table", 64), "come together"),
    (lambda a: (setattr(a.rot, "cos_table", 64), setattr(a.rot, "sin_table", 64), setattr(a.rot, "half_rot", 33)), "exceeds"),
    (lambda a: (setattr(a.rot, "cos_table", 64), setattr(a.rot, "sin_table", 64), setattr(a.rot, "half_rot", 32),
                setattr(a.rot, "positions", 64), setattr(a.rot, "axes", 5)), "axes"),
    (lambda a: setattr(a, "page_size", 0), "bad sizes"),
    (lambda a: setattr(a, "seqused_k", None), "null lengths"),
])
def test_c_append_refuses(spoil, match):
    a = _c_append()
    spoil(a)
    assert _lib.load().fa_paged_append(ctypes.byref(a), None) == 1
    assert match in _lib.load().fa_last_error().decode()


def test_exponent_and_encoder_of_the_definition():
    assert exponent(448.0) == 0 and exponent(448.0 * (1 + 2.0 ** -20)) == 1 and exponent(0.0) == -100
    x = torch.linspace(-500, 500, 4001, dtype=torch.float64)
    assert torch.equal(encode(x), x.float().clamp(-448, 448).to(CODE).double())
    tiny = torch.arange(-64, 65, dtype=torch.float64) * 2.0 ** -12
    assert torch.equal(encode(tiny), tiny.float().to(CODE).double())


def test_definition_keeps_and_codes_again():
    """A block with 5 rows that takes a row eight times larger: scale 8 times larger, rows coded again."""
    cache, _ = random_cache(1, 16, 16, 1, 64, 1)
    scale = torch.full((1, 1, 1), 127, dtype=torch.uint8).view(SCALE)
    x = torch.full((1, 1, 64), 8 * 448.0, dtype=torch.float64)
    code, factor = append(cache, scale, x, torch.tensor([0, 1]), torch.tensor([6]), torch.zeros(1, 1, dtype=torch.int32))
    assert factor.item() == 8 and (code[0, 5] == 448).all() and torch.equal(code[0, 6:], cache[0, 6:].double())
    assert torch.equal(code[0, :5], encode(cache[0, :5].double() / 8)) and scale_values(scale).item() == 1


def _attend(monkeypatch, **change):
    """Problem.validate of a block-scaled call on host tensors taken for GPU ones."""
    from flash_attn_mps_amd._problem import Problem
    k = torch.zeros(5, 32, 2, 64).to(CODE)
    scale = torch.zeros(5, 2, 2, dtype=torch.uint8).view(SCALE)
    args = dict(k=k, v=k.clone(), used_k=torch.tensor([4], dtype=torch.int32), table=torch.zeros(1, 2, dtype=torch.int32),
                k_descale=scale, v_descale=scale.clone())
    args.update(change)
    problem = Problem(torch.zeros(2, 4, 64, dtype=torch.float16), args.pop("k"), args.pop("v"), torch.tensor([0, 2], dtype=torch.int32),
                      2, 64, **args)
    cuda = torch.device("cuda")
    monkeypatch.setattr(torch.Tensor, "device", property(lambda t: cuda), raising=False)
    return problem.validate()


@pytest.mark.parametrize("change,error,match", [
    (dict(v_descale=None), ValueError, "come together"),
    (dict(v_descale=torch.zeros(5, 4, 2, dtype=torch.uint8).view(SCALE)), ValueError, "one shape"),
    (dict(v_descale=torch.zeros(1, 2)), ValueError, "v_descale"),
    (dict(k_descale=torch.zeros(4, 2, 2, dtype=torch.uint8).view(SCALE)), ValueError, "k_descale"),
    (dict(k_descale=torch.zeros(1, 2)), ValueError, "k_descale|v_descale"),
    (dict(k_descale=torch.zeros(5, 3, 2, dtype=torch.uint8).view(SCALE), v_descale=torch.zeros(5, 3, 2, dtype=torch.uint8).view(SCALE)),
     ValueError, "do not divide"),
    (dict(k=torch.zeros(5, 32, 2, 64, dtype=torch.float16), v=torch.zeros(5, 32, 2, 64, dtype=torch.float16)), TypeError, "float8_e4m3fn"),
    (dict(leftpad=torch.zeros(1, dtype=torch.int32)), ValueError, "left padding"),
])
def test_attention_refusals(monkeypatch, change, error, match):
    with pytest.raises(error, match=match):
        _attend(monkeypatch, **change)


def test_attention_takes_block_scales(monkeypatch):
    assert _attend(monkeypatch).block_scaled


def test_wide_entry_refuses_null_and_mismatched_arguments():
    lib = _lib.load()
    assert lib.fa_block_wide_fwd(None, None) == 1 and not lib.fa_block_wide_supported(None)
    a = _lib.BlockWideArgs()
    assert lib.fa_block_wide_fwd(ctypes.byref(a), None) == 1
    a.size = ctypes.sizeof(a)
    assert lib.fa_block_wide_fwd(ctypes.byref(a), None) == 1 and not _lib.supported("fa_block_wide_supported", a)


@pytest.mark.parametrize("shape,stride", [((), 0), ((1,), 0), ((2,), 1), ((1, 2), 1)])
def test_slot_writes_take_e8m0_values(shape, stride):
    """One value, or one per head, converts whatever its type; three dims are scales per block."""
    scale = torch.full(shape, 124, dtype=torch.uint8).view(SCALE)
    got, step = _cache._per_head_scale(scale, 2, torch.device("cpu"))
    assert got.dtype == torch.float32 and (got == 0.125).all() and got.numel() == 1 + stride and step == stride


def test_append_takes_e8m0_values_as_scales_per_head(launches):
    scale = torch.tensor([124, 130], dtype=torch.uint8).view(SCALE)
    paged(k_scale=scale, v_scale=scale[:1])
    args = launches[0][1]
    assert args.block == 0 and [d.scale_stride for d in args.kv] == [1, 0]
    with pytest.raises(ValueError, match="one per KV head"):
        paged(k_scale=torch.zeros(5, 2, dtype=torch.uint8).view(SCALE), v_scale=None)


@pytest.mark.parametrize("dim,route", [(128, "tiles"), (96, "generic")])
def test_attention_without_memory_for_a_workspace(monkeypatch, dim, route):
    """A workspace that cannot be had leaves a prefill to the tiles, or to the generic kernel."""
    from flash_attn_mps_amd import _attention
    from flash_attn_mps_amd._problem import Problem
    codes = torch.zeros(4, 64, 2, dim).to(CODE)
    scale = torch.zeros(4, 4, 2, dtype=torch.uint8).view(SCALE)
    q = torch.zeros(128, 32, dim, dtype=torch.bfloat16)
    p = Problem(q, codes, codes.clone(), torch.tensor([0, 128], dtype=torch.int32), 128, 200,
                used_k=torch.tensor([200], dtype=torch.int32), table=torch.zeros(1, 4, dtype=torch.int32), causal=True,
                k_descale=scale, v_descale=scale.clone())
    a = _attention.build_args(p, torch.empty_like(q), torch.empty(32, 128))
    assert _attention.takes_prefill(p, a) and p.wide is not None
    p.wide, empty = None, torch.empty

    def short_of_memory(*size, **kw):
        if size[0] >= 200 * 2 * dim:
            raise torch.OutOfMemoryError("out of memory")
        return empty(*size, **kw)

    monkeypatch.setattr(torch, "empty", short_of_memory)
    assert _attention.takes_prefill(p, a) == (route == "tiles") and p.wide is None
