"""rotary_embedding and append_paged_kvcache on an MI355X against their definitions
in 64 bits (tests/block_cache.py).

Tolerances.  A rotated value is two products and a sum in fp32, each off by at
most half an ulp of a value at most |a| + |b|: with the final rounding,
2^-23 (|a| + |b|) + half a step of the result's type.  Copied values are exact.  A
code is off by the step that a rotated value near a border may take: values
compare within one E4M3 step (2^-3 of the value, 2^-9 of the scale), and at most
one in a thousand differs at all; without rotation they are equal.
"""
import pytest
import torch

import flash_attn_mps_amd as fa
from block_cache import CODE, SCALE, append, encode, offsets, pages_for, random_cache, rotate, rows_of, scale_values

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def normal(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def tables(rows, half, dtype=torch.float32):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def assert_rotated(got, ref, x, dtype):
    """got within the tolerance above of ref (float64), NaN for NaN; x: the input."""
    got = got.detach().cpu().double()
    bar = 2.0 ** -23 * 2 * x.double().abs().amax(-1, keepdim=True) + HALF_STEP[dtype] * ref.abs() + 2.0 ** -25
    assert torch.equal(got.isnan(), ref.isnan())
    assert ((got - ref).abs() <= bar)[~ref.isnan()].all()


def assert_codes(got, ref, exact):
    """Codes within one step of ref, nearly all (exact: all) equal."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ~ref.isnan()
    off = (got - ref)[ok].abs()
    if exact:
        assert (off == 0).all()
    else:
        assert (off <= (ref[ok].abs() * 2.0 ** -3).clamp(min=2.0 ** -9)).all()
        assert (off > 0).double().mean() <= 1e-3


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,half,interleaved", [(128, 64, False), (128, 64, True), (80, 40, False), (72, 20, True),
                                                  (64, 16, False), (33, 7, False), (512, 256, True), (6, 3, True)])
def test_rotary_axes(device, dtype, dim, half, interleaved):
    tokens, hq, hk = 37, 6, 2
    for axes in (1, 3):
        q, k = normal((tokens, hq, dim), 1, dtype), normal((tokens, hk, dim), 2, dtype)
        cos, sin = tables(50, half)
        pos = torch.randint(0, 50, (axes, tokens), generator=torch.Generator().manual_seed(3))
        pair_axes = None if axes == 1 else [i % 3 if i % 2 else 0 for i in range(half)]
        out = fa.rotary_embedding(q.to(device), k.to(device), cos.to(device), sin.to(device),
                                  (pos[0] if axes == 1 else pos).to(device), pair_axes=pair_axes,
                                  rotary_interleaved=interleaved)
        for got, x in zip(out, (q, k)):
            assert got.is_contiguous() and got.dtype == dtype
            assert_rotated(got, rotate(x, cos, sin, pos, pair_axes, interleaved), x, dtype)
            assert torch.equal(got.cpu()[..., 2 * half:], x[..., 2 * half:])


def test_rotary_views_types_and_positions(device):
    """Views of a packed projection, strided 16-bit tables, int32 positions with strides, positions without a row, k absent."""
    tokens, dim, half = 300, 64, 32
    packed = normal((tokens, 12, dim), 1, torch.bfloat16)
    wide = tables(40, 2 * half, torch.bfloat16)
    cos, sin = (t[:, ::2] for t in wide)
    pos = torch.randint(-2, 42, (tokens, 2), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    q, k, _ = packed.to(device).split([8, 2, 2], 1)
    ref = [rotate(x, cos, sin, pos.T, [0, 1] * 16, True) for x in packed.split([8, 2, 2], 1)]
    gc, gs = (t.to(device)[:, ::2] for t in wide)
    out_q, out_k = fa.rotary_embedding(q, k, gc, gs, pos.to(device).T, pair_axes=tuple([0, 1] * 16))
    assert_rotated(out_q, ref[0], packed[:, :8], torch.bfloat16)
    assert_rotated(out_k, ref[1], packed[:, 8:10], torch.bfloat16)
    alone, none = fa.rotary_embedding(q, None, gc, gs, pos.to(device).T, pair_axes=tuple([0, 1] * 16))
    assert none is None and torch.equal(alone.view(torch.int16), out_q.view(torch.int16))
    # elements with a stride, and an odd token stride (no vectors)
    odd = normal((tokens, 3, 2 * dim + 1), 5, torch.bfloat16)
    x = odd[..., 1::2]
    got, _ = fa.rotary_embedding(odd.to(device)[..., 1::2], None, gc, gs, pos.to(device)[:, 0].contiguous(),
                                 rotary_interleaved=False)
    assert_rotated(got, rotate(x, cos, sin, pos.T[:1], None, False), x, torch.bfloat16)


class Append:
    """One append: inputs on the CPU, the call, and its definition."""

    def __init__(self, new, lengths, page, block, heads, dims, dtype, cache, seed, rot=None, axes=1, interleaved=True,
                 hq=4, padding=0, trig=torch.float32):
        self.dtype, self.block, self.cache, self.interleaved = dtype, block, cache, interleaved
        self.cu, self.used = offsets(new), torch.tensor(lengths, dtype=torch.int32)
        tokens = sum(new) + padding
        self.tokens, self.padding = tokens, padding
        self.table, self.pages = pages_for(lengths, page, seed)
        dk, dv = dims
        self.k, self.v = normal((tokens, heads, dk), seed + 1, dtype), normal((tokens, heads, dv), seed + 2, dtype)
        self.scale = [None, None]
        if cache == "block":
            (kc, ks), (vc, vs) = (random_cache(self.pages, page, block, heads, d, seed + 3 + i) for i, d in enumerate(dims))
            self.caches, self.scale = [kc, vc], [ks, vs]
        elif cache == "head":
            self.caches = [torch.zeros(self.pages, page, heads, d).to(CODE) for d in dims]
            self.scale = [torch.rand(heads, generator=torch.Generator().manual_seed(seed + 5 + i)) + 0.01 for i in range(2)]
        else:
            self.caches = [normal((self.pages, page, heads, d), seed + 3, dtype) for d in dims]
        self.q = self.cos = self.sin = self.positions = self.pair_axes = None
        if rot:
            rows = max(lengths) + 3
            self.q = normal((tokens, hq, dk), seed + 7, dtype)
            self.cos, self.sin = tables(rows, rot // 2, trig)
            if axes > 1:
                self.positions = torch.randint(0, rows, (axes, tokens), generator=torch.Generator().manual_seed(seed + 8))
                self.pair_axes = tuple(i * axes // (rot // 2) for i in range(rot // 2))

    def call(self, device, caches=None, scale=None):
        to = lambda t: None if t is None else t.to(device)  # noqa: E731
        caches = [to(c) for c in self.caches] if caches is None else caches
        scale = [to(s) for s in self.scale] if scale is None else scale
        q = fa.append_paged_kvcache(to(self.k), to(self.v), *caches, to(self.cu), to(self.used), to(self.table), q=to(self.q),
                                    rotary_cos=to(self.cos), rotary_sin=to(self.sin), positions=to(self.positions),
                                    pair_axes=self.pair_axes, rotary_interleaved=self.interleaved, k_scale=scale[0],
                                    v_scale=scale[1])
        return q, caches, scale

    def where(self):
        return rows_of(self.cu, self.used, self.table, self.caches[0].shape[1], self.pages, self.tokens)

    def turned(self):
        """float64 q and k after the rotation."""
        if self.cos is None:
            return None, self.k.double()
        pos = self.positions
        if pos is None:
            pos = torch.full((1, self.tokens), -1)
            for b in range(len(self.used)):
                n = int(self.cu[b + 1] - self.cu[b])
                pos[0, self.cu[b]:self.cu[b + 1]] = int(self.used[b]) - n + torch.arange(n)
        q = rotate(self.q, self.cos, self.sin, pos, self.pair_axes, self.interleaved)
        if self.positions is None:
            behind = int(self.cu[-1])
            q[behind:] = self.q[behind:].double()
        return q, rotate(self.k, self.cos, self.sin, pos, self.pair_axes, self.interleaved)

    def check(self, q, caches, scale):
        ref_q, ref_k = self.turned()
        if ref_q is not None:
            assert_rotated(q, ref_q, self.q, self.dtype)
        for i, (x, start) in enumerate(((ref_k, self.caches[0]), (self.v.double(), self.caches[1]))):
            exact = i == 1 or self.cos is None
            if self.cache == "block":
                code, factor = append(start, self.scale[i], x, self.cu, self.used, self.table)
                got = scale_values(scale[i])
                assert torch.equal(got, factor)
                assert_codes(caches[i], code, exact)
                continue
            ref = start.double().clone()
            for t, _, _, page, row in self.where():
                ref[page, row] = encode(x[t] / self.scale[i].double()[:, None]) if self.cache == "head" else x[t]
            if self.cache == "head":
                assert_codes(caches[i], ref, False)
            elif exact:
                assert torch.equal(caches[i].cpu().double(), ref)
            else:
                for t, _, _, page, row in self.where():
                    assert_rotated(caches[i][page, row], ref[page, row], self.k[t], self.dtype)
                    ref[page, row] = caches[i][page, row].cpu().double()
                assert torch.equal(caches[i].cpu().double(), ref)   # the other rows as they were


CASES = {
    "one token": dict(new=[1], lengths=[1], page=16, block=16, heads=2, dims=(128, 128), rot=128),
    "decode": dict(new=[1] * 9, lengths=[1, 16, 17, 32, 33, 64, 65, 100, 200], page=32, block=16, heads=8, dims=(128, 128), rot=128, axes=3,
                   interleaved=False),
    "ragged": dict(new=[5, 0, 70, 1, 33, 16], lengths=[5, 40, 100, 64, 33, 48], page=64, block=32, heads=3, dims=(64, 64), rot=32),
    "long": dict(new=[300, 17], lengths=[333, 17], page=256, block=64, heads=2, dims=(256, 256), rot=256, interleaved=False),
    "block of the page": dict(new=[130, 3], lengths=[140, 130], page=128, block=128, heads=1, dims=(80, 80), rot=80),
    "odd block": dict(new=[20, 4], lengths=[31, 9], page=15, block=5, heads=2, dims=(72, 72), rot=24),
    "one row a block": dict(new=[3, 4], lengths=[31, 4], page=16, block=1, heads=2, dims=(64, 64)),
    "odd dims": dict(new=[9, 30], lengths=[20, 30], page=16, block=16, heads=3, dims=(33, 17), rot=14, interleaved=False),
    "value dim": dict(new=[9, 30], lengths=[20, 30], page=16, block=16, heads=2, dims=(192, 128), rot=64, axes=2),
    "padded": dict(new=[2, 3], lengths=[20, 3], page=16, block=16, heads=2, dims=(64, 64), rot=64, padding=4),
    "padded, own positions": dict(new=[2, 3], lengths=[20, 3], page=16, block=16, heads=2, dims=(64, 64), rot=64, axes=2, padding=4),
    "wide": dict(new=[2], lengths=[18], page=16, block=16, heads=2, dims=(512, 512), rot=512, interleaved=False),
    "many requests": dict(new=[1] * 150, lengths=[1 + 3 * i % 50 for i in range(150)], page=16, block=16, heads=1, dims=(64, 64), rot=64),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cache", ["block", "same", "head"])
@pytest.mark.parametrize("name", CASES)
def test_append(device, name, cache, dtype):
    case = Append(**CASES[name], dtype=dtype, cache=cache, seed=11)
    case.check(*case.call(device))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_blocks_fill_token_by_token(device, dtype):
    """40 tokens one at a time: every step as defined, scales growing and rows coded again."""
    heads, dim, page, block = 2, 64, 32, 16
    grow = 2.0 ** (torch.arange(40) * 7 % 23 - 11).float()
    table = torch.tensor([[3, 1]], dtype=torch.int32)
    state = [[torch.full((4, page, heads, dim), 0.0).to(CODE), torch.full((4, 2, heads), 200, dtype=torch.uint8).view(SCALE)]
             for _ in range(2)]
    on_gpu = [[t.to(device) for t in s] for s in state]
    for n in range(1, 41):
        k, v = (normal((1, heads, dim), 50 + n + 100 * i, dtype) * grow[n - 1].to(dtype) for i in range(2))
        cu, used = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
        fa.append_paged_kvcache(k.to(device), v.to(device), on_gpu[0][0], on_gpu[1][0], cu.to(device), used.to(device),
                                table.to(device), k_scale=on_gpu[0][1], v_scale=on_gpu[1][1])
        for i, x in enumerate((k, v)):
            code, factor = append(*state[i], x.double(), cu, used, table)
            state[i] = [t.cpu() for t in on_gpu[i]]
            assert torch.equal(scale_values(state[i][1]), factor), n
            assert_codes(state[i][0], code, True)


@pytest.mark.parametrize("fill", [0.0, -0.0, 448.0, 448.5, 2.0 ** -120, 2.0 ** -140, 3e38, float("inf"), float("nan")])
def test_block_extremes(device, fill):
    """Blocks of one magnitude: zero, the border, below the smallest scale, the largest, infinities and NaN."""
    x = torch.full((20, 1, 64), fill)
    x[3, 0, 5] = 1.0 if fill != fill or fill == float("inf") else x[3, 0, 5]
    codes, scale = random_cache(3, 16, 16, 1, 64, 3)
    cu, used = torch.tensor([0, 20], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    got, got_scale = codes.to(device), scale.to(device)
    other, other_scale = codes.to(device), scale.to(device)
    fa.append_paged_kvcache(x.to(device), x.to(device), got, other, cu.to(device), used.to(device), table.to(device),
                            k_scale=got_scale, v_scale=other_scale)
    code, factor = append(codes, scale, x.double(), cu, used, table)
    assert torch.equal(scale_values(got_scale), factor) and torch.equal(scale_values(other_scale), factor)
    for c in (got, other):
        assert_codes(c, code, True)
        assert torch.equal(torch.signbit(c.cpu().float()), torch.signbit(code)) or fill != fill


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotated_infinities_saturate(device, interleaved, dtype):
    """An infinity turns into two, which leave the scale alone and become the largest codes."""
    x = normal((20, 2, 64), 5, dtype)
    x[3, 0, 4], x[17, 1, 25], x[9, 0, 60] = float("inf"), -float("inf"), float("inf")
    codes, scale = random_cache(3, 16, 16, 2, 64, 3)
    cu, used = torch.tensor([0, 20], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    table, (cos, sin) = torch.tensor([[2, 0]], dtype=torch.int32), tables(20, 16)
    cache, caches_scale = codes.to(device), scale.to(device)
    fa.append_paged_kvcache(x.to(device), x.to(device), cache, cache.clone(), cu.to(device), used.to(device), table.to(device),
                            rotary_cos=cos.to(device), rotary_sin=sin.to(device), rotary_interleaved=interleaved,
                            k_scale=caches_scale, v_scale=caches_scale.clone())
    turned = rotate(x, cos, sin, torch.arange(20)[None], None, interleaved)
    assert turned.isinf().sum() == 5
    code, factor = append(codes, scale, turned, cu, used, table)
    assert torch.equal(scale_values(caches_scale), factor)
    assert_codes(cache, code, False)


def test_pages_out_of_reach_are_skipped(device):
    """Pages that are negative or past the cache, positions past the table, lengths below the new rows."""
    for cache in ("block", "same", "head"):
        case = Append(new=[8, 20, 6, 4], lengths=[8, 40, 30, 20], page=16, block=16, heads=2, dims=(64, 64), dtype=torch.bfloat16,
                      cache=cache, seed=5, rot=64)
        case.table[0, 0] = -1
        case.table[1, 1] = case.pages + 3
        case.used[1], case.used[2] = 40 + 16 * case.table.shape[1], 4    # rows past the table; two rows before position 0
        case.cos, case.sin = tables(200, 32)
        case.check(*case.call(device))


def test_strided_caches_scales_and_metadata(device):
    """Caches and scales with heads outside the pages, rows as views, metadata with strides."""
    case = Append(new=[3, 20], lengths=[30, 20], page=32, block=16, heads=4, dims=(64, 64), dtype=torch.float16, cache="block", seed=9,
                  rot=64)
    swapped = [c.transpose(1, 2).contiguous().to(device).transpose(1, 2) for c in case.caches]
    scales = [s.permute(2, 0, 1).contiguous().to(device).permute(1, 2, 0) for s in case.scale]
    packed = torch.cat([case.q, case.k, case.v], 1).to(device)
    q, k, v = packed.split([4, 4, 4], 1)
    every = lambda t: t.to(device).repeat_interleave(2)[::2]  # noqa: E731
    wide = torch.zeros(2, 2 * case.table.shape[1], dtype=torch.int32)
    wide[:, ::2] = case.table
    out = fa.append_paged_kvcache(k, v, *swapped, every(case.cu), every(case.used), wide.to(device)[:, ::2], q=q,
                                  rotary_cos=case.cos.to(device), rotary_sin=case.sin.to(device), k_scale=scales[0],
                                  v_scale=scales[1])
    case.check(out, swapped, scales)


def test_two_streams_and_a_replayed_graph(device):
    """The same append on another stream, and captured and replayed with eager work between: equal every time."""
    case = Append(new=[1, 1, 40], lengths=[17, 64, 60], page=32, block=16, heads=4, dims=(128, 128), dtype=torch.bfloat16, cache="block",
                  seed=21, rot=128, axes=3)
    q, caches, scale = case.call(device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        q2, caches2, scale2 = case.call(device)
    torch.cuda.synchronize()
    case.check(q2, caches2, scale2)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    held = [to(t) for t in (case.k, case.v, case.cu, case.used, case.table, case.q, case.cos, case.sin, case.positions)]
    caches3, scale3 = [to(c) for c in case.caches], [to(s) for s in case.scale]

    def step():
        k, v, cu, used, table, qq, cos, sin, pos = held
        return fa.append_paged_kvcache(k, v, *caches3, cu, used, table, q=qq, rotary_cos=cos, rotary_sin=sin, positions=pos,
                                       pair_axes=case.pair_axes, k_scale=scale3[0], v_scale=scale3[1])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for c, s, c0, s0 in zip(caches3, scale3, case.caches, case.scale):
            c.copy_(c0)
            s.view(torch.uint8).copy_(s0.view(torch.uint8))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), q.view(torch.int16))
        for got, want in zip((*caches3, *scale3), (*caches, *scale)):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_cache_past_32_bit_offsets(device):
    """The last page of a cache of more than 2^32 elements."""
    page, heads, dim = 256, 8, 128
    pages = 2 ** 32 // (page * heads * dim) + 3
    cache = torch.empty(pages, page, heads, dim, dtype=CODE, device=device)
    other = torch.empty(pages, page, heads, dim, dtype=CODE, device=device)
    scale, other_scale = (torch.zeros(pages, 16, heads, dtype=torch.uint8, device=device).view(SCALE) for _ in range(2))
    x = normal((5, heads, dim), 4, torch.bfloat16)
    cu, used, table = (torch.tensor(t, dtype=torch.int32, device=device) for t in ([0, 5], [5], [[pages - 1]]))
    fa.append_paged_kvcache(x.to(device), x.to(device), cache, other, cu, used, table, k_scale=scale, v_scale=other_scale)
    ref, factor = append(torch.zeros(1, page, heads, dim).to(CODE), scale[-1:].cpu(), x.double(), cu.cpu(), used.cpu(),
                         torch.zeros(1, 1, dtype=torch.int32))
    for c, s in ((cache, scale), (other, other_scale)):
        assert torch.equal(c[-1, :5].cpu().double(), ref[0, :5]) and torch.equal(scale_values(s[-1:])[:, 0], factor[:, 0])


def test_nothing_to_do(device):
    empty = torch.zeros(0, 2, 64, dtype=torch.float16, device=device)
    cache = torch.zeros(1, 16, 2, 64, dtype=torch.float16, device=device)
    cu, used, table = (torch.zeros(n, dtype=torch.int32, device=device) for n in ((2,), (1,), (1, 1)))
    cos, sin = (t.to(device) for t in tables(4, 32))
    q = fa.append_paged_kvcache(empty, empty, cache, cache.clone(), cu, used, table, q=empty, rotary_cos=cos, rotary_sin=sin)
    assert q.shape == empty.shape
    a, b = fa.rotary_embedding(empty, empty, cos, sin, torch.zeros(0, dtype=torch.int64, device=device))
    assert a.shape == b.shape == empty.shape
    # no requests: every row lies behind the last one
    x = normal((3, 2, 64), 1, torch.float16).to(device)
    q = fa.append_paged_kvcache(x, x, cache, cache.clone(), cu[:1], used[:0], table[:0], q=x, rotary_cos=cos, rotary_sin=sin)
    assert torch.equal(q, x) and not cache.any()


def test_rows_of_no_request(device):
    """A batch of padding alone: nothing is written, q is copied."""
    q, k = normal((5, 4, 64), 1, torch.bfloat16).to(device), normal((5, 2, 64), 2, torch.bfloat16).to(device)
    codes, scale = (t.to(device) for t in random_cache(3, 16, 16, 2, 64, 3))
    held = codes.clone(), codes.clone(), scale.clone(), scale.clone()
    i32 = dict(dtype=torch.int32, device=device)
    cos, sin = (t.to(device) for t in tables(4, 32))
    for batch in (0, 2):
        out = fa.append_paged_kvcache(k, k, held[0], held[1], torch.zeros(batch + 1, **i32), torch.full((batch,), 7, **i32),
                                      torch.zeros(batch, 1, **i32), q=q, rotary_cos=cos, rotary_sin=sin, k_scale=held[2],
                                      v_scale=held[3])
        assert torch.equal(out, q)
        for x, was in zip(held, (codes, codes, scale, scale)):
            assert torch.equal(x.view(torch.uint8), was.view(torch.uint8))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotated_overflows_saturate(device, interleaved, dtype):
    """Finite keys whose rotation leaves fp32's range, to either side: infinities, as those of infinite keys.

    Tables of magnitude 1.5 (scaled rotary embeddings) and keys of 3e38: a product of 4.5e38 overflows, and its pair's
    other key is 1, so each result is one such product, its sign that of the formula."""
    x = normal((20, 2, 64), 5, dtype)
    big = torch.tensor(3e38).to(dtype)
    cos, sin = (t * 1.5 for t in tables(20, 16))
    angle = torch.where(torch.arange(16) % 2 == 0, 1.0, -1.0).expand(20, 16)     # sin = +-1.5 cos = 0
    cos[10:], sin[10:] = 0.0, 1.5 * angle[10:]
    for row, pair, high, sign in ((12, 4, False, 1), (13, 5, False, 1), (14, 4, True, 1), (15, 5, True, 1), (16, 4, True, -1), (17, 5, False, -1)):
        lo, hi = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + 16)
        x[row, 1, lo], x[row, 1, hi] = (1.0, sign * big) if high else (sign * big, 1.0)
    cu, used = torch.tensor([0, 20], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    turned = rotate(x, cos, sin, torch.arange(20)[None], None, interleaved).float().double()     # 4.5e38: infinite
    assert turned.isinf().sum() == 6 and not turned.isnan().any()
    for scales in ("block", "head"):
        codes, scale = random_cache(3, 16, 16, 2, 64, 3)
        cache, got_scale = codes.to(device), scale.to(device) if scales == "block" else torch.ones(2, device=device)
        fa.append_paged_kvcache(x.to(device), x.to(device), cache, cache.clone(), cu.to(device), used.to(device), table.to(device),
                                rotary_cos=cos.to(device), rotary_sin=sin.to(device), rotary_interleaved=interleaved,
                                k_scale=got_scale, v_scale=got_scale.clone())
        if scales == "block":
            code, factor = append(codes, scale, turned, cu, used, table)
            assert torch.equal(scale_values(got_scale), factor)
        else:
            code = codes.double()
            code[2], code[0, :4] = encode(turned[:16]), encode(turned[16:])
        assert_codes(cache, code, False)


def test_e8m0_scales_per_head(device):
    """E8M0 values in place of fp32 ones, for a slot write and an append: the same codes."""
    k, v = (normal((5, 2, 64), i, torch.bfloat16).to(device) for i in (1, 2))
    scale = torch.tensor([120, 125], dtype=torch.uint8, device=device).view(SCALE)
    i32 = dict(dtype=torch.int32, device=device)
    got = []
    for s in (scale, scale.float()):
        caches = [torch.zeros(2, 16, 2, 64, device=device).to(CODE) for _ in range(4)]
        fa.store_kvcache(k, v, caches[0], caches[1], torch.arange(3, 8, device=device), k_scale=s, v_scale=s[1:])
        fa.append_paged_kvcache(k, v, caches[2], caches[3], torch.tensor([0, 5], **i32), torch.tensor([8], **i32),
                                torch.zeros(1, 1, **i32), k_scale=s, v_scale=s[1:])
        got.append(torch.stack([c.view(torch.uint8) for c in caches]))
    assert torch.equal(*got) and torch.equal(got[0][:2], got[0][2:])


def test_default_scale_made_in_a_capture(device, monkeypatch):
    """An append without scales, captured first: the eager calls before the graph's first replay do not read what it writes."""
    from flash_attn_mps_amd import _cache
    monkeypatch.setattr(_cache, "_ONES", {}, raising=False)
    x = normal((5, 2, 64), 1, torch.bfloat16)
    rows = x.to(device)
    cu, used, table = (torch.tensor(t, dtype=torch.int32, device=device) for t in ([0, 5], [5], [[0]]))
    caches = [torch.zeros(1, 16, 2, 64, device=device).to(CODE) for _ in range(4)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.append_paged_kvcache(rows, rows, caches[0], caches[1], cu, used, table)
    fa.append_paged_kvcache(rows, rows, caches[2], caches[3], cu, used, table)
    torch.cuda.synchronize()
    for got in (caches[2:], caches):
        for c in got:
            assert torch.equal(c[0, :5].cpu().double(), encode(x.double()))
        graph.replay()
        torch.cuda.synchronize()
