"""Attention over a block-scaled cache on an MI355X against the CPU oracle in 64
bits on the values that the cache stands for (tests/block_cache.py).

Tolerances.  An output is sum p v / sum p.  A 16-bit kernel rounds each p to the
queries' type and the output to its own, each by at most half a step, 2^-8 of
the number in bf16 and 2^-11 in fp16, so an output is off by at most twice that
of sum p |v| / sum p, which the oracle gives for |v|.  Scores, sums and
exponentials are fp32's: a sixty-fourth of
that on top (2^-13 in bf16, 2^-16 in fp16, of a sum) covers scores up to 16 with an
error of 2^-20 of them, and 1e-6 what is near zero.  LSEs: the bar of the other
attention tests (harness.assert_parity), 1e-4.
"""
import pytest
import torch

from block_cache import CODE, SCALE, offsets, pages_for, random_cache, scale_values, values
from flash_attn_mps_amd import vllm
from harness import OUT_BAR, assert_parity, oracle_attention

pytestmark = pytest.mark.gpu

# fp32 outputs: sums in fp32 over up to 1000 keys, 2^-24 of each partial sum.
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 1000 * 2.0 ** -24}


class Call:
    def __init__(self, new, lengths, page, block, hq, hkv, dim, dtype=torch.bfloat16, dim_v=None, seed=1, low=-9, spread=2, spare=2):
        self.new, self.lengths, self.dtype = new, lengths, dtype
        self.table, pages = pages_for(lengths, page, seed, spare)
        self.k, self.ks = random_cache(pages, page, block, hkv, dim, seed + 1, low, spread)
        self.v, self.vs = random_cache(pages, page, block, hkv, dim_v or dim, seed + 2, low, spread)
        g = torch.Generator().manual_seed(seed + 3)
        self.q = torch.randn(sum(new), hq, dim, generator=g).to(dtype)
        self.cu, self.used = offsets(new), torch.tensor(lengths, dtype=torch.int32)
        self.hq = hq

    def gpu(self, device, max_q=None, max_k=None, move=lambda t: t, **kw):
        to = lambda t: t.to(device)  # noqa: E731
        kw.setdefault("causal", True)
        for name in ("s_aux", "alibi_slopes", "dynamic_causal"):
            if kw.get(name) is not None:
                kw[name] = to(kw[name])
        if "aux_tensors" in kw:
            kw["aux_tensors"] = [to(t) for t in kw["aux_tensors"]]
        return vllm.flash_attn_varlen_func(
            to(self.q), move(to(self.k)), move(to(self.v)), max_q or max(self.new), to(self.cu), max_k or max(self.lengths),
            seqused_k=to(self.used), block_table=to(self.table), k_descale=move(to(self.ks)), v_descale=move(to(self.vs)),
            return_softmax_lse=True, **kw)

    def oracle(self, **kw):
        names = dict(window_size="window", mask_mod="mask", aux_tensors="aux", dynamic_causal="causal", s_aux="sinks",
                     alibi_slopes="alibi", softmax_scale="scale")
        kw.setdefault("causal", True)
        if kw.get("dynamic_causal") is not None:
            kw.pop("causal")
        kw = {names.get(k, k): v for k, v in kw.items() if k not in ("deterministic", "num_splits")}
        q = self.q.double() if self.dtype != torch.float32 else self.q
        table = self.table.clamp(min=0)
        return oracle_attention(q, values(self.k, self.ks), values(self.v, self.vs), self.cu, used_k=self.used,
                                block_table=table, **kw)

    def check(self, device, max_q=None, max_k=None, move=lambda t: t, **kw):
        out, lse = self.gpu(device, max_q, max_k, move, **kw)
        torch.cuda.synchronize()
        ref, ref_lse = self.oracle(**kw)
        assert_parity(out, lse, ref, ref_lse, out.dtype, out_bar=float("inf"))
        held, self.v = self.v, (self.v.view(torch.uint8) & 0x7f).view(CODE)
        bar = 2 * HALF_STEP[out.dtype] * self.oracle(**kw)[0] * (1 + 2.0 ** -6) + 1e-6
        self.v = held
        off = (out.cpu().double() - ref).abs()
        assert (off <= bar).all(), f"off by up to {(off / bar).max():.3f} of the tolerance"
        return out, lse


RAGGED = [1, 15, 16, 17, 64, 100, 257]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 8, 128), (8, 4, 128), (32, 8, 128), (6, 2, 128), (48, 1, 128), (4, 4, 64), (16, 2, 64),
                                        (24, 8, 64), (4, 2, 256), (3, 1, 80), (4, 2, 32)])
def test_decode(device, hq, hkv, dim, dtype):
    """One row a request, every length that a 16-key group can end in."""
    lengths = [*RAGGED, 1000, 31, 33, 48, 63]
    Call([1] * len(lengths), lengths, 32, 16, hq, hkv, dim, dtype).check(device)


@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 32), (64, 64), (256, 64), (48, 16), (96, 48), (128, 128), (32, 8), (64, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_and_blocks(device, page, block, dim):
    call = Call([1, 1, 1, 1], [5, 130, 1, 700], page, block, 8, 2, dim)
    call.check(device)
    Call([3, 1, 40, 16], [5, 130, 40, 300], page, block, 8, 2, dim).check(device)


@pytest.mark.parametrize("rows", [2, 4, 16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_rows(device, rows, dtype):
    """Speculative rows; requests with fewer rows than the longest, one with no key before them."""
    new = [rows, 1, rows, max(1, rows - 1), rows]
    lengths = [rows, 1, 70, 333, 900]
    for hq, hkv, dim in ((8, 2, 128), (8, 8, 64), (4, 4, 128)):
        Call(new, lengths, 64, 32, hq, hkv, dim, dtype).check(device)
        Call(new, lengths, 64, 32, hq, hkv, dim, dtype).check(device, causal=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (3, 1)])
def test_prefill(device, dim, hq, hkv, dtype):
    new, lengths = [130, 1, 64, 257, 33, 0, 5], [130, 1, 200, 257, 1000, 40, 300]
    for causal in (True, False):
        Call(new, lengths, 64, 16, hq, hkv, dim, dtype).check(device, causal=causal)


FEATURES = {
    "window": dict(window_size=(40, 0)),
    "right window": dict(causal=False, window_size=(-1, 5)),
    "window of one": dict(window_size=(0, 0)),
    "softcap": dict(softcap=5.0),
    "softcap and window": dict(softcap=5.0, window_size=(100, 0)),
    "scale": dict(softmax_scale=-0.05),
    "one split": dict(num_splits=1),
    "splits": dict(num_splits=7),
}


@pytest.mark.parametrize("dim", [64, 128, 256, 96])
@pytest.mark.parametrize("rows", [1, 5, 90])
@pytest.mark.parametrize("name", FEATURES)
def test_features(device, name, rows, dim):
    kw = dict(FEATURES[name])
    new, lengths = [rows, min(rows, 3), 1], [max(300, rows), 50, 700]
    Call(new, lengths, 64, 32, 8, 2, dim, low=-9).check(device, **kw)


@pytest.mark.parametrize("rows", [1, 5, 90])
def test_sinks_flags_and_biases(device, rows):
    new, lengths = [rows, min(rows, 3), 1], [max(300, rows), 50, 700]
    call = Call(new, lengths, 64, 32, 8, 2, 128)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(9)) * 2
    call.check(device, s_aux=sinks)
    call.check(device, s_aux=sinks, window_size=(30, 0))
    call.check(device, dynamic_causal=torch.tensor([True, False, True]))
    call.check(device, alibi_slopes=torch.rand(8, generator=torch.Generator().manual_seed(10)))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_vllm_masks(device, rows, dim):
    new, lengths = [rows, rows], [max(300, rows), 170]
    call = Call(new, lengths, 64, 32, 4, 2, dim)
    tokens = sum(new)
    lo = torch.randint(-1, 100, (tokens,), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    ranges = torch.stack([lo, lo + 40], 1)
    prefix, window = torch.tensor([20, 3], dtype=torch.int32), torch.tensor([50], dtype=torch.int32)
    for softcap in (0.0, 5.0):
        call.check(device, mask_mod=vllm.mm_prefix_mask(64), aux_tensors=[ranges, call.cu], softcap=softcap)
        call.check(device, mask_mod=vllm.rswa_mask(), aux_tensors=[prefix, window], softcap=softcap)


def test_fp32_and_e4m3_queries(device):
    """Queries of the other types."""
    for rows in (1, 20):
        call = Call([rows, 1], [200, 50], 64, 32, 4, 2, 128, torch.float32)
        call.check(device)
        call.q = call.q.clamp(-3, 3).to(CODE)
        call.dtype = CODE
        call.check(device)


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("low,spread,dtype", [(-40, 3, torch.bfloat16), (20, 3, torch.bfloat16), (-15, 8, torch.float16), (-60, 60, torch.bfloat16)])
def test_wide_scales(device, rows, low, spread, dtype):
    """V of magnitudes from 2^-31 to 2^32, blocks far apart; K near 1, so that scores stay moderate."""
    call = Call([rows, 1], [200, 90], 64, 16, 4, 2, 128, dtype)
    _, call.vs = random_cache(call.v.shape[0], 64, 16, 2, 128, 77, low, spread)
    out, lse = call.gpu(device)
    ref, ref_lse = call.oracle()
    peak = float(values(call.v, call.vs).abs().max())
    # As weighted means of values up to `peak`: every error is a few roundings of them.
    assert ((out.cpu().double() - ref).abs().max() <= OUT_BAR[dtype] * peak / 4 + 2.0 ** -24).item()
    assert ((lse.cpu().double() - ref_lse).abs().max() <= 1e-4).item()


def test_scale_bytes(device):
    """Scales at the ends of their range: 2^-127 (byte 0), 2^-126, and 2^119 in values that bf16 holds."""
    for e in (0, 1, 246):
        call = Call([1, 40], [90, 50], 64, 16, 4, 2, 64)
        call.vs.view(torch.uint8).fill_(e)
        out, lse = call.gpu(device)
        ref, ref_lse = call.oracle()
        peak = 448 * 2.0 ** (e - 127)
        assert ((out.cpu().double() - ref).abs().max() <= peak * 2.0 ** -8 + 2.0 ** -133).item()
        assert ((lse.cpu().double() - ref_lse).abs().max() <= 1e-4).item()
        call = Call([1, 40], [90, 50], 64, 16, 4, 2, 64)
        call.ks.view(torch.uint8).fill_(min(e, 1))
        call.check(device)      # scores of zero: the mean of the values


@pytest.mark.parametrize("rows", [1, 4, 60])
def test_nan_reaches_the_rows_that_see_it(device, rows):
    """A NaN code, and a scale of 255, in one KV head: NaN for its query heads, the other heads at the bar; hidden ones
    (past the length, out of the window) reach nothing.

    Not bit for bit: heads that share matrix products with the NaN's, and rows whose tile holds the hidden one, run again
    in fp32, without the rounding of probabilities to the queries' type, 2^-9 of each: at most 2^-9 sum p |v| of an
    output, below the bar (2^-6.6) for these |v| < 4."""
    for dim in (64, 128):
        base = Call([rows, 1], [128 + rows, 90], 64, 16, 8, 4, dim)
        want, _ = base.gpu(device, causal=False)
        for which in ("code", "scale"):
            call = Call([rows, 1], [128 + rows, 90], 64, 16, 8, 4, dim)
            page = int(call.table[0, 1])
            if which == "code":
                call.k.view(torch.uint8)[page, 3, 1, 5] = 0x7f
            else:
                call.ks.view(torch.uint8)[page, 0, 1] = 255
            out, _ = call.gpu(device, causal=False)
            assert out[:rows, 2:4].isnan().all()
            out[:rows, 2:4] = want[:rows, 2:4]
            assert ((out - want).abs() <= OUT_BAR[torch.bfloat16]).all()
        call = Call([rows, 1], [128 + rows, 90], 64, 16, 8, 4, dim)
        first, second = int(call.table[0, 0]), int(call.table[1, 1])
        for codes, scale in ((call.k, call.ks), (call.v, call.vs)):
            codes.view(torch.uint8)[first, :16] = 0x7f            # out of every row's window
            scale.view(torch.uint8)[first, 0] = 255
            codes.view(torch.uint8)[second, 26:] = 0xff           # past the second request's length
            scale.view(torch.uint8)[second, 2:] = 255
        out, _ = call.gpu(device, window_size=(100, 0))
        ref, _ = base.gpu(device, window_size=(100, 0))
        assert ((out - ref).abs() <= OUT_BAR[torch.bfloat16]).all()


def test_empty_requests_and_padding(device):
    """No keys, no rows, rows behind the last request left as they were."""
    call = Call([1, 1, 1], [40, 0, 17], 16, 16, 8, 2, 128)
    out, lse = call.gpu(device)
    ref, ref_lse = call.oracle()
    assert_parity(out, lse, ref, ref_lse)
    assert not out[1].any() and torch.isneginf(lse[:, 1]).all()
    call = Call([1, 30, 0, 2], [40, 30, 17, 17], 16, 16, 8, 2, 128)
    call.q = torch.cat([call.q, torch.randn(3, 8, 128).to(torch.bfloat16)])
    mine = torch.full((36, 8, 128), 7.0, dtype=torch.bfloat16, device=device)
    out, _ = call.gpu(device, out=mine)
    assert out is mine and (mine[33:] == 7).all()
    ref, _ = call.oracle()
    assert ((mine[:33].cpu().double() - ref[:33]).abs() <= OUT_BAR[torch.bfloat16]).all()


def test_strided_caches(device):
    """Heads outside the pages' rows, scales likewise; caches as halves of one allocation."""
    swap = lambda t: t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype)  # noqa: E731
    halves = lambda t: torch.stack([t.view(torch.uint8)] * 2, 1).view(t.dtype)[:, 0]  # noqa: E731
    for dim, rows in ((128, 1), (64, 1), (128, 4), (128, 50), (256, 50)):
        call = Call([rows, 1], [200, 90], 64, 16, 8, 4, dim)
        want, _ = call.check(device)
        for move in (swap, halves):
            got, _ = call.check(device, move=move)
            assert got.shape == want.shape


def test_capacity_far_above_the_lengths(device):
    """max_seqlen_k as the capacity of the table: the same values."""
    for rows in (1, 4, 60):
        call = Call([rows, 1], [200, 90], 16, 16, 8, 2, 128)
        call.table = torch.nn.functional.pad(call.table, (0, 2048 - call.table.shape[1]), value=-1)
        call.check(device, max_k=2048 * 16)


def test_batch_invariance(device):
    """With num_splits=1 a request's rows do not depend on its neighbours."""
    for dim in (64, 128):
        call = Call([1, 40, 1, 7], [300, 200, 900, 7], 64, 32, 8, 2, dim)
        out, lse = call.gpu(device, num_splits=1)
        for b in range(4):
            alone = Call([1], [1], 64, 32, 8, 2, dim)
            alone.k, alone.v, alone.ks, alone.vs = call.k, call.v, call.ks, call.vs
            alone.q = call.q[call.cu[b]:call.cu[b + 1]]
            alone.new, alone.lengths = [call.new[b]], [call.lengths[b]]
            alone.cu, alone.used, alone.table = offsets(alone.new), call.used[b:b + 1], call.table[b:b + 1]
            got, got_lse = alone.gpu(device, num_splits=1)
            assert torch.equal(got, out[call.cu[b]:call.cu[b + 1]]) and torch.equal(got_lse, lse[:, call.cu[b]:call.cu[b + 1]])


def test_cache_past_32_bit_offsets(device):
    """The last pages of a cache of more than 2^32 elements."""
    page, heads, dim = 256, 8, 128
    pages = 2 ** 32 // (page * heads * dim) + 3
    call = Call([1, 30], [300, 200], page, 16, 16, heads, dim, spare=0)
    cache = [torch.zeros(pages, page, heads, dim, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros(pages, 16, heads, dtype=torch.uint8, device=device) for _ in range(2)]
    for big, small in zip((*cache, *scales), (call.k, call.v, call.ks, call.vs)):
        big[-3:] = small.view(torch.uint8).to(device)
    table = (call.table + pages - 3).to(device)
    for max_q, rows in ((30, slice(None)), (1, slice(0, 1))):
        n = 2 if max_q > 1 else 1
        out = vllm.flash_attn_varlen_func(
            call.q[rows].to(device), cache[0].view(CODE), cache[1].view(CODE), max_q, call.cu[:n + 1].to(device), 300,
            seqused_k=call.used[:n].to(device), block_table=table[:n], causal=True, k_descale=scales[0].view(SCALE),
            v_descale=scales[1].view(SCALE))
        ref, _ = call.oracle()
        assert ((out.cpu().double() - ref[rows]).abs() <= OUT_BAR[torch.bfloat16]).all()


def test_replayed_graph_and_second_stream(device):
    """Captured, replayed with eager calls between, and on another stream: the eager result every time."""
    for rows in (1, 4, 60):
        call = Call([rows, 1], [200, 2000], 64, 32, 8, 2, 128)
        want, want_lse = call.gpu(device)
        to = lambda t: t.to(device)  # noqa: E731
        held = [to(t) for t in (call.q, call.k, call.v, call.cu, call.used, call.table, call.ks, call.vs)]

        def step():
            q, k, v, cu, used, table, ks, vs = held
            return vllm.flash_attn_varlen_func(q, k, v, rows if rows > 1 else 1, cu, 2000, seqused_k=used, block_table=table, causal=True,
                                               k_descale=ks, v_descale=vs, return_softmax_lse=True)

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            out, lse = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = step()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
            call.gpu(device)


def test_append_then_attend(device):
    """The operators together, as a serving step: a prompt is appended with its rotation and attended to, then tokens one
    by one, against dense attention in 64 bits over the rows that the cache holds."""
    import flash_attn_mps_amd as fa
    from block_cache import rotate
    heads, hq, dim, page, block = 2, 8, 64, 32, 16
    g = torch.Generator().manual_seed(3)
    total, prompt = 80, 70
    q, k, v = (torch.randn(total, h, dim, generator=g).to(torch.bfloat16) for h in (hq, heads, heads))
    angle = torch.arange(total, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    cos, sin = angle.cos().float(), angle.sin().float()
    table = torch.tensor([[4, 1, 0]], dtype=torch.int32, device=device)
    caches = [torch.zeros(5, page, heads, dim, dtype=torch.uint8, device=device).view(CODE) for _ in range(2)]
    scales = [torch.zeros(5, page // block, heads, dtype=torch.uint8, device=device).view(SCALE) for _ in range(2)]
    turned = rotate(q, cos, sin, torch.arange(total)[None], None, False)
    at = 0
    while at < total:
        n = prompt if at == 0 else 1
        cu, used = torch.tensor([0, n], dtype=torch.int32, device=device), torch.tensor([at + n], dtype=torch.int32, device=device)
        rows = slice(at, at + n)
        qr = fa.append_paged_kvcache(k[rows].to(device), v[rows].to(device), *caches, cu, used, table, q=q[rows].to(device),
                                     rotary_cos=cos.to(device), rotary_sin=sin.to(device), rotary_interleaved=False,
                                     k_scale=scales[0], v_scale=scales[1])
        out = vllm.flash_attn_varlen_func(qr, *caches, n, cu, at + n, seqused_k=used, block_table=table, causal=True,
                                          k_descale=scales[0], v_descale=scales[1])
        held = [values(c, s)[table[0].cpu().long()].flatten(0, 1)[:at + n] for c, s in zip(caches, scales)]
        ref, _ = oracle_attention(qr.cpu(), *held, torch.tensor([0, n], dtype=torch.int32),
                                  cu_k=torch.tensor([0, at + n], dtype=torch.int32), causal=True)
        assert ((out.cpu().double() - ref).abs() <= OUT_BAR[torch.bfloat16]).all()
        assert ((qr.cpu().double() - turned[rows]).abs() <= 2.0 ** -8 * turned[rows].abs() + 2.0 ** -20).all()
        # The cache against the rows themselves: half an E4M3 step of each value, or of the block's smallest step.
        for x, c in ((rotate(k[:at + n], cos, sin, torch.arange(at + n)[None], None, False), held[0]), (v[:at + n].double(), held[1])):
            bar = x.abs() * 2.0 ** -4 + x.abs().max() * 2.0 ** -17
            assert ((c - x).abs() <= 2 * bar).all()     # coded again: two roundings where the scale grew
        at += n


@pytest.fixture
def wide(monkeypatch):
    """Prefill by way of 16-bit rows whatever the sizes; the entry points that ran."""
    from flash_attn_mps_amd import _attention, _lib
    monkeypatch.setattr(_attention, "_WIDE_ROWS", 0)
    ran, real = [], _lib.call
    monkeypatch.setattr(_lib, "call", lambda name, *a: (ran.append(name), real(name, *a))[1])
    return ran


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim,dim_v", [(4, 4, 64, 64), (8, 2, 128, 128), (3, 1, 256, 256), (4, 2, 80, 80), (4, 2, 32, 32),
                                              (2, 1, 72, 72), (6, 2, 96, 96), (4, 2, 192, 128)])
def test_wide_prefill(device, wide, hq, hkv, dim, dim_v, dtype):
    new, lengths = [130, 1, 64, 257, 33, 0, 18], [130, 1, 200, 257, 1000, 40, 300]
    for causal in (True, False):
        Call(new, lengths, 64, 16, hq, hkv, dim, dtype, dim_v).check(device, causal=causal)
    Call([40, 20], [90, 300], 48, 8, hq, hkv, dim, dtype, dim_v).check(device)      # odd pages, blocks of 8
    assert wide.count("fa_block_wide_fwd") == 3


@pytest.mark.parametrize("dim", [64, 128, 256, 96])
@pytest.mark.parametrize("name", [n for n in FEATURES if n != "splits"])
def test_wide_features(device, wide, name, dim):
    for new, lengths in (([90, 3, 1], [300, 50, 700]), ([600, 40], [900, 1500])):
        call = Call(new, lengths, 64, 32, 8, 2, dim)
        call.check(device, **FEATURES[name])
        call.check(device, s_aux=torch.linspace(-2, 2, 8), **FEATURES[name])
    assert ("fa_block_wide_fwd" in wide) == (name != "one split")


def test_wide_masks_and_biases(device, wide):
    for dim in (64, 128, 256):
        call = Call([60, 40], [300, 170], 64, 32, 4, 2, dim)
        lo = torch.randint(-1, 100, (100,), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
        ranges = torch.stack([lo, lo + 40], 1)
        prefix, window = torch.tensor([20, 3], dtype=torch.int32), torch.tensor([50], dtype=torch.int32)
        for softcap in (0.0, 5.0):
            call.check(device, mask_mod=vllm.mm_prefix_mask(64), aux_tensors=[ranges, call.cu], softcap=softcap)
            call.check(device, mask_mod=vllm.rswa_mask(), aux_tensors=[prefix, window], softcap=softcap)
        call.check(device, dynamic_causal=torch.tensor([True, False]))
        call.check(device, alibi_slopes=torch.rand(4, generator=torch.Generator().manual_seed(10)))
    assert not {"fa_block_prefill_fwd", "fa_block_attn_fwd"} & set(wide)   # (single-row requests may decode)


@pytest.mark.parametrize("low,spread,dtype", [(-40, 3, torch.bfloat16), (20, 3, torch.bfloat16), (-15, 8, torch.float16), (-60, 60, torch.bfloat16),
                                              (-126, 0, torch.bfloat16)])
def test_wide_scales_of_values(device, wide, low, spread, dtype):
    test_wide_scales(device, 70, low, spread, dtype)


def test_wide_not_finite(device, wide):
    """As test_nan_reaches_the_rows_that_see_it, and fp16 queries over values past fp16's range."""
    test_nan_reaches_the_rows_that_see_it(device, 60)
    for row in (0, 17):
        call = Call([64, 40], [128, 90], 64, 16, 8, 4, 128)
        want, _ = call.gpu(device)
        page = int(call.table[0, 1])
        call.v.view(torch.uint8)[page, row, 1, 5] = 0xff     # seen by the rows from position 64 + row on
        out, _ = call.gpu(device)
        assert out[row:64, 2:4, 5].isnan().all()
        out[row:64, 2:4] = want[row:64, 2:4]
        assert ((out - want).abs() <= OUT_BAR[torch.bfloat16]).all()
    call = Call([50], [90], 64, 16, 4, 2, 128, torch.float16)
    call.v.view(torch.uint8)[:, ::7, :, 3] = 0x7e            # 448 * 2^8
    call.vs.view(torch.uint8).fill_(127 - 9)
    call.vs.view(torch.uint8)[:, 1].fill_(127 + 8)
    out, _ = call.gpu(device)
    ref, _ = call.oracle()
    small = ref.abs() < 6e4
    assert ((out.cpu().double() - ref).abs() <= 2.0 ** -9 * ref.abs() + 2.0 ** -10 * 4e4)[small].all()
    assert (out.cpu()[~small].abs() >= 5.9e4).all()


def beyond_16_bits(device, rows, dtype):
    """One key, then one value, past the 16-bit type's range.  The key meets a small negative
    query: its score is -0.6, where an infinity in its place would leave it out unseen."""
    byte = 127 + (10 if dtype == torch.float16 else 120)     # 448 * 2^10 = 458752; 448 * 2^120 = 1.75 * 2^128
    for which in ("k", "v")[dtype == torch.bfloat16:]:
        call = Call([rows, 1], [200, 30], 64, 16, 4, 2, 128, dtype)
        codes, scales = (call.k, call.ks) if which == "k" else (call.v, call.vs)
        page = int(call.table[0, 0])
        codes.view(torch.uint8)[page, 16:32, 1] = 0
        codes.view(torch.uint8)[page, 20, 1, 7] = 0x7e
        scales.view(torch.uint8)[page, 1, 1] = byte
        call.q[:, 2:, 7] = -2.0 ** -16
        call.check(device)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_keys_and_values_beyond_16_bits(device, rows, dtype):
    beyond_16_bits(device, rows, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_keys_and_values_beyond_16_bits(device, wide, dtype):
    beyond_16_bits(device, 70, dtype)
    assert "fa_block_wide_fwd" in wide


def test_wide_layouts_and_replays(device, wide):
    test_strided_caches(device)
    test_empty_requests_and_padding(device)
    test_capacity_far_above_the_lengths(device)
    test_replayed_graph_and_second_stream(device)
    test_cache_past_32_bit_offsets(device)


def test_wide_workspace_has_a_limit(device, wide, monkeypatch):
    """Past the limit the tiles run, or the generic kernel for what they do not take."""
    from flash_attn_mps_amd import _attention
    monkeypatch.setattr(_attention, "_WIDE_BYTES", 1000)
    Call([40], [90], 64, 16, 4, 2, 128).check(device)
    Call([40], [90], 64, 16, 4, 2, 96).check(device)
    assert wide[-1] == "fa_block_attn_fwd" and "fa_block_prefill_fwd" in wide and "fa_block_wide_fwd" not in wide


@pytest.mark.parametrize("dim", [256, 80])
def test_single_rows_that_the_decode_kernel_leaves(device, dim):
    call = Call([1] * 5, [5, 130, 1, 700, 64], 64, 32, 8, 2, dim)
    call.check(device)
    call.check(device, window_size=(40, 0), softcap=5.0)
    call.check(device, s_aux=torch.linspace(-2, 2, 8))


def test_wide_length_past_the_callers_maximum(device, wide):
    """A length past max_seqlen_k: the keys up to it, and the other requests as ever."""
    call = Call([40, 30], [90, 200], 64, 16, 4, 2, 128)
    want, _ = call.gpu(device)
    call.used[1] = 220
    call.table = torch.nn.functional.pad(call.table, (0, 1), value=0)
    out, _ = call.gpu(device, max_k=200)
    assert torch.equal(out[:40], want[:40]) and torch.equal(out[40:], want[40:])


def test_wide_keys_before_every_window_are_not_read(device, wide):
    """Pages and scales that hold NaN before the first row's window change no bit."""
    for dim, rows in ((128, 40), (256, 40), (64, 200)):
        call = Call([rows, rows], [700 + rows, 300 + rows], 64, 16, 8, 2, dim)
        want, want_lse = call.gpu(device, window_size=(77, 0))
        for b, length in enumerate((700, 300)):
            for page in call.table[b, :(length - 77) // 64].tolist():
                for t in (call.k, call.v, call.ks, call.vs):
                    t.view(torch.uint8)[page] = 255
            edge = int(call.table[b, (length - 77) // 64])
            for t in (call.k, call.v):
                t.view(torch.uint8)[edge, :(length - 77) % 64] = 0x7f
        out, lse = call.gpu(device, window_size=(77, 0))
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("keys", [90, 700, 2000])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_wide_sums_past_fp32(device, wide, dim, keys):
    """Values of one sign up to 2^127 under nearly equal weights: their sum leaves fp32's range, their mean does not."""
    for byte, kw in ((246, {}), (244, dict(softcap=5.0)), (240, dict(window_size=(keys // 2, 0))), (238, dict(causal=False))):
        call = Call([40, 30], [keys, 60], 64, 16, 4, 2, dim)
        call.q = call.q * 2.0 ** -8
        call.v = (call.v.view(torch.uint8) & 0x7f).view(CODE)
        call.vs.view(torch.uint8).fill_(byte)
        call.check(device, **kw)
    assert "fa_block_wide_fwd" in wide


def test_wide_scale_bytes(device, wide):
    test_scale_bytes(device)


@pytest.mark.parametrize("more", [20, 200])
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
def test_wide_length_past_the_callers_maximum_behind_a_window(device, wide, dim, more):
    """As with a length of max_seqlen_k: the rows' places, the keys that they see, and the rows that meet a NaN."""
    for kw in (dict(window_size=(50, 0)), dict(window_size=(9, 0), softcap=5.0)):
        call = Call([40, 30], [90, 400], 64, 16, 4, 2, dim)
        call.v.view(torch.uint8)[int(call.table[1, 5]), 60, 1, 5] = 0x7f    # key 380: rows 10 and on
        want, want_lse = call.gpu(device, **kw)
        call.used[1] = 400 + more
        call.table = torch.nn.functional.pad(call.table, (0, 4), value=0)
        out, lse = call.gpu(device, max_k=400, **kw)
        bits = lambda t: t.view(torch.int16)  # noqa: E731
        assert torch.equal(bits(out), bits(want)) and torch.equal(lse, want_lse)
        assert out[50:60, 2:, 5].isnan().all() and not out[:50].isnan().any() and not out[:, :2].isnan().any()


def test_no_memory_for_a_workspace(device, wide, monkeypatch):
    """The tiles run, or the generic kernel for what they do not take."""
    empty = torch.empty

    def short_of_memory(*size, **kw):
        if kw.get("dtype") == torch.bfloat16 and isinstance(size[0], int):
            raise torch.OutOfMemoryError("out of memory")
        return empty(*size, **kw)

    monkeypatch.setattr(torch, "empty", short_of_memory)
    Call([40, 1], [90, 300], 64, 16, 4, 2, 128).check(device)
    Call([40, 1], [90, 300], 64, 16, 4, 2, 96).check(device)
    assert wide[-1] == "fa_block_attn_fwd" and "fa_block_prefill_fwd" in wide and "fa_block_wide_fwd" not in wide


@pytest.mark.parametrize("lengths", [[128, 90], [2100, 1500]])
@pytest.mark.parametrize("dim", [128, 256, 80])
def test_wide_not_finite_beside_features(device, wide, dim, lengths):
    """A NaN in a key, then in a value, of one KV head, with softcap, windows and (long keys) key splits: the rows that
    see it, their heads, the value's dim alone; all else at the bar of the same call without it.  Not bit for bit, as in
    test_nan_reaches_the_rows_that_see_it."""
    rows, at = 64, lengths[0] - 64 + 17          # row 17's own key
    for kw in ({}, dict(softcap=5.0), dict(window_size=(30, 0)), dict(softcap=5.0, window_size=(30, 0)), dict(causal=False)):
        sees = torch.arange(rows) >= (0 if kw.get("causal") is False else 17)
        if "window_size" in kw:
            sees &= torch.arange(rows) <= 17 + 30
        base = Call([rows, 40], lengths, 64, 16, 8, 4, dim)
        want, want_lse = base.gpu(device, **kw)
        for which in ("k", "v"):
            call = Call([rows, 40], lengths, 64, 16, 8, 4, dim)
            getattr(call, which).view(torch.uint8)[int(call.table[0, at // 64]), at % 64, 1, 5] = 0xff
            out, lse = call.gpu(device, **kw)
            nan = torch.zeros(rows + 40, 8, dim, dtype=torch.bool)
            nan[:rows, 2:4][sees] = True
            if which == "v":
                nan[..., :5] = nan[..., 6:] = False
            assert torch.equal(out.isnan().cpu(), nan)
            keep = ~nan
            assert ((out.cpu() - want.cpu()).abs() <= OUT_BAR[torch.bfloat16])[keep].all()
            clean = ~nan.any(-1).T if which == "k" else torch.ones(8, rows + 40, dtype=torch.bool)
            assert ((lse.cpu() - want_lse.cpu()).abs() <= 1e-4)[clean].all() and torch.isneginf(lse.cpu()[~clean]).all()
    assert "fa_block_wide_fwd" in wide


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("lengths", [[200, 90], [1800, 1200]])
def test_wide_beyond_16_bits_beside_features(device, wide, dim, lengths):
    """Keys and values past the 16-bit type's range with softcap, windows and key splits: as beyond_16_bits."""
    for dtype in (torch.float16, torch.bfloat16):
        byte = 127 + (10 if dtype == torch.float16 else 120)
        for kw in ({}, dict(softcap=5.0), dict(softcap=5.0, window_size=(180, 0))):
            for which in ("k", "v")[dtype == torch.bfloat16:]:
                call = Call([70, 30], lengths, 64, 16, 4, 2, dim, dtype)
                codes, scales = (call.k, call.ks) if which == "k" else (call.v, call.vs)
                page, block = int(call.table[0, (lengths[0] - 60) // 64]), (lengths[0] - 60) % 64 // 16
                codes.view(torch.uint8)[page, 16 * block:16 * block + 16, 1] = 0
                codes.view(torch.uint8)[page, 16 * block + 4, 1, 7] = 0x7e
                scales.view(torch.uint8)[page, block, 1] = byte
                call.q[:, 2:, 7] = -2.0 ** -16
                call.check(device, **kw)
    assert "fa_block_wide_fwd" in wide


def scales_apart(device, rows, low, spread, dtype, dim, **kw):
    """As test_wide_scales, each output held to its own sum p |v|: rows, heads and dims of small blocks too.  Beside that
    only the types' smallest steps: 2^-24 in fp16 (values and outputs, half a step each), 2^-132 in bf16."""
    call = Call([rows, 3], [200, 90], 64, 16, 4, 2, dim, dtype)
    _, call.vs = random_cache(call.v.shape[0], 64, 16, 2, dim, 77, low, spread)
    out, lse = call.gpu(device, **kw)
    ref, ref_lse = call.oracle(**kw)
    call.v = (call.v.view(torch.uint8) & 0x7f).view(CODE)
    bar = 2 * HALF_STEP[dtype] * call.oracle(**kw)[0] * (1 + 2.0 ** -5) + (2.0 ** -24 if dtype == torch.float16 else 2.0 ** -132)
    off = (out.cpu().double() - ref).abs()
    assert (off <= bar).all(), f"off by up to {(off / bar).max():.3f} of the tolerance"
    assert ((lse.cpu().double() - ref_lse).abs().max() <= 1e-4).item()


APART = [(-40, 3, torch.bfloat16), (20, 3, torch.bfloat16), (-15, 8, torch.float16), (-60, 60, torch.bfloat16)]


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("low,spread,dtype", APART)
def test_scales_apart(device, rows, low, spread, dtype):
    scales_apart(device, rows, low, spread, dtype, 128)
    scales_apart(device, rows, low, spread, dtype, 64, window_size=(20, 0))


@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("low,spread,dtype", APART)
def test_wide_scales_apart(device, wide, low, spread, dtype, dim):
    scales_apart(device, 70, low, spread, dtype, dim)
    scales_apart(device, 70, low, spread, dtype, dim, window_size=(20, 0))
    scales_apart(device, 70, low, spread, dtype, dim, window_size=(0, 0))
    assert "fa_block_wide_fwd" in wide
