"""The operators of a block-scaled 8-bit KV cache that this library is measured
on: rotary positions of one to several axes, the append of keys and values to a
paged cache with that rotation on the way, and attention that reads the cache.

A block-scaled cache holds E4M3 codes [pages, page_size, Hkv, D] and one power
of two (E8M0) for each block of `block` tokens and head, [pages, page_size /
block, Hkv]: a value is code * scale.  An append gives a block the smallest
scale >= 2^-100 under which its largest new magnitude is at most 448; a block
that already holds rows of the request keeps the larger of that and its old
scale, and its rows are coded again when it grows.

A case names an operator (`kind`), its sizes, and `shape`: the seed of its
request lengths, so that a case's work does not depend on its input values.
Head counts, head dims, page sizes and lengths are those of this repository's
benchmark and configurations, or generic.
"""
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "block": 1}
CODE, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
DEVICE = "cuda"


def _library():
    path = os.path.abspath("flash-attn-mps_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_attn_mps_amd as fa
    from flash_attn_mps_amd import vllm
    return fa, vllm


# ------------------------------------------------------------ cases

def listed():
    return [
        # Rotary positions alone.  One token of a text and image model: latency and launches.
        dict(name="rope_step", kind="rope", tokens=1, hq=32, hkv=8, dim=128, rot=128, axes="16,24,24", split=True,
             interleaved=False, dtype="fp16", shape=1),
        # The patches of a few images in an encoder: two axes (row, column), q and k views of one packed
        # projection, 80-dim heads.
        dict(name="rope_image", kind="rope", tokens=9001, hq=16, hkv=16, dim=80, rot=80, axes="20,20", split=False,
             interleaved=False, dtype="bf16", shape=2),
        # The append.  One token of one chat.
        dict(name="append_b1", kind="append", batch=1, new=1, lo=700, hi=700, hq=16, hkv=8, dim=128, rot=128, axes="64",
             interleaved=False, dtype="fp16", cache="block", page=256, block=64, shape=3),
        # A decode step of a loaded server, long contexts in 16-token pages.
        dict(name="append_b64", kind="append", batch=64, new=1, lo=512, hi=32768, hq=32, hkv=8, dim=128, rot=128,
             axes="16,24,24", interleaved=False, dtype="bf16", cache="block", page=16, block=16, shape=4),
        # A whole prefill batch, 36K tokens: the bytes of q, k, v and the cache.
        dict(name="append_prefill", kind="append", batch=16, new=0, lo=256, hi=4096, hq=16, hkv=8, dim=128, rot=128,
             axes="64", interleaved=False, dtype="bf16", cache="block", page=64, block=32, shape=5),
        # Chunks of long prompts into a 16-bit cache: half of each head rotates, pairs next to each other.
        dict(name="append_16bit", kind="append", batch=3, new=1365, lo=100, hi=9000, hq=16, hkv=4, dim=256, rot=128,
             axes="64", interleaved=True, dtype="fp16", cache="fp16", page=64, block=0, shape=6),
        # Attention over the cache.  One token of one chat: latency.
        dict(name="decode_b1", kind="attend", batch=1, rows=1, lo=700, hi=700, hq=16, hkv=8, dim=128, dtype="fp16",
             page=256, block=64, window=-1, softcap=0.0, sinks=False, shape=3),
        # A decode step of a loaded server: 1M keys, 2.2 GB of cache.
        dict(name="decode_b64", kind="attend", batch=64, rows=1, lo=512, hi=32768, hq=32, hkv=8, dim=128, dtype="bf16",
             page=16, block=16, window=-1, softcap=0.0, sinks=False, shape=4),
        # Four drafted rows a request, 64-dim heads in large groups, sinks and a window.
        dict(name="decode_rows4", kind="attend", batch=32, rows=4, lo=300, hi=12000, hq=64, hkv=8, dim=64, dtype="bf16",
             page=64, block=32, window=4095, softcap=0.0, sinks=True, shape=7),
        # Prompts from their first token.
        dict(name="prefill_b16", kind="attend", batch=16, rows=0, lo=256, hi=4096, hq=16, hkv=8, dim=128, dtype="bf16",
             page=64, block=32, window=-1, softcap=0.0, sinks=False, shape=5),
        # Chunks of 512 rows behind long prefixes.
        dict(name="chunk_long", kind="attend", batch=2, rows=512, lo=9001, hi=24000, hq=32, hkv=8, dim=128, dtype="bf16",
             page=16, block=16, window=-1, softcap=0.0, sinks=False, shape=8),
        # 256-dim heads, softcap, a local window.
        dict(name="prefill_d256", kind="attend", batch=8, rows=0, lo=100, hi=3000, hq=16, hkv=8, dim=256, dtype="fp16",
             page=64, block=16, window=1023, softcap=50.0, sinks=False, shape=9),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """A case of the same ranges that costs no more than the largest listed ones."""
    while True:
        case = _draw(rng)
        cost = work(case)
        if cost["bytes"] < 2e9 and cost["flops"] < 5e11:
            return case


def _draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend"])
    dim = rng.choice([64, 80, 128, 128, 256]) if kind != "attend" else rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    case = dict(kind=kind, hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv, dim=dim, dtype=rng.choice(["fp16", "bf16"]),
                shape=rng.randrange(1 << 20))
    if kind != "attend":
        half = rng.choice([dim // 2, dim // 4])
        count = rng.choice([1, 1, 2, 3])
        first = half // count
        case.update(rot=2 * half, axes=",".join(str(n) for n in [half - first * (count - 1)] + [first] * (count - 1)),
                    interleaved=rng.random() < 0.5)
    if kind == "rope":
        return dict(case, tokens=_log_uniform(rng, 1, 9000), split=rng.random() < 0.5)
    page = rng.choice([16, 64, 256])
    case.update(page=page, block=rng.choice([n for n in (16, 32, 64) if n <= page]))
    if kind == "append":
        case["cache"] = rng.choice(["block", "block", "block", case["dtype"]])
        if rng.random() < 0.5:      # a few new tokens a request
            case.update(batch=_log_uniform(rng, 1, 64), new=rng.choice([1, 1, 1, 2, 5]), lo=1, hi=_log_uniform(rng, 16, 8192))
        else:
            case.update(batch=rng.randint(1, 8), new=0, lo=1, hi=_log_uniform(rng, 16, 4096))
        return case
    case.update(window=rng.choice([-1, -1, -1, _log_uniform(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0]),
                sinks=rng.random() < 0.3)
    form = rng.random()
    if form < 0.5:
        case.update(batch=_log_uniform(rng, 1, 128), rows=rng.choice([1, 1, 1, 2, 5]), lo=1, hi=_log_uniform(rng, 16, 16384))
    elif form < 0.75:
        case.update(batch=rng.randint(1, 8), rows=0, lo=1, hi=_log_uniform(rng, 16, 4096))
    else:
        case.update(batch=rng.randint(1, 4), rows=_log_uniform(rng, 17, 512), lo=1, hi=_log_uniform(rng, 16, 16384))
    return case


def _requests(case):
    """(new rows, keys after them) of each request."""
    rng = random.Random(case["shape"])
    lengths = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    new = case["new"] if case["kind"] == "append" else case["rows"]
    return ([new] * len(lengths), [n + new for n in lengths]) if new else (lengths, lengths)


# ------------------------------------------------------------ inputs

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cu(lengths):
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=DEVICE), _i32(lengths).cumsum(0, dtype=torch.int32)])


def _codes(g, shape):
    """E4M3 codes of blocks whose largest magnitude is near 448: 112 N(0, 1)."""
    out = torch.empty(shape, dtype=CODE, device=DEVICE)
    flat, step = out.flatten(0, 1), 1 << 17
    for i in range(0, flat.shape[0], step):     # in pieces: the fp32 draw is four times the result
        part = flat[i:i + step]
        part.copy_(torch.randn(part.shape, generator=g, device=DEVICE).mul_(112).clamp_(-448, 448))
    return out


def _scales(g, shape, low):
    """2^low .. 2^(low + 2): blocks of one head differ."""
    return torch.randint(127 + low, 130 + low, shape, generator=g, device=DEVICE, dtype=torch.uint8).view(SCALE)


def _trig(rot, positions, dtype):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * inv
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _pair_axes(case):
    """The axis of each rotated pair: sections of consecutive pairs."""
    return tuple(a for a, n in enumerate(case["axes"].split(",")) for _ in range(int(n)))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, hq, hkv, dim, dtype = case["kind"], case["hq"], case["hkv"], case["dim"], DTYPES[case["dtype"]]
    s = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)

    if kind == "rope":
        tokens, axes = case["tokens"], case["axes"].count(",") + 1
        if case["split"]:
            s["q"], s["k"] = normal(tokens, hq, dim), normal(tokens, hkv, dim)
        else:       # views of one projection, as a packed layer hands them on
            s["q"], s["k"], _ = normal(tokens, hq + 2 * hkv, dim).split([hq, hkv, hkv], 1)
        s["cos"], s["sin"] = _trig(case["rot"], 4096, torch.float32)
        s["positions"] = torch.randint(0, 4096, (axes, tokens), generator=g, device=DEVICE)
        s["pair_axes"] = _pair_axes(case)
        return s

    rows, lengths = _requests(case)
    tokens, page, block = sum(rows), case["page"], case["block"]
    need = [-(-n // page) for n in lengths]
    pool, width = sum(need), max(need)
    perm = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    start, count = _cu(need)[:-1].long(), _i32(need)
    column = torch.arange(width, device=DEVICE)
    s["table"] = torch.where(column < count[:, None], perm[(start[:, None] + column).clamp_(max=pool - 1)], 0)
    s.update(cu=_cu(rows), lengths=_i32(lengths), max_q=max(rows), max_k=max(lengths))
    s["q"] = normal(tokens, hq, dim)
    cache = (pool, page, hkv, dim)
    if case.get("cache", "block") == "block":
        s["k_cache"], s["v_cache"] = _codes(g, cache), _codes(g, cache)
        s["k_scale"] = _scales(g, (pool, page // block, hkv), -8)
        s["v_scale"] = _scales(g, (pool, page // block, hkv), -9)
    else:
        s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = normal(*cache), normal(*cache), None, None
    if kind == "append":
        s["k"], s["v"] = normal(tokens, hkv, dim), normal(tokens, hkv, dim)
        s["cos"], s["sin"] = _trig(case["rot"], s["max_k"], torch.float32)
        axes = case["axes"].count(",") + 1
        s["pair_axes"] = _pair_axes(case) if axes > 1 else None
        # Several axes: the tokens of an image share positions, so they lie behind the cache's.
        s["positions"] = torch.randint(0, s["max_k"], (axes, tokens), generator=g, device=DEVICE) if axes > 1 else None
        return s
    s["sinks"] = torch.randn(hq, generator=g, device=DEVICE) if case["sinks"] else None
    s["out"] = torch.empty(tokens, hq, dim, dtype=dtype, device=DEVICE)
    return s


# ------------------------------------------------------------ the plain forms

def _rotate(x, cos, sin, positions, pair_axes, interleaved):
    """x [T, H, D] with pair i of each head turned by the angle of positions[pair_axes[i]] (fp32)."""
    half = cos.shape[1]
    axis = torch.tensor(pair_axes, device=x.device)
    at, pair = positions[axis].T, torch.arange(half, device=x.device)
    c, s = cos[at, pair].float()[:, None], sin[at, pair].float()[:, None]
    x = x.float()
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, rest], -1)


def _values_of(scale):
    return torch.exp2(scale.view(torch.uint8).float() - 127)


def _append_block(x, cache, scale, where, first, old, kept):
    """x [T, H, D] (fp32) into block-scaled `cache` at (page, row) = where; first: the (page, row)
    at which each request's first new row lies, `old` rows of whose block it keeps."""
    page, row = where
    page_size, per = cache.shape[1], scale.shape[1]
    block = page_size // per
    slot, first_slot = page * per + row // block, first[0] * per + first[1] // block
    heads = x.shape[1]
    most = torch.zeros(cache.shape[0] * per, heads, device=x.device).index_reduce_(0, slot, x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
    exponent = torch.where(most > 0, exponent, -100).clamp_(min=-100)
    flat = scale.view(torch.uint8).flatten(0, 1)
    before = flat[first_slot].int() - 127
    exponent[first_slot] = torch.where(kept[:, None], torch.maximum(exponent[first_slot], before), exponent[first_slot])
    # The rows that the first blocks keep, under their new scale.
    rows = torch.arange(block, device=x.device)
    at = (first_slot // per)[:, None], (first_slot % per * block)[:, None] + rows
    codes = cache[at]
    again = (codes.float() * torch.exp2((before - exponent[first_slot]).float())[:, None, :, None]).to(CODE)
    stays = (rows < old[:, None])[:, :, None, None]
    cache[at] = torch.where(stays, again.float(), codes.float()).to(CODE)
    flat[slot] = (exponent[slot] + 127).to(torch.uint8)
    cache[page, row] = (x * torch.exp2(-exponent[slot].float())[..., None]).clamp_(-448, 448).to(CODE)


def _append(s):
    case = s["case"]
    cu, lengths, page_size = s["cu"].long(), s["lengths"].long(), s["k_cache"].shape[1]
    new = cu[1:] - cu[:-1]
    token = torch.arange(s["k"].shape[0], device=cu.device)
    request = torch.searchsorted(cu[1:], token, right=True)
    position = (lengths - new)[request] + token - cu[request]
    where = s["table"][request, position // page_size].long(), position % page_size
    turn = position[None] if s["positions"] is None else s["positions"]
    axes = s["pair_axes"] or (0,) * s["cos"].shape[1]
    q, k = (_rotate(x, s["cos"], s["sin"], turn, axes, case["interleaved"]) for x in (s["q"], s["k"]))
    v = s["v"].float()
    if s["k_scale"] is None:
        s["k_cache"][where], s["v_cache"][where] = k.to(s["k_cache"].dtype), v.to(s["v_cache"].dtype)
        return q.to(s["q"].dtype), s["k_cache"], s["v_cache"]
    before = lengths - new
    old = before % case["block"]
    first = s["table"].gather(1, (before // page_size)[:, None])[:, 0].long(), before % page_size
    _append_block(k, s["k_cache"], s["k_scale"], where, first, old, old > 0)
    _append_block(v, s["v_cache"], s["v_scale"], where, first, old, old > 0)
    return q.to(s["q"].dtype), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _gathered(cache, scale, table):
    """The values of each request's pages, [B, Hkv, keys, D] in fp32."""
    value = cache[table.long()].float()                                     # [B, W, P, H, D]
    factor = _values_of(scale)[table.long()]                                # [B, W, P / block, H]
    value = value.unflatten(2, (factor.shape[2], -1)).mul_(factor[:, :, :, None, :, None])
    return value.flatten(1, 3).transpose(1, 2)


def _attend(s):
    case = s["case"]
    hkv, rows, group = case["hkv"], s["max_q"], case["hq"] // case["hkv"]
    cu, lengths = s["cu"].long(), s["lengths"].long()
    new, row = cu[1:] - cu[:-1], torch.arange(rows, device=cu.device)
    real = row < new[:, None]                                               # [B, R]
    at = (cu[:-1, None] + row).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = _gathered(s["k_cache"], s["k_scale"], s["table"]), _gathered(s["v_cache"], s["v_scale"], s["table"])
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(case["dim"] ** -0.5)
    if case["softcap"]:
        score = score.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    score = score.unflatten(2, (group, rows))                               # [B, Hkv, group, R, K]
    key, position = torch.arange(k.shape[2], device=cu.device), (lengths - new)[:, None] + row
    seen = key <= position[..., None]
    if case["window"] >= 0:
        seen &= key >= position[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -torch.inf)
    top = score.amax(-1)
    if s["sinks"] is not None:
        sink = s["sinks"].view(hkv, group)[None, :, :, None]
        top = torch.maximum(top, sink)
    weight = score.sub_(top[..., None]).exp_()
    total = weight.sum(-1)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(weight.flatten(2, 3), v).unflatten(2, (group, rows)) / total[..., None]
    out, lse = out.permute(0, 3, 1, 2, 4).flatten(2, 3), (top + total.log()).permute(0, 3, 1, 2).flatten(2, 3)
    return out[real].to(s["q"].dtype), lse[real].T.contiguous()


def run(state):
    s, case = state, state["case"]
    if case["kind"] == "rope":
        if own:
            fa, _ = _library()
            return fa.rotary_embedding(s["q"], s["k"], s["cos"], s["sin"], s["positions"], pair_axes=s["pair_axes"],
                                       rotary_interleaved=case["interleaved"])
        return tuple(_rotate(x, s["cos"], s["sin"], s["positions"], s["pair_axes"], case["interleaved"]).to(x.dtype)
                     for x in (s["q"], s["k"]))
    if case["kind"] == "append":
        # The caches come back as they are held: E4M3 codes and E8M0 scales are both floating types.
        if own:
            fa, _ = _library()
            q = fa.append_paged_kvcache(s["k"], s["v"], s["k_cache"], s["v_cache"], s["cu"], s["lengths"], s["table"],
                                        q=s["q"], rotary_cos=s["cos"], rotary_sin=s["sin"], positions=s["positions"],
                                        pair_axes=s["pair_axes"], rotary_interleaved=case["interleaved"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
            caches = (s["k_cache"], s["v_cache"])
            return (q, *caches) if s["k_scale"] is None else (q, *caches, s["k_scale"], s["v_scale"])
        return _append(s)
    if own:
        _, vllm = _library()
        window = case["window"]
        return vllm.flash_attn_varlen_func(
            s["q"], s["k_cache"], s["v_cache"], s["max_q"], s["cu"], s["max_k"], seqused_k=s["lengths"],
            block_table=s["table"], causal=True, window_size=(window, -1 if window < 0 else 0), softcap=case["softcap"],
            k_descale=s["k_scale"], v_descale=s["v_scale"], s_aux=s["sinks"], out=s["out"], return_softmax_lse=True)
    return _attend(s)


# ------------------------------------------------------------ work, 64-bit result

def work(case):
    hq, hkv, dim, size = case["hq"], case["hkv"], case["dim"], BYTES[case["dtype"]]
    if case["kind"] == "rope":
        heads, tokens, axes = hq + hkv, case["tokens"], case["axes"].count(",") + 1
        trig = min(tokens * axes, 4096) * case["rot"] // 2 * 8
        return {"bytes": 2 * tokens * heads * dim * size + trig + 8 * axes * tokens,
                "flops": 3 * tokens * heads * case["rot"]}
    rows, lengths = _requests(case)
    tokens = sum(rows)
    if case["kind"] == "append":
        axes, cached = case["axes"].count(",") + 1, BYTES[case["cache"]]
        trig = min(tokens * axes, max(lengths)) * case["rot"] // 2 * 8
        blocks = sum(-(-n // case["block"]) for n in rows) if case["block"] else 0
        moved = 2 * tokens * hq * dim * size + 2 * tokens * hkv * dim * (size + cached) + 2 * blocks * hkv
        positions = 8 * axes * tokens if axes > 1 else 0
        return {"bytes": moved + trig + positions + 12 * len(rows), "flops": 3 * tokens * (hq + hkv) * case["rot"]}
    pairs = keys = 0
    for new, length in zip(rows, lengths):
        most = length if case["window"] < 0 else case["window"] + 1
        first = length - new + 1
        full = max(0, min(new, most - first + 1))        # rows that see less than the window
        pairs += full * first + full * (full - 1) // 2 + (new - full) * most
        keys += min(length, most + new - 1)
    moved = 2 * keys * hkv * dim + 2 * -(-keys // case["block"]) * hkv + 2 * tokens * hq * dim * size + 4 * tokens * hq
    return {"bytes": moved, "flops": 4 * pairs * hq * dim}


def _turn64(x, case, s, positions):
    """The rotation as a complex product."""
    half = s["cos"].shape[1]
    axis = list(s["pair_axes"] or [0] * half)
    angle = torch.stack([torch.complex(s["cos"].double(), s["sin"].double())[positions[a], i]
                         for i, a in enumerate(axis)], -1)[:, None]
    y = x.double().clone()
    even = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
    odd = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
    z = torch.complex(y[..., even], y[..., odd]) * angle
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _code64(x):
    """x rounded to the nearest E4M3 value, ties to even, at most 448 in magnitude."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(-6, 8)
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _block64(cache, scale, x, page_of, start, block):
    """Rows x [n, H, D] appended at positions start .. of one request, block by block."""
    size, end = cache.shape[1], start + x.shape[0]
    for begin in range(start // block * block, end, block):
        page, row = int(page_of[begin // size]), begin % size
        lo, hi = max(begin, start), min(begin + block, end)
        part = x[lo - start:hi - start]
        most = part.abs().amax((0, 2))
        power = torch.ceil(torch.log2((most / 448).clamp(min=2.0 ** -200))).clamp(min=-100)
        before = scale[page, row // block]
        if lo > begin:
            now = torch.maximum(torch.exp2(power), before)
            held = cache[page, row:row + lo - begin]
            cache[page, row:row + lo - begin] = _code64(held * (before / now)[:, None])
        else:
            now = torch.exp2(power)
        scale[page, row // block] = now
        cache[page, row + lo - begin:row + hi - begin] = _code64(part / now[:, None])


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return tuple(_turn64(x, case, s, s["positions"]) for x in (s["q"], s["k"]))
    rows, lengths = _requests(case)
    if case["kind"] == "append":
        position = torch.cat([torch.arange(n - new, n, device=DEVICE) for new, n in zip(rows, lengths)])
        turn = position[None] if s["positions"] is None else s["positions"]
        q, k, v = _turn64(s["q"], case, s, turn), _turn64(s["k"], case, s, turn), s["v"].double()
        page, at = case["page"], 0
        block_scaled = s["k_scale"] is not None
        scales = [torch.exp2(x.view(torch.uint8).double() - 127) for x in (s["k_scale"], s["v_scale"])] if block_scaled else []
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        for b, (new, length) in enumerate(zip(rows, lengths)):
            table = s["table"][b].tolist()
            for i, x in enumerate((k[at:at + new], v[at:at + new])):
                if block_scaled:
                    _block64(caches[i], scales[i], x, table, length - new, case["block"])
                    continue
                where = position[at:at + new]
                caches[i][s["table"][b].long()[where // page], where % page] = x
            at += new
        return (q, *caches, *scales)
    hq, hkv, dim, at = case["hq"], case["hkv"], case["dim"], 0
    outs, lses = [], []
    for b, (new, length) in enumerate(zip(rows, lengths)):
        pages = s["table"][b, :-(-length // case["page"])].long()
        k, v = ((s[c][pages].double().unflatten(1, (-1, case["block"]))
                 * torch.exp2(s[f][pages].view(torch.uint8).double() - 127)[:, :, None, :, None]).flatten(0, 2)[:length]
                for c, f in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
        where = torch.arange(length - new, length, device=DEVICE)[:, None]
        key = torch.arange(length, device=DEVICE)
        hidden = (key > where) | ((key < where - case["window"]) if case["window"] >= 0 else torch.zeros_like(key > where))
        out, lse = [], []
        for h in range(hq):
            score = s["q"][at:at + new, h].double() @ k[:, h // (hq // hkv)].T / dim ** 0.5
            if case["softcap"]:
                score = case["softcap"] * torch.tanh(score / case["softcap"])
            score = score.masked_fill(hidden, -torch.inf)
            if s["sinks"] is not None:
                score = torch.cat([score, s["sinks"][h].double().expand(new, 1)], 1)
            lse.append(torch.logsumexp(score, 1))
            weight = torch.exp(score - lse[-1][:, None])[:, :length]
            out.append(weight @ v[:, h // (hq // hkv)])
        outs.append(torch.stack(out, 1))
        lses.append(torch.stack(lse))
        at += new
    return torch.cat(outs), torch.cat(lses, 1)
