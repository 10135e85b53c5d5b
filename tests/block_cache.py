"""A block-scaled cache on the CPU in 64 bits: what append_paged_kvcache leaves and
what attention reads, from their definitions, and inputs for their tests.

E4M3 rounds to nearest by at most half a step: 2^-4 of a value in the normal range
(4 significant bits), 2^-10 of the scale below it.
"""
import torch

CODE, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu


def scale_values(scale):
    """E8M0 scales as float64 (255: NaN)."""
    e = scale.detach().cpu().view(torch.uint8).double()
    return torch.where(e == 255, torch.nan, torch.exp2(e - 127))


def values(cache, scale):
    """The values [pages, P, H, D] of codes and scales, float64."""
    block = cache.shape[1] // scale.shape[1]
    return cache.detach().cpu().double() * scale_values(scale).repeat_interleave(block, 1)[..., None]


def exponent(most):
    """The smallest e >= -100 with most <= 448 * 2^e."""
    e = -100
    while most > 448.0 * 2.0 ** e:
        e += 1
    return e


def encode(x):
    """The nearest E4M3 values of float64 x, ties to even, saturating at 448; NaN is kept."""
    a = x.abs()
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6, max=448.0)))
    step = torch.exp2(e - 3)
    y = (torch.round(a / step) * step).clamp(max=448.0)
    return torch.where(x.isnan(), x, torch.copysign(y, x))


def rotate(x, cos, sin, positions, pair_axes, interleaved):
    """x [T, H, D] float64; positions [axes, T]; NaN where the tables have no row."""
    x, half = x.double().clone(), cos.shape[1]
    for i in range(half):
        p = positions[pair_axes[i] if pair_axes else 0].long()
        ok = (p >= 0) & (p < cos.shape[0])
        at = p.clamp(0, max(cos.shape[0] - 1, 0))
        c, s = (torch.where(ok, t.double()[at, i], torch.nan)[:, None] for t in (cos, sin))
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, w = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x


def rows_of(cu, used, table, page_size, pages, tokens):
    """(token, request, position, page, row) of every row that is written."""
    out = []
    for b in range(len(used)):
        n = int(cu[b + 1]) - int(cu[b])
        for j in range(n):
            p = int(used[b]) - n + j
            if p < 0 or p // page_size >= table.shape[1]:
                continue
            page = int(table[b, p // page_size])
            if 0 <= page < pages:
                out.append((int(cu[b]) + j, b, p, page, p % page_size))
    return out


def append(cache, scale, x, cu, used, table):
    """float64 (values of the codes, scales) of a block-scaled cache after the rows x [T, H, D] (float64) are appended."""
    code, scales = cache.detach().cpu().double().clone(), scale_values(scale)
    size = cache.shape[1]
    block = size // scale.shape[1]
    written = {}
    for t, b, p, page, row in rows_of(cu, used, table, size, cache.shape[0], x.shape[0]):
        written.setdefault((page, row // block, b), []).append((t, p, row))
    for (page, j, b), rows in written.items():
        first = min(row for _, _, row in rows)
        kept = first - j * block
        for h in range(x.shape[1]):
            new = torch.stack([x[t, h] for t, _, _ in rows])
            finite = new[new.isfinite()]
            s = 2.0 ** exponent(float(finite.abs().max()) if finite.numel() else 0.0)
            if kept:
                old = float(scales[page, j, h])
                s = s if s > old else old
                part = slice(j * block, j * block + kept)
                code[page, part, h] = encode(code[page, part, h] * (old / s)) if s != old else code[page, part, h]
            scales[page, j, h] = s
            for (_, _, row), values_ in zip(rows, new):
                code[page, row, h] = encode(values_ / s)
    return code, scales


def pages_for(lengths, page, seed, spare=2):
    """(block table [B, width] int32 over a shuffled pool, pages in the pool); unused entries are -1."""
    need = [-(-n // page) for n in lengths]
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max([*need, 1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(need) + spare


def random_cache(pages, page, block, heads, dim, seed, low=-9, spread=4):
    """Codes of any finite magnitude, and scales 2^low .. 2^(low + spread)."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(pages, page, heads, dim, generator=g) * 100).clamp(-448, 448).to(CODE)
    e = torch.randint(127 + low, 127 + low + spread + 1, (pages, page // block, heads), generator=g)
    return codes, e.to(torch.uint8).view(SCALE)


def offsets(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32)
