"""Plain 64-bit forms of the quantised key/value cache, for the tests: written from the formulas, token by token or head by
head, on any device."""
import math

import torch


def rotate64(x, cos_sin, positions, interleaved):
    """x [n, h, d] fp64; the first cos_sin.shape[1] channels turn by row positions[n]."""
    rot = cos_sin.shape[1]
    out = x.clone()
    half = rot // 2
    t = cos_sin.double()[positions.long()]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = t[:, i, None], t[:, half + i, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def norm64(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def _rows_of(cache, page_table, b, count):
    """(pages, places, there) of the first `count` tokens of sequence b."""
    p = torch.arange(count, device=page_table.device)
    col = p // cache.page_size
    inside = col < page_table.shape[1]
    page = page_table[b].long()[col.clamp(max=max(page_table.shape[1] - 1, 0))]
    there = inside & (page >= 0) & (page < cache.num_pages)
    return torch.where(there, page, 0), p % cache.page_size, there


def held64(cache, which, page_table, b, count):
    """[count, heads, d] fp64: what the cache holds of the first `count` tokens of sequence b (missing pages: NaN)."""
    codes = getattr(cache, which + "_codes")
    if count == 0:
        return torch.empty((0, cache.n_kv_heads, cache.head_dim), dtype=torch.float64, device=codes.device)
    page, place, there = _rows_of(cache, page_table, b, count)
    c, s = codes[page, :, place], getattr(cache, which + "_scales")[page, :, place].double()[..., None]
    if cache.kv_format == "fp8":
        x = c.view(torch.float8_e4m3fn).double()
    elif cache.kv_format == "int8":
        x = c.view(torch.int8).double()
    else:
        x = torch.stack([c % 16, c // 16], -1).flatten(-2).double() - getattr(cache, which + "_zeros")[page, :, place].double()[..., None]
    return torch.where(there[:, None, None], x * s, math.nan)


def scales64(cache, which, page_table, b, count):
    """[count, heads] fp64: the scales of the first `count` tokens of sequence b (missing pages: NaN)."""
    s = getattr(cache, which + "_scales")
    if count == 0:
        return torch.empty((0, cache.n_kv_heads), dtype=torch.float64, device=s.device)
    page, place, there = _rows_of(cache, page_table, b, count)
    return torch.where(there[:, None], s[page, :, place].double(), math.nan)


def score_slack64(q, k, sees, scale):
    """[t, h]: what rounding the keys to fp16 (unit 2^-11, a product's error uniform in it: 2^-11 / sqrt 3 of the product) may add
    to a score: 6 sigma of a row's worst seen token."""
    g = q.shape[1] // k.shape[1]
    k = torch.where(sees.any(0)[:, None, None], k, 0.0)
    out = [((q[:, h].double() ** 2) @ (k[:, h // g] ** 2).T * sees).amax(1).sqrt() for h in range(q.shape[1])]
    return torch.stack(out, 1) * abs(scale) * 2.0 ** -11 * 6 / math.sqrt(3)


def attend64(q, k, v, sees, scale, v_scales=None):
    """q [t, h, d], k / v [l, hkv, d] fp64, sees bool [t, l] -> (result [t, h, d], sum of p |v| [t, h, d]); zeros where a row sees
    nothing.  Tokens that no row may see can hold anything.

    With v_scales [l, hkv], the sum also counts what the smallest weights may lose.  The weights of the codes v / scale are
    p * scale; as fp16 numbers with the largest at 2^15 at most (2^14 at least, the maximum being known to a fp32 rounding)
    they are off by up to half of fp16's smallest step, 2^-25: 2^-39 of the largest weight, times the token's |code|.  It is
    counted as 2^9.5 times that, because the caller multiplies the whole sum by 2^-9.5."""
    g = q.shape[1] // k.shape[1]
    any_row = sees.any(0)
    k, v = torch.where(any_row[:, None, None], k, 0.0), torch.where(any_row[:, None, None], v, 0.0)
    if v_scales is not None:
        v_scales = torch.where(any_row[:, None], v_scales, 1.0)
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    empty = ~sees.any(1)
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ k[:, h // g].T * scale).masked_fill(~sees, -math.inf)
        s[empty] = 0.0
        p = torch.softmax(s, -1) * sees
        out[:, h], size[:, h] = p @ v[:, h // g], p @ v[:, h // g].abs()
        if v_scales is not None:
            vs = v_scales[:, h // g].clamp(min=1e-30)
            top = (p * vs).amax(1, keepdim=True) if p.shape[1] else torch.zeros((p.shape[0], 1), dtype=p.dtype, device=p.device)
            size[:, h] += 2.0 ** -29.5 * top * (sees.double() @ (v[:, h // g].abs() / vs[:, None]))
    return out, size


def make_cache(lens, heads, d, fmt, page_size, seed, spare=3, device="cuda:0", garbage=True):
    """A cache whose first lens[b] tokens of every sequence hold values of about N(0, 1); all other slots hold the worst bytes
    there are (NaN codes, NaN scales).  Returns (cache, page_table [B, P] with -1 behind the last page)."""
    from gemlite_b200 import QuantizedKVCache
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page_size) for n in lens]
    width, total = max(pages + [1]), sum(pages) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    cache = QuantizedKVCache(total, page_size, heads, d, fmt, device=device)
    used = torch.zeros((total, page_size), dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[int(table[b, p // page_size]), p % page_size] = True
    used = used.to(device)[:, None]
    dev = torch.Generator(device=device).manual_seed(seed)
    for w in "kv":
        codes, scales = getattr(cache, w + "_codes"), getattr(cache, w + "_scales")
        if fmt == "fp8":
            c = (torch.randn(codes.shape, generator=dev, device=device) * 120).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        elif fmt == "int8":
            c = (torch.randn(codes.shape, generator=dev, device=device) * 40).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            c = torch.randint(0, 256, codes.shape, generator=dev, device=device, dtype=torch.uint8)
            z = torch.randint(0, 16, scales.shape, generator=dev, device=device, dtype=torch.uint8)
            getattr(cache, w + "_zeros").copy_(torch.where(used, z, torch.full_like(z, 255)) if garbage else z)
        s = (torch.rand(scales.shape, generator=dev, device=device) + 0.5) * {"fp8": 1 / 120, "int8": 1 / 40, "int4": 1 / 5}[fmt]
        if garbage:
            c = torch.where(used[..., None], c, torch.full_like(c, 0x7F))
            s = torch.where(used, s, torch.full_like(s, math.nan))
        codes.copy_(c)
        scales.copy_(s)
    return cache, table.to(device)
