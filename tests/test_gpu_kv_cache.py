"""GPU: the quantised key/value cache against plain 64-bit forms (tests/kv_util.py): writing (head norms, rotary positions,
quantisation, slots), reading back, attention for single tokens, drafted trees and prompt chunks; and what must not happen:
slots, rows and results touched that are nobody's, garbage in unseen slots that reaches a result."""
import math

import pytest
import torch

from tests.kv_util import attend64, held64, make_cache, norm64, rotate64, scales64, score_slack64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FMTS = ("fp8", "int8", "int4")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


# ---- write ------------------------------------------------------------------------------------------------------------------
def _check_held(got, want, scale, fmt, codes_top):
    """`got` is what the cache holds, `want` the unquantised 64-bit values.  Half a step of the code's format, plus what fp32
    arithmetic (norm, rotation, division: a dozen operations of 2^-24 relative to the row's largest value) may add."""
    top = want.abs().amax(-1, keepdim=True)
    slack = 12 * 2.0 ** -24 * 2 * top
    if fmt == "fp8":
        # e4m3: half a step is 2^-4 of the value; below the smallest normal number half of 2^-9 (codes are value / scale)
        step = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale)
    else:
        step = 0.5 * scale
    # a value within `slack` of a border may take the neighbouring code: the bound moves by the same slack
    assert bool(((got - want).abs() <= step * (1 + 2.0 ** -20) + slack).all()), ((got - want).abs() - step - slack).max()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d,dtype,hq,hkv,rot,inter,norm,page", [
    (128, torch.bfloat16, 8, 2, 128, False, True, 16), (64, torch.float16, 5, 5, 64, True, True, 7),
    (128, torch.float16, 3, 1, 48, False, False, 1), (64, torch.bfloat16, 24, 4, 0, False, True, 64),
    (128, torch.bfloat16, 2, 2, 16, True, False, 33)])
def test_write_matches_the_formula(lib, fmt, d, dtype, hq, hkv, rot, inter, norm, page):
    from gemlite_b200 import KVBatch, rotary_table
    ctx, new = [0, 5, 130, 31], [3, 0, 1, 17]
    n_pad, total = 4, sum(new)
    cache, table = make_cache([c + t for c, t in zip(ctx, new)], hkv, d, fmt, page, seed=d + rot + page)
    before = {w: getattr(cache, w).clone() for w in ("k_codes", "v_codes", "k_scales", "v_scales")}
    qkv = _randn(rot + page, total + n_pad, (hq + 2 * hkv) * d, dtype=dtype, scale=2.0)
    q, k, v = (x.view(total + n_pad, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    wq, wk = ((1 + 0.3 * _randn(s, d, dtype=torch.float32)).to(dtype) for s in (1, 2)) if norm else (None, None)
    pos = torch.cat([torch.arange(c, c + t) for c, t in zip(ctx, new)] + [torch.full((n_pad,), 10 ** 9)]).to(DEV)
    cs = rotary_table(200, rot, 10000.0, DEV) if rot else None
    off = _i32([0] + torch.tensor(new).cumsum(0).tolist())
    out = cache.write(q, k, v, KVBatch(table, _i32(ctx), off), positions=pos, cos_sin=cs, q_norm=wq, k_norm=wk, eps=1e-5, interleaved=inter)

    q64, k64, v64 = (x[:total].double() for x in (q, k, v))
    q64, k64 = norm64(q64, wq, 1e-5), norm64(k64, wk, 1e-5)
    if rot:
        q64, k64 = rotate64(q64, cs, pos[:total], inter), rotate64(k64, cs, pos[:total], inter)
    # one rounding to 16 bits, and fp32 arithmetic relative to the rotated pair's size
    tol = torch.finfo(dtype).eps / 2 * q64.abs() + 16 * 2.0 ** -24 * q64.abs().amax(-1, keepdim=True)
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 0)            # half of fp16's smallest step
    assert bool(((out[:total].double() - q64).abs() <= tol).all())

    at = 0
    written = torch.zeros((cache.num_pages, page), dtype=torch.bool, device=DEV)
    for b, (c, t) in enumerate(zip(ctx, new)):
        for w, want in (("k", k64), ("v", v64)):
            got = held64(cache, w, table, b, c + t)[c:]
            scale = torch.stack([getattr(cache, w + "_scales")[int(table[b, p // page]), :, p % page] for p in range(c, c + t)])[..., None].double() if t else torch.zeros(1, device=DEV)
            _check_held(got, want[at:at + t], scale, fmt, None)
        for p in range(c, c + t):
            written[int(table[b, p // page]), p % page] = True
        at += t
    # every other slot is as it was, bit for bit
    for w, old in before.items():
        new_t, keep = getattr(cache, w), ~written[:, None]
        if new_t.dim() == 4:
            keep = keep[..., None]
        same = (new_t.view(torch.uint8) if new_t.dtype == torch.uint8 else new_t.view(torch.int32)) == (old if old.dtype == torch.uint8 else old.view(torch.int32))
        assert bool((same | ~keep).all()), w


def test_write_scales_and_codes_by_hand(lib):
    from gemlite_b200 import KVBatch
    x = torch.zeros(4, 1, 64, device=DEV)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2] = 254.0, -127.0, 1.0            # int8 scale 2
    x[1] = 0.0                                                        # an all-zero row: the smallest scale
    x[2, 0, 5] = math.inf
    x[3, 0, 6] = math.nan
    for fmt in FMTS:
        cache, table = make_cache([4], 1, 64, fmt, 4, seed=1)
        b = x.to(torch.bfloat16)
        assert cache.write(None, b, b, KVBatch(table, _i32([0]))) is None
        page = int(table[0, 0])
        s, c = cache.k_scales[page, 0], cache.k_codes[page, 0]
        assert torch.equal(cache.v_scales[page, 0].view(torch.int32), s.view(torch.int32)) and torch.equal(cache.v_codes[page, 0], c)
        top = {"fp8": 254.0 / 448, "int8": 2.0, "int4": 381.0 / 15}[fmt]
        assert abs(float(s[0]) - top) <= 2.0 ** -23 * top and float(s[1]) == float(torch.tensor(1e-6))
        assert bool(s[2:].isnan().all()) and int(c[2:].max()) == 0
        if fmt == "int8":
            assert c[0, :3].view(torch.int8).tolist() == [127, -64, 0]   # -63.5 and 0.5 are ties: to the even neighbour
        if fmt == "int4":
            assert int(cache.k_zeros[page, 0, 0]) == 5 and int(c[0, 0]) == 15 | 0 << 4 and int(c[0, 1]) == 5 | 5 << 4
        k, v = cache.read(table, _i32([4]), out_dtype=torch.float32)
        assert bool(k[0, 2:].isnan().all()) and bool((k[0, 1] == 0).all()) and torch.equal(k[0, :2], v[0, :2])


def test_write_outside_the_table_and_the_pool(lib):
    """Positions outside the rotation's table give NaN rows; tokens without a page are dropped; nothing else changes."""
    from gemlite_b200 import KVBatch, rotary_table
    cache, table = make_cache([8, 8], 2, 64, "fp8", 4, seed=2)
    page = table.clone()
    table[1, 1] = 10 ** 6                                             # a page that is not there
    k = _randn(3, 12, 2, 64)
    before = cache.k_codes.clone()
    pos = torch.tensor([0, 1, 2, 7, -1, 5] * 2, device=DEV)
    out = cache.write(k, k, k, KVBatch(table, _i32([4, 4]), _i32([0, 6, 12])), positions=pos, cos_sin=rotary_table(6, 64, device=DEV))
    bad = torch.tensor([False, False, False, True, True, False] * 2, device=DEV)
    assert bool(out[bad].isnan().all()) and not bool(out[~bad].isnan().any())
    # sequence 0: tokens 4..7 fit, 8 and 9 are behind the table; sequence 1 has no page for its tokens
    changed = (cache.k_codes != before).flatten(2).any(2).any(1)
    assert changed.nonzero().flatten().tolist() == [int(page[0, 1])]
    assert bool(cache.k_scales[int(page[0, 1]), :, 3].isnan().all()) and not bool(cache.k_scales[int(page[0, 1]), :, :3].isnan().any())


# ---- read -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d,page,out_dtype", [(128, 16, torch.bfloat16), (64, 5, torch.float16), (128, 48, torch.float32)])
def test_read_matches_the_formula(lib, fmt, d, page, out_dtype):
    lens = [0, 1, 33, 97]
    cache, table = make_cache(lens, 3, d, fmt, page, seed=page)
    if page == 16:
        table[3, 2] = -1                                              # a hole: zeros
    for max_len in (None, 97, 40, 1000):
        k, v = cache.read(table, _i32(lens), max_len=max_len, out_dtype=out_dtype)
        L = table.shape[1] * page if max_len is None else max_len
        assert k.shape == v.shape == (4, L, 3, d) and k.dtype == out_dtype
        for x, w in ((k, "k"), (v, "v")):
            for b, n in enumerate(lens):
                n = min(n, L)
                want = held64(cache, w, table, b, n)
                want = torch.where(want.isnan(), 0.0, want)           # (all held values are numbers)
                tol = torch.finfo(out_dtype).eps / 2 * want.abs() + 2.0 ** -24 * want.abs() + (2.0 ** -25 if out_dtype == torch.float16 else 0)
                assert bool(((x[b, :n].double() - want).abs() <= tol).all())
                assert bool((x[b, n:] == 0).all())


# ---- attend -----------------------------------------------------------------------------------------------------------------
def _tree(seed, new, width):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for t in new:
        m = torch.zeros((t, width), dtype=torch.bool)
        for i in range(t):
            if i:
                m[i] = m[int(torch.randint(0, i, (1,), generator=g))]
            m[i, i] = True
        rows.append(m)
    return torch.cat(rows).to(DEV)


def _check_attend(cache, table, ctx, new, q, mask, out, scale=None, rounds_codes=False):
    """Against fp64.  Per element: half a step of the output's type, and of sum p |v|: 2^-11 for the weights' rounding to fp16,
    2^-12 for the exponents (scores of up to about 40 with fp32 sums over 128 products: 40 * 128 * 2^-24 * log2 e < 2^-11
    at the very worst, and sums do not line up), doubled for the denominator; what the smallest weights lose in fp16 is
    counted by attend64 (first run without it: a weight of 2^-34 beside one of 1, on a channel where the large one's code is
    0, was off by 0.8 %; its fp16 number 2^-19 has a step of 2^-24).

    rounds_codes: the kernel for many rows rounds scaled values and keys to fp16: 2^-11 of sum p |v| for the values, and for
    the keys twice (numerator, denominator) what score_slack64 says; its smallest weights have 2^-31 of the largest as their
    last normal order, 2^8 times the other kernel's floor."""
    rounds_codes = rounds_codes or max(new) * (q.shape[1] // cache.n_kv_heads) > 32
    at = 0
    for b, (c, t) in enumerate(zip(ctx, new)):
        if t == 0:
            continue
        cap = min(c + t, table.shape[1] * cache.page_size)
        k, v = held64(cache, "k", table, b, cap), held64(cache, "v", table, b, cap)
        col = table[b, torch.arange(cap, device=DEV) // cache.page_size]
        hole = (col < 0) | (col >= cache.num_pages)
        sees = torch.zeros((t, cap), dtype=torch.bool, device=DEV)
        sees[:, :min(c, cap)] = True
        own = torch.ones((t, t), device=DEV).tril().bool() if mask is None else torch.nn.functional.pad(mask[at:at + t].bool(), (0, t))[:, :t]
        sees[:, min(c, cap):] = own[:, :cap - min(c, cap)]
        sees &= ~hole
        want, size = attend64(q[at:at + t], k, v, sees, 1 / math.sqrt(cache.head_dim) if scale is None else scale,
                              scales64(cache, "v", table, b, cap))
        tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -9.5 * size + (2.0 ** -25 if q.dtype == torch.float16 else 0)
        if rounds_codes:
            plain = attend64(q[at:at + t], k, v, sees, 1 / math.sqrt(cache.head_dim) if scale is None else scale)[1]
            slack = score_slack64(q[at:at + t], k, sees, 1 / math.sqrt(cache.head_dim) if scale is None else scale)
            tol = tol + 2.0 ** -11 * plain + 2 * slack[..., None] * plain + (2.0 ** 8 - 1) * 2.0 ** -9.5 * (size - plain)
        err = (out[at:at + t].double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol.clamp(min=1e-30)).max()))
        at += t


SHAPES = [  # hq, hkv, page, cached tokens, new tokens
    (8, 1, 16, [0, 1, 31, 32, 33, 127, 128, 129, 500], [1] * 9),
    (4, 4, 64, [70], [1]),
    (8, 2, 48, [1500, 3, 0], [1, 1, 1]),
    (8, 2, 5, [90, 0, 257, 64, 12], [7, 1, 0, 5, 2]),
    (6, 2, 16, [200, 10], [16, 9]),
    (16, 2, 32, [300, 0], [64, 33]),
    (5, 1, 128, [1000], [40]),
    (32, 2, 64, [0, 150], [100, 60]),
    # several pieces per block: many sequences of one or two tiles; few long ones; units of one and of two row blocks mixed
    (16, 4, 16, [17 * i % 150 for i in range(48)], [1 + i % 5 for i in range(48)]),
    (24, 8, 32, [1400, 90, 2100, 700], [40, 1, 45, 100]),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attend_matches_the_formula(lib, fmt, d, dtype, shape):
    from gemlite_b200 import KVBatch
    hq, hkv, page, ctx, new = SHAPES[shape]
    cache, table = make_cache([c + t for c, t in zip(ctx, new)], hkv, d, fmt, page, seed=shape)
    q = _randn(shape, sum(new), hq, d, dtype=dtype, scale=1.5)
    off = _i32([0] + torch.tensor(new).cumsum(0).tolist())
    batch = KVBatch(table, _i32(ctx), off, max_len=max(c + t for c, t in zip(ctx, new)), max_new=max(new))
    for kernel in (0, 1, 2):
        _check_attend(cache, table, ctx, new, q, None, cache.attend(q, batch, kernel_override=kernel), rounds_codes=kernel == 2)
    tree = _tree(shape, new, max(new))
    _check_attend(cache, table, ctx, new, q, tree, cache.attend(q, batch, mask=tree))
    # any mask: rows that see none of the new tokens (nothing at all where nothing is cached), tokens that nobody sees
    g = torch.Generator(device=DEV).manual_seed(shape)
    some = torch.rand(tree.shape, generator=g, device=DEV) < 0.3
    some[::3] = False
    for kernel in (0, 1, 2):
        _check_attend(cache, table, ctx, new, q, some, cache.attend(q, batch, mask=some, kernel_override=kernel), rounds_codes=kernel == 2)
    # bounds that say nothing (all rows might be one sequence's: the kernel for many rows) or too little change no result
    # beyond that kernel's roundings and the order of sums
    for kw in ({}, {"max_len": 1, "max_new": 1}):
        _check_attend(cache, table, ctx, new, q, tree, cache.attend(q, KVBatch(table, _i32(ctx), off, **kw), mask=tree.to(torch.uint8)), rounds_codes=True)


@pytest.mark.parametrize("fmt", FMTS)
def test_attend_empty_rows_give_zeros_and_rows_of_nobody_stay(lib, fmt):
    from gemlite_b200 import KVBatch
    cache, table = make_cache([2, 3], 2, 64, fmt, 4, seed=5)
    q = _randn(1, 9, 4, 64)
    out = torch.full_like(q, 7.0)
    mask = torch.zeros(9, 3, dtype=torch.bool, device=DEV)
    mask[3, 0] = True
    got = cache.attend(q, KVBatch(table, _i32([0, 0]), _i32([1, 3, 6])), mask=mask, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[0] == 7).all()) and bool((out[6:] == 7).all())
    assert bool((out[[1, 2, 4, 5]] == 0).all())
    v = held64(cache, "v", table, 1, 1)[0]
    assert bool(((out[3].double() - v.repeat_interleave(2, 0)).abs() <= 2.0 ** -7 * v.repeat_interleave(2, 0).abs() + 1e-6).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,hq", [(3, 4), (40, 16)])
def test_attend_unseen_tokens_have_no_influence(lib, fmt, T, hq):
    """NaN and infinity in new tokens that only some rows see, in pages that are missing and in slots behind the end."""
    from gemlite_b200 import KVBatch
    ctx = 61
    cache, table = make_cache([ctx + T], 2, 128, fmt, 16, seed=6)
    q = _randn(2, T, hq, 128)
    mask = torch.ones(T, T, dtype=torch.bool, device=DEV).tril()
    mask[:, 1] = False
    mask[1, 1] = True                                               # only row 1 sees token 1
    batch = KVBatch(table, _i32([ctx]))
    want = cache.attend(q, batch, mask=mask)
    page, place = int(table[0, (ctx + 1) // 16]), (ctx + 1) % 16
    for scale, code in ((math.nan, 0x7F), (math.inf, 0x7F), (1.0, 0x7F), (1.0, 0xFF)):
        cache.k_scales[page, :, place] = scale
        cache.v_scales[page, :, place] = scale
        cache.k_codes[page, :, place] = code
        cache.v_codes[page, :, place] = code
        got = cache.attend(q, batch, mask=mask)
        keep = [i for i in range(T) if i != 1]
        assert torch.equal(got[keep], want[keep]), (scale, code)
        if fmt == "fp8" or not math.isfinite(scale):
            assert not bool(got[1].isfinite().any())
    # a sequence with a hole: its tokens count as absent
    hole = table.clone()
    hole[0, 1] = cache.num_pages
    _check_attend(cache, hole, [ctx - 1], [1], q[:1], None, cache.attend(q[:1], KVBatch(hole, _i32([ctx - 1]))))


def test_attend_one_token_far_above_the_rest_and_scales_far_apart(lib):
    """Weights over many orders of magnitude: one token's value scale is 2^20 times the others'; large scores."""
    from gemlite_b200 import KVBatch
    for fmt in FMTS:
        cache, table = make_cache([400], 1, 128, fmt, 16, seed=8)
        page = int(table[0, 3])
        cache.v_scales[page, :, 5] *= 2.0 ** 20
        cache.v_scales[int(table[0, 20])] *= 2.0 ** -30
        cache.v_scales[int(table[0, 21])] = 0.0                      # a scale of zero is a value of zero
        q = _randn(3, 1, 8, 128, scale=6.0)
        _check_attend(cache, table, [399], [1], q, None, cache.attend(q, KVBatch(table, _i32([399])), scale=0.05), scale=0.05)
        cache.v_scales.zero_()
        assert bool((cache.attend(q, KVBatch(table, _i32([399]))) == 0).all())


@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 1e6, 1e30])
def test_attend_queries_of_any_size(lib, magnitude):
    """bf16 queries far outside fp16's range, with a scale that brings the scores back."""
    from gemlite_b200 import KVBatch
    cache, table = make_cache([200], 2, 64, "int8", 32, seed=9)
    q = _randn(4, 2, 4, 64, scale=magnitude)
    _check_attend(cache, table, [198], [2], q, None, cache.attend(q, KVBatch(table, _i32([198])), scale=0.1 / magnitude), scale=0.1 / magnitude)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("kernel", [1, 2])
def test_attend_with_a_scale_of_zero_or_below(lib, scale, kernel):
    from gemlite_b200 import KVBatch
    cache, table = make_cache([300, 40], 2, 64, "fp8", 32, seed=15)
    q = _randn(6, 6, 8, 64)
    _check_attend(cache, table, [297, 37], [3, 3], q, None, cache.attend(q, KVBatch(table, _i32([297, 37])), scale=scale, kernel_override=kernel),
                  scale=scale, rounds_codes=kernel == 2)


def test_attend_scales_far_apart_for_many_rows(lib):
    """The kernel for many rows folds scales into the codes only where they are near each other."""
    from gemlite_b200 import KVBatch
    for fmt in FMTS:
        cache, table = make_cache([520], 1, 128, fmt, 16, seed=18)
        page = int(table[0, 3])
        cache.v_scales[page, :, 5] *= 2.0 ** 20
        cache.k_scales[int(table[0, 7])] *= 2.0 ** -13
        cache.v_scales[int(table[0, 20])] *= 2.0 ** -30
        cache.v_scales[int(table[0, 21])] = 0.0
        q = _randn(3, 20, 8, 128, scale=2.0)
        _check_attend(cache, table, [500], [20], q, None, cache.attend(q, KVBatch(table, _i32([500])), scale=0.05), scale=0.05)


def test_attend_strided_and_misaligned_queries(lib):
    from gemlite_b200 import KVBatch
    cache, table = make_cache([100], 2, 64, "fp8", 16, seed=10)
    batch = KVBatch(table, _i32([95]))
    flat = _randn(5, 5 * 8 * 64 + 8)
    base = flat[:5 * 8 * 64].view(5, 8, 64)
    want = cache.attend(base.contiguous(), batch)
    wide = torch.zeros(5, 20, 64, dtype=base.dtype, device=DEV)
    wide[:, 3:19:2] = base
    assert torch.equal(cache.attend(wide[:, 3:19:2], batch), want)
    odd = torch.empty(5 * 8 * 64 + 3, dtype=base.dtype, device=DEV)[3:].view(5, 8, 64)      # 6 bytes off
    odd.copy_(base)
    assert torch.equal(cache.attend(odd, batch), want)
    last = base.transpose(1, 2).contiguous().transpose(1, 2)                                # channels not contiguous
    assert torch.equal(cache.attend(last, batch), want)


def test_long_cache_offsets_pass_32_bits(lib):
    """Codes of more than 4 GB: slots at the far end are written, read and attended to."""
    from gemlite_b200 import KVBatch, QuantizedKVCache
    pages, ps, heads = 4300, 128, 64
    cache = QuantizedKVCache(pages, ps, heads, 128, "fp8", device=DEV)
    assert cache.k_codes.numel() > 2 ** 32
    table = torch.arange(pages - 2, pages, dtype=torch.int32, device=DEV)[None].contiguous()
    k, v, q = _randn(1, 130, heads, 128), _randn(2, 130, heads, 128), _randn(3, 1, heads, 128)
    cache.write(None, k, v, KVBatch(table, _i32([0])))
    kk, vv = cache.read(table, _i32([130]), max_len=130, out_dtype=torch.float32)
    assert bool(((kk[0] - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 2.0 ** -10 * 5 / 448).all())
    got = cache.attend(q, KVBatch(table, _i32([129])))
    want, size = attend64(q, kk[0].double(), vv[0].double(), torch.ones(1, 130, dtype=torch.bool, device=DEV), 128 ** -0.5)
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9.5 * size).all())
    assert int(cache.k_codes[:pages - 2].count_nonzero()) == 0


# ---- a run of them together --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
def test_prompt_draft_accept_decode(lib, fmt):
    """A prompt in two chunks, a tree of drafts, the accepted branch written again in order, one more token: the codes are
    those of writing the same tokens in one go, and every step's attention follows the formula."""
    from gemlite_b200 import KVBatch, rotary_table
    hq, hkv, d, page = 8, 2, 128, 16
    cache, table = make_cache([100], hkv, d, fmt, page, seed=11)
    plain, table2 = make_cache([100], hkv, d, fmt, page, seed=12)
    cs, w = rotary_table(128, d, device=DEV), (1 + 0.1 * _randn(0, d)).to(torch.bfloat16)
    q, k, v = _randn(1, 60, hq, d, scale=1.2), _randn(2, 60, hkv, d), _randn(3, 60, hkv, d)
    pos = torch.arange(60, device=DEV)

    def step(rows, ctx, positions, mask=None):
        b = KVBatch(table, _i32([ctx]))
        qr = cache.write(q[rows], k[rows], v[rows], b, positions=positions, cos_sin=cs, q_norm=w, k_norm=w)
        out = cache.attend(qr, b, mask=mask)
        _check_attend(cache, table, [ctx], [len(rows)], qr, mask, out)
        return b

    step(list(range(0, 33)), 0, pos[:33])
    step(list(range(33, 50)), 33, pos[33:50])
    mask = torch.eye(6, dtype=torch.bool, device=DEV)               # 0 -> 1, 2; 2 -> 3, 4; 4 -> 5
    for i, p in ((1, 0), (2, 0), (3, 2), (4, 2), (5, 4)):
        mask[i] |= mask[p]
    depth = mask.sum(1) - 1
    b = step([50, 51, 52, 53, 54, 55], 50, 50 + depth, mask)
    taken = [50, 52, 54, 55]                                          # the branch 0, 2, 4, 5
    one = KVBatch(table, b.ctx_lens)
    assert cache.write(None, k[taken], v[taken], one, positions=pos[50:54], cos_sin=cs, k_norm=w) is None
    step([56], 54, pos[54:55])
    rows = list(range(50)) + taken + [56]
    plain.write(None, k[rows], v[rows], KVBatch(table2, _i32([0])), positions=pos[:55], cos_sin=cs, k_norm=w)
    for x, y in zip(cache.read(table, _i32([55]), out_dtype=torch.float32), plain.read(table2, _i32([55]), out_dtype=torch.float32)):
        assert torch.equal(x[:, :55], y[:, :55])


def test_decoder_layer_linears_with_the_cache(lib):
    """tp.LlamaLinears: without a cache as before; with one, the output projection's input is the attention of the formula."""
    from gemlite_b200 import KVBatch, rotary_table, tp
    hidden, hq, hkv, d = 512, 8, 2, 64
    layer = tp.LlamaLinears(hidden, 1024, hq, hkv, d, 1, 0, DEV, seed=3)
    cache, table = make_cache([40, 9], hkv, d, "fp8", 16, seed=21)
    x = _randn(1, 5, hidden)
    seen = []
    layer.o.register_forward_pre_hook(lambda m, a: seen.append(a[0].clone()))
    layer.qkv.register_forward_hook(lambda m, a, y: seen.append(y.clone()))
    layer(x)
    assert torch.equal(seen[1], seen[0][:, :hq * d])
    seen.clear()
    batch, cs = KVBatch(table, _i32([36, 8]), _i32([0, 4, 5])), rotary_table(64, d, device=DEV)
    pos = torch.tensor([36, 37, 38, 39, 8], device=DEV)
    y = layer(x, cache, batch, positions=pos, cos_sin=cs)
    assert y.shape == x.shape and bool(y.isfinite().all())
    qkv, attn = seen
    q = qkv[:, :hq * d].view(5, hq, d)
    q64 = rotate64(q.double(), cs, pos, False)
    tol = torch.finfo(q.dtype).eps / 2 * q64.abs() + 16 * 2.0 ** -24 * q64.abs().amax(-1, keepdim=True)
    rotated = cache.write(q, qkv[:, hq * d:(hq + hkv) * d].view(5, hkv, d), qkv[:, (hq + hkv) * d:].view(5, hkv, d), batch, positions=pos, cos_sin=cs)
    assert bool(((rotated.double() - q64).abs() <= tol).all())
    _check_attend(cache, table, [36, 8], [4, 1], rotated, None, attn.view(5, hq, d))


def test_graph_capture_streams_and_repeats(lib):
    """A captured step replays with what the tensors hold then; two graphs and a side stream do not share scratch; the same
    call gives the same bits."""
    from gemlite_b200 import KVBatch
    hq, hkv, d, page = 8, 2, 128, 16
    cache, table = make_cache([2000, 1200], hkv, d, "fp8", page, seed=13)
    ctx = _i32([1999, 600])
    q = _randn(1, 2, hq, d)
    batch = KVBatch(table, ctx)
    want = cache.attend(q, batch)
    assert all(torch.equal(cache.attend(q, batch), want) for _ in range(20))
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(cache.attend(q, batch))
        graphs.append(g)
    ctx.copy_(_i32([1000, 1100]))
    later = cache.attend(q, batch)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], later) and torch.equal(outs[1], later) and not torch.equal(later, want)


@pytest.mark.parametrize("T,hq", [(5, 4), (24, 8)])
def test_masks_of_other_widths_and_strides(lib, T, hq):
    """Narrower than the new tokens (the rest counts as False), no columns at all, one row for all (stride 0), values other than 1."""
    from gemlite_b200 import KVBatch
    cache, table = make_cache([50 + T], 2, 64, "int8", 16, seed=16)
    q, batch = _randn(7, T, hq, 64), KVBatch(table, _i32([50]))
    narrow = torch.ones(T, 3, dtype=torch.bool, device=DEV)
    for mask in (narrow, narrow[:, :0], narrow[:1].expand(T, 3), torch.nn.functional.pad(narrow, (0, 40))[:, :T + 30]):
        want = torch.zeros(T, T, dtype=torch.bool, device=DEV)
        w = min(mask.shape[1], T)
        want[:, :w] = mask[:, :w]
        _check_attend(cache, table, [50], [T], q, want, cache.attend(q, batch, mask=mask))
    wide = torch.randint(0, 256, (T, T), dtype=torch.uint8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    wide[0] = 0
    _check_attend(cache, table, [50], [T], q, wide != 0, cache.attend(q, batch, mask=wide))


def test_whole_step_in_a_graph(lib):
    """Write, attend and read captured once, replayed with new lengths and inputs in place."""
    from gemlite_b200 import KVBatch, rotary_table
    cache, table = make_cache([200, 200], 2, 64, "int4", 16, seed=17)
    other, _ = make_cache([200, 200], 2, 64, "int4", 16, seed=17)
    cs, ctx, pos = rotary_table(256, 64, device=DEV), _i32([10, 40]), _i32([10, 40])
    q, k, v = _randn(1, 2, 8, 64), _randn(2, 2, 2, 64), _randn(3, 2, 2, 64)

    def step(c):
        b = KVBatch(table, ctx, max_len=200)
        y = c.attend(c.write(q, k, v, b, positions=pos, cos_sin=cs), b)
        return (y, *c.read(table, ctx + 1, max_len=200, out_dtype=torch.float16))

    step(cache), step(other)                     # (the caches hold the same; the first step writes to both)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step(cache)
    for n in range(3):
        q.copy_(_randn(10 + n, 2, 8, 64)), k.copy_(_randn(20 + n, 2, 2, 64)), v.copy_(_randn(30 + n, 2, 2, 64))
        ctx.add_(_i32([1, 50])), pos.copy_(ctx)
        g.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert bool(got[0].isfinite().all()) and all(torch.equal(x, y) for x, y in zip(got, want))


# ---- refusals ----------------------------------------------------------------------------------------------------------------
def test_refusals(lib):
    from gemlite_b200 import KVBatch, QuantizedKVCache
    cache, table = make_cache([20], 2, 64, "fp8", 16, seed=14)
    batch = KVBatch(table, _i32([10]))
    q, k = _randn(1, 2, 4, 64), _randn(2, 2, 2, 64)
    with pytest.raises(ValueError):
        QuantizedKVCache(1, 16, 2, 64, "fp4")
    with pytest.raises(NotImplementedError):
        QuantizedKVCache(1, 16, 2, 96, "fp8")
    with pytest.raises(ValueError):
        QuantizedKVCache(0, 16, 2, 64, "fp8")
    with pytest.raises(ValueError):
        KVBatch(table.long(), _i32([10]))
    with pytest.raises(ValueError):
        KVBatch(table, _i32([10, 11]))
    with pytest.raises(ValueError):
        KVBatch(table, _i32([10]), _i32([0]))
    with pytest.raises(RuntimeError):
        KVBatch(table.cpu(), _i32([10]))
    with pytest.raises(NotImplementedError):
        cache.attend(q.float(), batch)
    with pytest.raises(ValueError):
        cache.attend(_randn(1, 2, 3, 64), batch)                     # 3 heads over 2
    with pytest.raises(ValueError):
        cache.attend(_randn(1, 2, 4, 128), batch)
    with pytest.raises(ValueError):
        cache.attend(q, batch, mask=torch.ones(3, 2, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError):
        cache.attend(q, batch, mask=torch.ones(2, 2, device=DEV))
    with pytest.raises(ValueError):
        cache.attend(q, batch, out=torch.empty(2, 4, 64, dtype=torch.float16, device=DEV))
    with pytest.raises(ValueError):
        cache.write(q, k, k[:1], batch)
    with pytest.raises(ValueError):
        cache.write(q.half(), k, k, batch)
    with pytest.raises(ValueError):
        cache.write(q, k, k, batch, cos_sin=torch.zeros(4, 64, device=DEV))          # no positions
    with pytest.raises(ValueError):
        cache.write(q, k, k, batch, cos_sin=torch.zeros(4, 24, device=DEV), positions=_i32([0, 1]))
    with pytest.raises(ValueError):
        cache.write(q, k, k, batch, q_norm=torch.ones(32, device=DEV))
    with pytest.raises(ValueError):
        cache.write(_randn(1, 3, 4, 64), _randn(2, 3, 2, 64), _randn(2, 3, 2, 64), KVBatch(table.repeat(2, 1), _i32([1, 1])))   # 3 rows, 2 sequences
    with pytest.raises(NotImplementedError):
        cache.read(table, _i32([10]), out_dtype=torch.int8)
    # nothing to do is fine
    assert cache.attend(q[:0], batch).shape == (0, 4, 64)
    assert cache.attend(q[:0], KVBatch(table[:0], _i32([]))).shape == (0, 4, 64)
    cache.write(q[:0], k[:0], k[:0], batch)
    assert cache.read(table[:0], _i32([]))[0].shape[0] == 0
