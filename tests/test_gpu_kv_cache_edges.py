"""GPU: the quantised key/value cache where its numbers and its promises are stretched: scales of zero over long stretches,
what a row does not see, against plain 64-bit forms (tests/kv_util.py)."""
import math

import pytest
import torch

from tests.kv_util import make_cache, norm64
from tests.test_gpu_kv_cache import DEV, FMTS, _check_attend, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("fmt", FMTS)
def test_long_stretches_of_zero_scales(lib, fmt, kernel):
    """30016 slots that were never written (scales of zero, scores of zero), then ordinary tokens: the zeros weigh as much as
    their scores say.  24 sequences of 8 heads share the pages, so that a block's piece holds more than 12000 tokens."""
    from gemlite_b200 import KVBatch
    B, hkv, n, zero = 24, 8, 40000, 30016
    cache, table = make_cache([n], hkv, 64, fmt, 64, seed=32)
    pages = table[0, :zero // 64].long()
    cache.k_scales[pages] = 0.0
    cache.v_scales[pages] = 0.0
    table = table.expand(B, -1).contiguous()
    q = _randn(33, B, hkv, 64)
    out = cache.attend(q, KVBatch(table, _i32([n - 1] * B), max_len=n, max_new=1), kernel_override=kernel)
    _check_attend(cache, table, [n - 1] * B, [1] * B, q, None, out, rounds_codes=kernel == 2)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ctx,hq", [(0, 16), (61, 16), (700, 16), (700, 64), (61, 2)])
def test_later_tokens_of_a_chunk_do_not_reach_earlier_rows(lib, fmt, ctx, hq):
    """No mask: row i sees the new tokens up to its own.  Whatever scales and codes the last one holds, the rows before it keep
    every bit."""
    from gemlite_b200 import KVBatch
    T, hkv = 40, 2
    cache, table = make_cache([ctx + T], hkv, 128, fmt, 16, seed=30)
    q = _randn(31, T, hq, 128, dtype=torch.float16, scale=1.5)
    batch = KVBatch(table, _i32([ctx]), max_len=ctx + T, max_new=T)
    page, at = int(table[0, (ctx + T - 1) // 16]), (ctx + T - 1) % 16
    for kernel in (0, 1, 2):
        want = cache.attend(q, batch, kernel_override=kernel)
        kept = [t.clone() for t in (cache.k_scales, cache.v_scales, cache.k_codes, cache.v_codes)]
        for ks, vs, code in ((2.0 ** -14, 1.0, None), (1.0, 2.0 ** -14, None), (1.0, 2.0 ** 6, None), (2.0 ** 20, 2.0 ** 20, 0x55), (0.0, 0.0, 0),
                             (math.inf, math.inf, 0x7F), (math.nan, math.nan, 0xFF), (1.0, 1.0, 0x7F)):
            cache.k_scales[page, :, at] *= ks
            cache.v_scales[page, :, at] *= vs
            if code is not None:
                cache.k_codes[page, :, at] = code
                cache.v_codes[page, :, at] = code
            got = cache.attend(q, batch, kernel_override=kernel)
            for t, old in zip((cache.k_scales, cache.v_scales, cache.k_codes, cache.v_codes), kept):
                t.copy_(old)
            assert torch.equal(got[:-1], want[:-1]), (kernel, ks, vs, code)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,ctx,T", [(1, 61, 40), (1, 700, 40), (24, 700, 40), (48, 1100, 16)])
def test_unseen_tokens_over_many_tiles(lib, fmt, B, ctx, T):
    """One draft token that only row 1 sees gets a key 64 times as large, so that row 1's maximum rises far on the last tile: all
    other rows keep every bit.  24 and 48 sequences: pieces of many tiles, whose running maxima matter."""
    from gemlite_b200 import KVBatch
    hkv, hq = 8, 64
    cache, table = make_cache([ctx + T] * B, hkv, 128, fmt, 16, seed=30)
    q = _randn(31, B * T, hq, 128, dtype=torch.float16, scale=1.5)
    mask = torch.ones(T, T, dtype=torch.bool, device=DEV).tril()
    mask[:, 1] = False
    mask[1, 1] = True
    mask = mask.repeat(B, 1)
    batch = KVBatch(table, _i32([ctx] * B), max_len=ctx + T, max_new=T)
    want = cache.attend(q, batch, mask=mask)
    others = torch.arange(B * T, device=DEV) % T != 1
    pages = table[:, (ctx + 1) // 16].long()
    for factor in (64.0, 2.0 ** -20):
        cache.k_scales[pages, :, (ctx + 1) % 16] *= factor
        got = cache.attend(q, batch, mask=mask)
        assert not torch.equal(got[~others], want[~others])
        assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_that_span_more_than_fp32(lib, fmt):
    """Finite bf16 rows keep finite values, also where the largest less the smallest number is beyond fp32: each comes back within
    half a step (e4m3: 2^-4 of it, codes below its smallest normal number 2^-10 of the scale).  2.7e38 and -3e38 over 15
    steps are 3.8e37 each: 8 below the zero point (-3.04e38) and 7 above it (2.66e38) are fp32 numbers."""
    from gemlite_b200 import KVBatch
    cache, table = make_cache([8], 1, 64, fmt, 16, seed=1)
    x = _randn(1, 2, 1, 64)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2] = 2.7e38, -3e38, 1e38
    batch = KVBatch(table, _i32([0]))
    cache.write(None, x, x, batch)
    for got in cache.read(table, _i32([2]), max_len=2, out_dtype=torch.float32):
        scale = cache.k_scales[int(table[0, 0]), 0, :2, None].double()
        step = torch.maximum(2.0 ** -4 * x[:, 0].double().abs(), 2.0 ** -10 * scale) if fmt == "fp8" else 0.5 * scale
        top = x[:, 0].double().abs().amax(-1, keepdim=True)
        assert bool(((got[0, :, 0].double() - x[:, 0].double()).abs() <= step + 2.0 ** -20 * top).all())


@pytest.mark.parametrize("size", [1e18, 1e19, 1e25, 3e38])
def test_norm_of_large_heads(lib, size):
    """Head norms of bf16 rows whose mean square is no fp32 number; a row with an infinity among them stays no number."""
    from gemlite_b200 import KVBatch
    cache, table = make_cache([8], 1, 64, "int8", 16, seed=1)
    x = _randn(1, 3, 6, 64)
    x = (x / x.abs().amax().float() * size).to(torch.bfloat16)
    x[2, :, 7] = math.inf
    w = 1 + 0.3 * _randn(2, 64, dtype=torch.float32)
    k = x[:, :1]
    out = cache.write(x, k, k, KVBatch(table, _i32([0])), q_norm=w, k_norm=w)
    want = norm64(x.double(), w, 1e-6)[:2]
    # one rounding to bf16; the reciprocal root is rounded to 2^-149 beside 2^-128 at the least
    assert bool(((out[:2].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -22 + 8 * 2.0 ** -24) * want.abs()).all())
    assert bool(out[2, :, 7].isnan().all())
    key = cache.read(table, _i32([3]), max_len=3, out_dtype=torch.float32)[0]
    scale = want[:, :1].abs().amax(-1, keepdim=True) / 127
    assert bool(((key[0, :2].double() - want[:, :1]).abs() <= 0.5 * scale * (1 + 2.0 ** -10)).all()) and bool(key[0, 2].isnan().all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,hq", [(1, 8), (4, 8), (24, 32), (150, 32)])
@pytest.mark.parametrize("graph", [False, True])
def test_overwritten_slots_are_read_anew(lib, fmt, T, hq, graph):
    """write and attend in turn on the same slots, launched while the kernels before them still run: every attend sees what the
    write before it left, as it does when each call is waited for."""
    from gemlite_b200 import KVBatch
    hkv, steps, ctx = 2, 30, 200
    cache, table = make_cache([ctx + T] * 6, hkv, 128, fmt, 16, seed=40)
    n = 6 * T
    q, k, v = _randn(41, n, hq, 128), _randn(42, steps, n, hkv, 128), _randn(43, steps, n, hkv, 128)
    batch = KVBatch(table, _i32([ctx] * 6), max_len=ctx + T, max_new=T)

    def step(i):
        cache.write(None, k[i], v[i], batch)
        return cache.attend(q, batch)

    want = []
    for i in range(steps):
        want.append(step(i))
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = [step(i) for i in range(steps)]
        g.replay()
    else:
        got = [step(i) for i in range(steps)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_status_after_clean_launches(lib):
    """(A wait that runs out cannot be made on a GPU without work left in flight.)"""
    from gemlite_b200 import KVBatch, kv_cache
    cache, table = make_cache([300], 2, 128, "fp8", 16, seed=50)
    out = cache.attend(_randn(51, 40, 16, 128), KVBatch(table, _i32([260])))
    assert kv_cache.attend_status() == 0 == kv_cache.attend_status(DEV, clear=False) and bool(out.isfinite().all())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert kv_cache.attend_status("cuda") == 0


# ---- many sequences, many rows -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kernel,B", [(1, 129), (1, 700), (2, 641), (2, 1500)])
def test_more_sequences_than_threads(lib, kernel, B):
    """Where a thread that adds up the work takes several sequences."""
    from gemlite_b200 import KVBatch
    ctx, new = [(37 * i) % 211 for i in range(B)], [(i * 5) % 4 for i in range(B)]
    ctx[B // 2] = 3000
    cache, table = make_cache([c + t for c, t in zip(ctx, new)], 2, 64, "int8", 16, seed=60)
    q = _randn(61, sum(new), 4, 64)
    batch = KVBatch(table, _i32(ctx), _i32([0] + torch.tensor(new).cumsum(0).tolist()), max_len=3003, max_new=3)
    _check_attend(cache, table, ctx, new, q, None, cache.attend(q, batch, kernel_override=kernel), rounds_codes=kernel == 2)


@pytest.mark.parametrize("masked", [False, True])
def test_many_rows_repeat_streams_and_graphs(lib, masked):
    """The tcgen05 kernel: the same call gives the same bits; two graphs and side streams share no scratch; a replay sees the lengths
    that the tensors hold then."""
    from gemlite_b200 import KVBatch
    hq, hkv, T = 64, 8, 50
    cache, table = make_cache([2000, 1200, 300], hkv, 128, "fp8", 16, seed=62)
    ctx = _i32([1950, 600, 0])
    q = _randn(63, 3 * T, hq, 128)
    mask = torch.ones(T, T, dtype=torch.bool, device=DEV).tril().repeat(3, 1) if masked else None
    batch = KVBatch(table, ctx)
    want = cache.attend(q, batch, mask=mask)
    assert all(torch.equal(cache.attend(q, batch, mask=mask), want) for _ in range(20))
    side, graphs, outs = torch.cuda.Stream(), [], []
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(cache.attend(q, batch, mask=mask))
        graphs.append(g)
    ctx.copy_(_i32([1000, 1100, 250]))
    later = cache.attend(q, batch, mask=mask)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = []
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager.append(cache.attend(q, batch, mask=mask))
    torch.cuda.synchronize()
    assert all(torch.equal(x, later) for x in outs + eager) and not torch.equal(later, want)


def test_long_cache_with_many_rows(lib):
    """Codes of more than 4 GB under the tcgen05 kernel: pages at the far end."""
    from gemlite_b200 import KVBatch, QuantizedKVCache
    pages, ps, heads, T = 4300, 128, 64, 66
    cache = QuantizedKVCache(pages, ps, heads, 128, "fp8", device=DEV)
    assert cache.k_codes.numel() > 2 ** 32
    table = torch.arange(pages - 2, pages, dtype=torch.int32, device=DEV)[None].contiguous()
    k, v, q = _randn(1, 130, heads, 128), _randn(2, 130, heads, 128), _randn(3, T, heads, 128)
    cache.write(None, k, v, KVBatch(table, _i32([0])))
    out = cache.attend(q, KVBatch(table, _i32([130 - T])), kernel_override=2)
    _check_attend(cache, table, [130 - T], [T], q, None, out, rounds_codes=True)


# ---- what a write leaves, bit for bit ------------------------------------------------------------------------------------------
def _codes32(x, fmt):
    """Codes, scales and zero points of the rows of x (fp32, on the CPU) by the formulas, every operation rounded to fp32 by itself."""
    if fmt == "int4":
        lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
        scale = ((hi - lo) / torch.full_like(lo, 15)).clamp(min=1e-6)
        zero = (-lo / scale).round().clamp(0, 15)
        c = ((x / scale).round() + zero).clamp(0, 15).to(torch.uint8)
        return c[..., 0::2] | c[..., 1::2] << 4, scale[..., 0], zero[..., 0].to(torch.uint8)
    top = 448.0 if fmt == "fp8" else 127.0
    most = x.abs().amax(-1, keepdim=True)
    scale = (most / torch.full_like(most, top)).clamp(min=1e-6)
    c = (x / scale).clamp(-top, top)
    c = c.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "fp8" else c.round().to(torch.int8).view(torch.uint8)
    return c, scale[..., 0], None


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d,hkv,dtype,inter", [(128, 8, torch.bfloat16, False), (64, 3, torch.float16, True)])
def test_written_bits(lib, fmt, d, hkv, dtype, inter):
    """Codes, scales and zero points equal those of the formulas in fp32 (the norm's sum of squares in fp64), and nobody's slots
    keep all of theirs, zero points too."""
    from gemlite_b200 import KVBatch, rotary_table
    ctx, new, page = [0, 33, 70], [500, 1, 90], 16
    cache, table = make_cache([c + t for c, t in zip(ctx, new)], hkv, d, fmt, page, seed=70)
    names = ["k_codes", "v_codes", "k_scales", "v_scales"] + (["k_zeros", "v_zeros"] if fmt == "int4" else [])
    want = {n: getattr(cache, n).cpu().clone() for n in names}
    n = sum(new)
    k, v = _randn(71, n, hkv, d, dtype=dtype, scale=2.0), _randn(72, n, hkv, d, dtype=dtype, scale=3.0)
    w, cs = (1 + 0.3 * _randn(73, d, dtype=torch.float32)).to(dtype), rotary_table(700, d, device=DEV)
    pos = torch.cat([torch.arange(c, c + t) for c, t in zip(ctx, new)])
    cache.write(None, k, v, KVBatch(table, _i32(ctx), _i32([0] + torch.tensor(new).cumsum(0).tolist())), positions=pos.to(DEV), cos_sin=cs, k_norm=w,
                eps=1e-5, interleaved=inter)

    x = k.cpu().float()
    mean = (x.double().square().sum(-1, keepdim=True) / d).float()
    # (torch's CPU square root in fp32 is an ulp off for some arguments; through fp64 it is the correctly rounded one)
    x = x * (torch.ones_like(mean) / (mean + 1e-5).double().sqrt().float()) * w.cpu().float()
    t = cs.cpu()[pos][:, None]
    cos, sin = t[..., :d // 2], t[..., d // 2:]
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :d // 2], x[..., d // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    x = torch.stack([ra, rb], -1).flatten(-2) if inter else torch.cat([ra, rb], -1)
    rows = torch.cat([torch.full((t,), b) for b, t in enumerate(new)])
    pages, places = table.cpu()[rows, pos // page].long(), pos % page
    for which, y in (("k", x), ("v", v.cpu().float())):
        for name, value in zip(("_codes", "_scales", "_zeros"), _codes32(y, fmt)):
            if value is not None:
                want[which + name][pages, :, places] = value
    for name in names:
        got, ref = getattr(cache, name).cpu(), want[name]
        as_bits = (lambda t: t.view(torch.int32)) if ref.dtype == torch.float32 else (lambda t: t)
        assert torch.equal(as_bits(got), as_bits(ref)), (name, int((as_bits(got) != as_bits(ref)).sum()))


def test_compiled_layer_with_the_cache(lib):
    """torch.compile breaks its graph at the cache's calls, which run as they do without it: same results, also when lengths,
    buffers and batches change between calls."""
    from gemlite_b200 import KVBatch, QuantizedKVCache, rotary_table, tp
    layer = tp.LlamaLinears(512, 1024, 8, 2, 64, 1, 0, DEV, seed=3)
    cs = rotary_table(64, 64, device=DEV)
    compiled = torch.compile(layer, backend="eager")
    caches = [make_cache([40, 9], 2, 64, "fp8", 16, seed=21)[0] for _ in range(2)]
    table = make_cache([40, 9], 2, 64, "fp8", 16, seed=21)[1]
    for i, (ctx, new) in enumerate((([36, 8], [4, 1]), ([30, 2], [1, 1]), ([0, 0], [9, 9]))):
        n = sum(new)
        x = _randn(80 + i, n, 512)
        batch = KVBatch(table, _i32(ctx), _i32([0] + torch.tensor(new).cumsum(0).tolist()))
        pos = torch.cat([torch.arange(c, c + t) for c, t in zip(ctx, new)]).to(DEV)
        with torch.no_grad():
            want = layer(x, caches[0], batch, positions=pos, cos_sin=cs)
            got = compiled(x, caches[1], batch, positions=pos, cos_sin=cs)
        assert torch.equal(got, want)
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8))
        caches[1].k_scales = caches[1].k_scales.clone()
