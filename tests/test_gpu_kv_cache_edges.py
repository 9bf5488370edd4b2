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
