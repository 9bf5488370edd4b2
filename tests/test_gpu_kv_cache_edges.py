"""GPU: the quantised key/value cache where its numbers and its promises are stretched: scales of zero over long stretches,
what a row does not see, against plain 64-bit forms (tests/kv_util.py)."""
import math

import pytest
import torch

from tests.kv_util import make_cache
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
