"""A paged key/value cache in low bits and the attention that reads it.

The low-bit layers leave decode bound by the bytes of the cache once contexts grow; this module keeps those bytes in
8 or 4 bits.  Three calls make the step between a fused qkv projection and the output projection::

    cache = QuantizedKVCache(num_pages, page_size, n_kv_heads, head_dim, kv_format="fp8", device="cuda:0")
    batch = KVBatch(page_table, ctx_lens, q_offsets, max_new=1)  # which pages, how many tokens cached, which rows are new
    q = cache.write(q, k, v, batch, positions=pos, cos_sin=table, q_norm=wq, k_norm=wk)
    y = cache.attend(q, batch)                                   # or attend(q, batch, mask=tree_mask)

``write`` normalises the heads of queries and keys, rotates them and quantises keys and values into their slots in one
pass; ``attend`` serves single tokens, trees of drafted tokens and chunks of prompts; ``read`` gives plain tensors back.
The reference has no counterpart (its layers end at the projections).

Verified drafts: the accepted tokens' keys and values are still in hand after the step, so a second ``write`` of those
rows (``q=None``) with the old ``ctx_lens`` puts them in order; the codes are the ones the first write made.

The kernels read ``page_table``, ``ctx_lens`` and ``q_offsets`` on the device at run time: a captured graph sees what they
hold when it is replayed.  Nothing is kept between calls and no call synchronises; a workspace comes from torch's
allocator per call, so calls on several streams and captured graphs do not share one.
"""
import ctypes
import math
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .dtypes import DType

KV_FORMATS = {"fp8": 0, "int8": 1, "int4": 2}
_DTYPE_CODES = {torch.float16: DType.FP16.value, torch.bfloat16: DType.BF16.value, torch.float32: DType.FP32.value}
_HALF_CODES = {torch.float16: DType.FP16.value, torch.bfloat16: DType.BF16.value}
_INT32_MAX = 2 ** 31 - 1


def rotary_table(max_positions: int, rot_dim: int, base: float = 10000.0, device="cuda:0") -> Tensor:
    """fp32 [max_positions, rot_dim]: cosines, then sines, of position * base^(-2i / rot_dim).  The angles are formed in
    fp64: at position 100000 an fp32 angle is off by up to 2^-8."""
    if rot_dim <= 0 or rot_dim % 2 != 0:
        raise ValueError("rot_dim must be a positive even number, got %d" % rot_dim)
    freq = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)


def attend_status(device=None, clear: bool = True) -> int:
    """0, unless a bounded wait of the kernel for many rows gave up on `device` since the status was last cleared: the rows
    that it left unfinished are NaN.  Synchronises the current stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    status = ctypes.c_int32()
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(_lib.lib().gl_kv_attend_status(ctypes.byref(status), int(clear), stream))
    return status.value


def _index_tensor(t, what, dim):
    _lib.require_cuda(t, what)
    if t.dtype != torch.int32 or t.dim() != dim or (t.numel() > 0 and t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError("%s must be an int32 tensor of %d dimension(s), contiguous in the last one" % (what, dim))
    return t


class KVBatch:
    """The sequences of one call.

    page_table [B, P] int32: pages of every sequence in order (entries outside the pool, such as -1: no page there).
    ctx_lens [B] int32: tokens that the cache holds of it already.
    q_offsets [B + 1] int32: its new tokens are rows q_offsets[b] .. q_offsets[b + 1] of the call's operands (ascending,
    rows behind the last one belong to nobody); None: the rows divide evenly.
    max_len / max_new: bounds, known to the host, of cached + new and of new tokens per sequence.  They shape launches (with
    q_offsets and without max_new, a batch of decoding sequences goes to the kernel for many rows, at three times the time);
    results change with them only by the kernels' roundings and the order of sums, also where they are too small.
    Default: what the table holds, and all rows.
    """

    def __init__(self, page_table: Tensor, ctx_lens: Tensor, q_offsets: Optional[Tensor] = None,
                 max_len: Optional[int] = None, max_new: Optional[int] = None):
        self.page_table, self.ctx_lens, self.q_offsets = page_table, ctx_lens, q_offsets
        self.max_len = None if max_len is None else max(0, min(int(max_len), _INT32_MAX))
        self.max_new = None if max_new is None else max(0, min(int(max_new), _INT32_MAX))
        self._check()

    def __reduce__(self):
        return type(self), (self.page_table, self.ctx_lens, self.q_offsets, self.max_len, self.max_new)

    def _check(self):
        """Tensors may be replaced: the next call comes here again."""
        page_table, ctx_lens, q_offsets = _index_tensor(self.page_table, "page_table", 2), _index_tensor(self.ctx_lens, "ctx_lens", 1), self.q_offsets
        shape, device = tuple(page_table.shape), page_table.device
        if ctx_lens.shape[0] != shape[0]:
            raise ValueError("ctx_lens has %d entries for %d sequences" % (ctx_lens.shape[0], shape[0]))
        if q_offsets is not None and _index_tensor(q_offsets, "q_offsets", 1).shape[0] != shape[0] + 1:
            raise ValueError("q_offsets must have %d entries (sequences + 1), got %d" % (shape[0] + 1, q_offsets.shape[0]))
        if ctx_lens.device != device or (q_offsets is not None and q_offsets.device != device):
            raise ValueError("page_table, ctx_lens and q_offsets must be on one device")
        self.device, self.shape, self.table_stride = device, shape, page_table.stride(0)
        self._checked = page_table, ctx_lens, q_offsets


class QuantizedKVCache:
    """Pages of quantised keys and values.

    kv_format: "fp8" (e4m3), "int8", one fp32 scale per token and head; "int4": unsigned 4-bit codes with a scale and a
    zero point per token and head, even channel in the low nibble.  Buffers ([num_pages, n_kv_heads, page_size, ...]):
    k_codes, v_codes (uint8), k_scales, v_scales (fp32), k_zeros, v_zeros (uint8, int4 only).  They may be replaced (the next
    call checks them as ``from_buffers`` does); copies and pickles of a cache go by their own buffers.
    """

    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, kv_format: str = "fp8", device="cuda:0"):
        if kv_format not in KV_FORMATS:
            raise ValueError("kv_format must be one of %s, got %r" % (sorted(KV_FORMATS), kv_format))
        if min(num_pages, page_size, n_kv_heads) <= 0:
            raise ValueError("num_pages, page_size and n_kv_heads must be positive")
        shape, row = (num_pages, n_kv_heads, page_size), head_dim // 2 if kv_format == "int4" else head_dim
        new = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
        zeros = (new(*shape, dtype=torch.uint8), new(*shape, dtype=torch.uint8)) if kv_format == "int4" else (None, None)
        self._take(new(*shape, row, dtype=torch.uint8), new(*shape, row, dtype=torch.uint8), new(*shape, dtype=torch.float32),
                   new(*shape, dtype=torch.float32), kv_format, *zeros)

    @classmethod
    def from_buffers(cls, k_codes: Tensor, v_codes: Tensor, k_scales: Tensor, v_scales: Tensor, kv_format: str = "fp8",
                     k_zeros: Optional[Tensor] = None, v_zeros: Optional[Tensor] = None):
        """A cache over existing buffers of the layout above (they are used, not copied)."""
        self = cls.__new__(cls)
        self._take(k_codes, v_codes, k_scales, v_scales, kv_format, k_zeros, v_zeros)
        return self

    def __setattr__(self, name, value):
        if name != "_args":
            object.__setattr__(self, "_args", None)
        object.__setattr__(self, name, value)

    def __reduce__(self):
        return type(self).from_buffers, (self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.kv_format, self.k_zeros, self.v_zeros)

    def _check(self):
        """The buffers are those, and lie where, the last check saw them; else they are checked again."""
        if self._args is None or self._addresses != [at() for at in self._address_of]:
            self._take(self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.kv_format, self.k_zeros, self.v_zeros)

    def _take(self, k_codes, v_codes, k_scales, v_scales, kv_format, k_zeros, v_zeros):
        if kv_format not in KV_FORMATS:
            raise ValueError("kv_format must be one of %s, got %r" % (sorted(KV_FORMATS), kv_format))
        int4 = kv_format == "int4"
        _lib.require_cuda(k_codes, "k_codes")
        if k_codes.dim() != 4:
            raise ValueError("codes must be [num_pages, n_kv_heads, page_size, row], got %s" % (tuple(k_codes.shape),))
        for name, t, dtype, shape in (("k_codes", k_codes, torch.uint8, k_codes.shape), ("v_codes", v_codes, torch.uint8, k_codes.shape),
                                      ("k_scales", k_scales, torch.float32, k_codes.shape[:3]), ("v_scales", v_scales, torch.float32, k_codes.shape[:3]),
                                      ("k_zeros", k_zeros, torch.uint8, k_codes.shape[:3]), ("v_zeros", v_zeros, torch.uint8, k_codes.shape[:3])):
            if name.endswith("zeros") and not int4:
                if t is not None:
                    raise ValueError("%s: only the int4 format has zero points" % name)
                continue
            _lib.require_cuda(t, name)
            if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError("%s must be a contiguous %s tensor of shape %s on %s" % (name, dtype, tuple(shape), k_codes.device))
        self.kv_format, self.device = kv_format, k_codes.device
        self.num_pages, self.n_kv_heads, self.page_size, row = k_codes.shape
        self.head_dim = 2 * row if int4 else row
        if self.head_dim not in (64, 128):
            raise NotImplementedError("head_dim %d (64 and 128 are supported)" % self.head_dim)
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.k_zeros, self.v_zeros = k_zeros, v_zeros
        a = _lib.GLKvArgs()
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_zeros", "v_zeros"):
            setattr(a, name, _lib.ptr(getattr(self, name)))
        a.format, a.num_pages, a.page_size = KV_FORMATS[kv_format], self.num_pages, self.page_size
        a.n_kv_heads, a.head_dim = self.n_kv_heads, self.head_dim
        self._address_of = tuple(t.data_ptr for t in (k_codes, v_codes, k_scales, v_scales, k_zeros, v_zeros) if t is not None)
        self._addresses = [at() for at in self._address_of]
        self._args = bytes(a)

    # -- argument plumbing (a decode step makes these calls once per layer: what they cost the host counts) ----------------------
    def _on_device(self, t, what):
        if not isinstance(t, Tensor) or t.device != self.device:
            _lib.require_cuda(t, what)
            raise ValueError("%s is on %s, the cache on %s" % (what, t.device, self.device))
        return t

    def _rows(self, x, what, heads=None):
        """(tensor, address, token stride, head stride, tokens, heads) of a [tokens, heads, head_dim] operand; copied only
        where the kernels could not read it with 16-byte loads."""
        self._on_device(x, what)
        if x.dtype not in _HALF_CODES:
            raise NotImplementedError("%s must be float16 or bfloat16, got %s" % (what, x.dtype))
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError("%s must be [tokens, %s, %d], got %s" % (what, "heads" if heads is None else heads, self.head_dim, tuple(shape)))
        n, h, _ = shape
        sn, sh, sd = x.stride()
        if n <= 1:
            sn = 0
        if h == 1:
            sh = 0
        at = x.data_ptr()
        if sd != 1 or (sn | sh) & 7 or at & 15:
            x = x.clone(memory_format=torch.contiguous_format)
            at, sn, sh = x.data_ptr(), h * self.head_dim, self.head_dim
        return x, at, sn, sh, n, h

    def _batch_args(self, batch, n):
        page_table, ctx_lens, q_offsets = batch._checked
        if batch.page_table is not page_table or batch.ctx_lens is not ctx_lens or batch.q_offsets is not q_offsets:
            batch._check()
            page_table, ctx_lens, q_offsets = batch._checked
        if batch.device != self.device:
            raise ValueError("the batch is on %s, the cache on %s" % (batch.device, self.device))
        a = _lib.GLKvArgs.from_buffer_copy(self._args)
        B, P = batch.shape
        a.page_table, a.page_table_stride, a.lens = page_table.data_ptr(), batch.table_stride, ctx_lens.data_ptr()
        if q_offsets is not None:
            a.q_offsets = q_offsets.data_ptr()
            a.max_new = n if batch.max_new is None else batch.max_new
        elif B > 0:
            if n % B != 0:
                raise ValueError("%d rows do not divide evenly over %d sequences; give the batch q_offsets" % (n, B))
            a.max_new = n // B if batch.max_new is None else batch.max_new
        a.batch, a.max_pages, a.n_tokens = B, P, n
        a.max_len = min(P * self.page_size, _INT32_MAX) if batch.max_len is None else batch.max_len
        return a

    def _call(self, fn, a):
        index = self.device.index
        if torch._C._cuda_getDevice() == index:
            status = fn(ctypes.byref(a), _lib.current_stream_ptr(self.device))
        else:
            with torch.cuda.device(index):
                status = fn(ctypes.byref(a), _lib.current_stream_ptr(self.device))
        if status:
            _lib.check(status)

    # -- operators -----------------------------------------------------------------------------------------------------
    def write(self, q: Optional[Tensor], k: Tensor, v: Tensor, batch: KVBatch, positions: Optional[Tensor] = None,
              cos_sin: Optional[Tensor] = None, q_norm: Optional[Tensor] = None, k_norm: Optional[Tensor] = None,
              eps: float = 1e-6, interleaved: bool = False) -> Optional[Tensor]:
        """Head norms and rotation of queries and keys, and keys and values into the slots behind each sequence's
        ``ctx_lens`` tokens; returns the queries [tokens, heads, head_dim] (None for ``q=None``).

        q / k / v [tokens, heads, head_dim] fp16 or bf16 (views of a fused projection's output are read in place).
        q_norm / k_norm [head_dim]: weights of x / sqrt(mean x^2 + eps) * w, or None.  cos_sin: fp32 [rows, rot_dim] as
        ``rotary_table`` makes it, rotating the first rot_dim channels (a multiple of 16) by row positions[n]: pairs
        (i, i + rot_dim / 2), or (2i, 2i + 1) with ``interleaved``; None: no rotation.

        Arithmetic is fp32 and rounded once.  A row (one token's head) with an infinity or NaN is stored as codes 0 with the
        scale NaN.  A position outside the table gives NaN queries and such a key row.  Tokens whose page does not exist are
        dropped.  A page must not be written for two sequences, or twice for one, in a call.  Rows of the result that belong to no
        sequence are not written."""
        self._check()
        k, k_at, ksn, ksh, n, _ = self._rows(k, "k", self.n_kv_heads)
        v, v_at, vsn, vsh, vn, _ = self._rows(v, "v", self.n_kv_heads)
        dtype = k.dtype
        if vn != n or v.dtype != dtype:
            raise ValueError("k and v must have the same tokens and dtype")
        a = self._batch_args(batch, n)
        a.k, a.k_stride_n, a.k_stride_h, a.v, a.v_stride_n, a.v_stride_h = k_at, ksn, ksh, v_at, vsn, vsh
        a.x_dtype = _HALF_CODES[dtype]
        out = None
        if q is not None:
            q, q_at, qsn, qsh, qn, qh = self._rows(q, "q")
            if qn != n or q.dtype != dtype:
                raise ValueError("q and k must have the same tokens and dtype")
            out = q.new_empty((n, qh, self.head_dim))
            a.q, a.q_stride_n, a.q_stride_h, a.n_q_heads, a.out = q_at, qsn, qsh, qh, out.data_ptr()
        keep = []
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None:
                self._on_device(w, name)
                if w.shape != (self.head_dim,) or w.dtype not in _DTYPE_CODES:
                    raise ValueError("%s must be a float tensor of %d weights" % (name, self.head_dim))
                if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
                    w = w.float()
                w = w.contiguous()
                keep.append(w)
                setattr(a, name, w.data_ptr())
                a.norm_dtype = _DTYPE_CODES[w.dtype]
        a.eps, a.interleaved = eps, int(interleaved)
        if cos_sin is not None:
            self._on_device(cos_sin, "cos_sin")
            if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.shape[0] > _INT32_MAX:
                raise ValueError("cos_sin must be a contiguous float32 tensor [positions, rot_dim]")
            if cos_sin.shape[1] % 16 != 0 or not 0 < cos_sin.shape[1] <= self.head_dim:
                raise ValueError("rot_dim must be a multiple of 16 up to head_dim, got %d" % cos_sin.shape[1])
            if positions is None or positions.shape != (n,):
                raise ValueError("the rotation needs positions of shape (%d,)" % n)
            self._on_device(positions, "positions")
            if positions.dtype == torch.int64:
                positions = positions.clamp(-1, _INT32_MAX).to(torch.int32)
            if positions.dtype != torch.int32:
                raise ValueError("positions must be int32 or int64, got %s" % positions.dtype)
            positions = positions.contiguous()
            if cos_sin.data_ptr() & 15:
                cos_sin = cos_sin.clone()
            a.cos_sin, a.positions, a.rot_dim, a.table_rows = cos_sin.data_ptr(), positions.data_ptr(), cos_sin.shape[1], cos_sin.shape[0]
            if a.table_rows == 0:
                raise ValueError("cos_sin has no rows")
        if n > 0 and a.batch > 0:
            self._call(_lib.lib().gl_kv_write, a)
        return out

    def read(self, page_table: Tensor, lens: Tensor, max_len: Optional[int] = None, out_dtype: torch.dtype = torch.bfloat16):
        """(keys, values) [B, max_len, n_kv_heads, head_dim] of the first lens[b] tokens of every sequence, zeros behind them
        and where a page does not exist.  max_len defaults to what the table holds; longer sequences are cut there."""
        if out_dtype not in _DTYPE_CODES:
            raise NotImplementedError("out_dtype %s is not supported" % out_dtype)
        self._check()
        batch = KVBatch(page_table, lens)
        a = self._batch_args(batch, 0)
        if max_len is not None:
            if not 0 <= max_len <= _INT32_MAX:
                raise ValueError("max_len %d" % max_len)
            a.max_len = max_len
        shape = (a.batch, a.max_len, self.n_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=out_dtype, device=self.device)
        v = torch.empty(shape, dtype=out_dtype, device=self.device)
        a.out, a.out_v, a.x_dtype = k.data_ptr(), v.data_ptr(), _DTYPE_CODES[out_dtype]
        if k.numel() > 0:
            self._call(_lib.lib().gl_kv_read, a)
        return k, v

    def attend(self, q: Tensor, batch: KVBatch, mask: Optional[Tensor] = None, scale: Optional[float] = None,
               out: Optional[Tensor] = None, kernel_override: int = 0) -> Tensor:
        """softmax(scale * q K^T) V over the cache: every query sees the ``ctx_lens`` cached tokens of its sequence, and of
        the sequence's new tokens (written before this call) the ones its row of ``mask`` names.

        q [tokens, heads, head_dim] fp16 or bf16, heads a multiple of n_kv_heads.  mask: bool or uint8 [tokens, W], column j
        = the sequence's j-th new token (a tree's ancestor mask; columns that are not there count as False); None: the
        new tokens up to the query's own (single tokens, prompt chunks).  A row that sees nothing gives zeros; what a row does not
        see has no influence on it, whatever those slots hold.  scale defaults to 1 / sqrt(head_dim).
        Result like q (contiguous); rows that belong to no sequence are not written."""
        self._check()
        q, at, sn, sh, n, h = self._rows(q, "q")
        if h == 0 or h % self.n_kv_heads != 0:
            raise ValueError("%d query heads do not divide over %d kv heads" % (h, self.n_kv_heads))
        if out is None:
            out = q.new_empty((n, h, self.head_dim))
        else:
            self._on_device(out, "out")
            if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() & 15:
                raise ValueError("out must be a contiguous, 16-byte aligned %s tensor of shape %s" % (q.dtype, tuple(q.shape)))
        a = self._batch_args(batch, n)
        a.q, a.q_stride_n, a.q_stride_h, a.n_q_heads, a.out, a.x_dtype = at, sn, sh, h, out.data_ptr(), _HALF_CODES[q.dtype]
        a.softmax_scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        a.kernel_override = kernel_override
        if mask is not None:
            self._on_device(mask, "mask")
            if mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 or mask.shape[0] != n:
                raise ValueError("mask must be a bool or uint8 tensor [%d, new tokens], got %s %s" % (n, mask.dtype, tuple(mask.shape)))
            if mask.stride(1) != 1 and mask.shape[1] > 1:
                mask = mask.contiguous()
            if mask.numel() == 0:                      # no columns: the cached tokens only
                mask = torch.zeros((n, 1), dtype=torch.uint8, device=self.device)
            a.mask, a.mask_stride, a.mask_cols = mask.data_ptr(), mask.stride(0), mask.shape[1]
        if n == 0 or a.batch == 0:
            return out
        L = _lib.lib()
        if torch._C._cuda_getDevice() == self.device.index:
            self._attend(L, a)
        else:
            with torch.cuda.device(self.device.index):
                self._attend(L, a)
        return out

    def _attend(self, L, a):
        at = ctypes.byref(a)
        need = L.gl_kv_attend_workspace_bytes(at)
        if need:
            ws = self.k_codes.new_empty(need)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        status = L.gl_kv_attend(at, _lib.current_stream_ptr(self.device))
        if status:
            _lib.check(status)
