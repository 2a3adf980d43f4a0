"""
8-bit operands with block scales, the matrix product of two of them, and the join of a block with its residual stream
(sugar_fp8_quant / sugar_fp8_dequant / sugar_fp8_linear / sugar_block_join of include/sugar_amd.h):

    w = quantize_block_fp8(weight)                              # [out, in] -> BlockFP8, once
    a = quantize_block_fp8(rows)                                # [R, in] float32 / bfloat16
    y = block_fp8_linear(a, w, scale=s, shift=t, relu=True)     # relu(a @ w.T) * s + t, [R, out]
    j = block_join(u, residual, gate=g, row_off=off, post=RowNorm("rms", w1), pre=RowNorm("rms", w2), quantized=True)
    y = block_fp8_linear(j.quantized, w)                        # the next block's first product

The precision "fp8" of the embedding path runs on the same kernels.  Calls run on the current stream of the tensors'
device, allocate only their outputs (none when they are passed in) and never synchronise, so they can be captured into a
graph; there is no backward pass: tensors that require a gradient are refused while gradients are recorded, and so are the
dual tensors of forward-mode differentiation.
"""
import collections
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

_DT = {torch.float32: _lib.SUGAR_F32, torch.bfloat16: _lib.SUGAR_BF16}
NORMS = {"affine": 1, "rms": 2, "layer": 3}
MAX_JOIN_COLS = 8192
MAX_COLS = 1 << 24                                     # channels of an operand, outputs of a product (32-bit integers at the C ABI)
F32_MAX, INF = torch.finfo(torch.float32).max, float("inf")
# (torch.cuda.current_stream builds an object, torch.cuda.current_device looks whether the GPU is initialised: 1.3 us of a 10 us call)
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_FN = {}


def _up(v, m):
    return (v + m - 1) // m * m


def _gpu(dev):
    if dev.type != "cuda":
        raise _lib.SugarError("sugar_amd runs on an MI355X only: tensors must be CUDA tensors (no CPU fallback)")
    return dev


def _has_tangent(t):
    """Whether t is a dual tensor of forward-mode differentiation (its requires_grad is False, torch.no_grad() does not matter)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _same_device(dev, tensors):
    """All on `dev` (a GPU), none of them part of a recorded gradient or of a forward derivative."""
    _gpu(dev)
    for t in tensors:
        if t.device != dev:
            raise ValueError("tensors on %s and %s" % (dev, t.device))
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("no backward pass: call under torch.no_grad() or detach the inputs")
    if forward_ad._current_level >= 0 and any(_has_tangent(t) for t in tensors):
        raise ValueError("no forward derivative: a dual tensor; pass its primal (torch.autograd.forward_ad.unpack_dual)")


def _call(dev, name, *args):
    """One library call on the current stream of `dev`, with that device current."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_lib.lib(), name)
    idx = dev.index
    if _current_device() == idx:
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc < 0:
        _lib.check(rc, name)


def _rows(what, x):
    """x as a matrix whose columns lie next to each other (a copy when they do not), its rows, columns, row stride, type."""
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError("%s: expected [rows, columns], got %s" % (what, tuple(shape)))
    rows, cols = shape
    dtype = _DT.get(x.dtype)
    if dtype is None:
        raise ValueError("%s: dtype %s not in %s" % (what, x.dtype, [str(d) for d in _DT]))
    if cols >= MAX_COLS:
        raise ValueError("%s: %d columns, fewer than %d are taken" % (what, cols, MAX_COLS))
    ld, step = x.stride()
    if step != 1 or ld < cols:                          # (all but the plain case)
        x = x.resolve_neg()                             # (one column of z.conj().imag: the memory holds the values negated)
        ld = _row_stride(x)
        if ld is None:
            x, ld = x.contiguous(), cols
    return x, rows, cols, ld, dtype


def _row_stride(x):
    """Elements from row to row of a matrix with adjacent columns, None for any other (a single row has no stride of its own:
    torch leaves any number there)."""
    r, c = x.shape
    ld, step = x.stride()
    if step != 1 and c != 1:
        return None
    if r <= 1:
        return max(c, ld)
    return ld if ld >= c else None


def _out(what, out, shape, dtypes, dev):
    """Row stride of a tensor to write into."""
    if out.requires_grad and torch.is_grad_enabled() or _has_tangent(out):
        raise ValueError("%s: an output that requires a gradient, or a dual tensor" % what)
    if tuple(out.shape) != tuple(shape) or out.dtype not in dtypes or out.device != dev:
        raise ValueError("%s: expected %s %s on %s, got %s %s on %s" % (what, tuple(shape), "/".join(str(d) for d in dtypes), dev,
                                                                        tuple(out.shape), out.dtype, out.device))
    ld = _row_stride(out)
    if ld is None or out.is_neg():
        raise ValueError("%s: the columns of an output must be contiguous, its rows apart, its values not a negated view" % what)
    return ld


def _span(t, ld=0):
    """(first byte, bytes of a row, bytes from row to row, rows) of a matrix with row stride `ld`, or of a vector."""
    shape, size = t.shape, t.element_size()
    if len(shape) == 1:
        return t.data_ptr(), shape[0] * size, 0, 1
    return t.data_ptr(), shape[1] * size, ld * size, shape[0]


def _apart(what, out, others, itself=()):
    """The memory of an output that was passed in (a _span) must not be that of anything else a call reads or writes, save
    exactly that of one of `itself`.  Column slices of one buffer are apart."""
    p, width, step, rows = out
    end = p + (rows - 1) * step + width
    for other in others:
        q, w, st, r = other
        if q >= end or p >= q + (r - 1) * st + w or not rows or not r:
            continue
        if st == step and step:
            off = (q - p) % step
            if off >= width and off + w <= step:
                continue
        if other == out and other in itself:
            continue
        raise ValueError("%s: the output shares memory with another operand" % what)


def _vector(what, v, n):
    """A contiguous float32 vector of n (other float types and strides are converted)."""
    if v.dtype is torch.float32 and v.shape == (n,) and v.is_contiguous() and not (n == 1 and v.is_neg()):
        return v
    if v.dim() != 1 or v.shape[0] != n or not v.dtype.is_floating_point:
        raise ValueError("%s: expected a floating vector of %d, got %s %s" % (what, n, v.dtype, tuple(v.shape)))
    return v.resolve_neg().to(torch.float32).contiguous()


class BlockFP8(object):
    """
    [rows, cols] in 8 bits: value[r, c] = data[r, c] * 2^(exponent[r, c // 128] - 127).
      data      float8_e4m3fn [rows, >= round_up(cols, 128)], zeros from column `cols` on; rows 16-byte aligned
      exponent  uint8 [rows, >= round_up(blocks, 4)], blocks = ceil(cols / 128); rows 4-byte aligned; 255 stands for NaN
    Row slices (`x[10:20]`) share the memory.  `BlockFP8(data, exponent, cols)` takes existing tensors as they are.
    """
    BLOCK = 128
    __slots__ = ("_data", "_exponent", "_buf", "rows", "cols", "_ld", "_lde")

    def __init__(self, data, exponent, cols):
        cols = int(cols)
        blocks = -(-cols // self.BLOCK)
        if data.dim() != 2 or data.dtype != torch.float8_e4m3fn or exponent.dim() != 2 or exponent.dtype != torch.uint8:
            raise ValueError("BlockFP8: data float8_e4m3fn [rows, n], exponent uint8 [rows, n]; got %s %s, %s %s"
                             % (data.dtype, tuple(data.shape), exponent.dtype, tuple(exponent.shape)))
        if not 1 <= cols < MAX_COLS or data.shape[1] < blocks * self.BLOCK or exponent.shape[1] < _up(blocks, 4) or data.shape[0] != exponent.shape[0]:
            raise ValueError("BlockFP8: %d columns need data [rows, >= %d] and exponent [rows, >= %d], got %s and %s"
                             % (cols, blocks * self.BLOCK, _up(blocks, 4), tuple(data.shape), tuple(exponent.shape)))
        if data.device != exponent.device:
            raise ValueError("BlockFP8: data on %s, exponent on %s" % (data.device, exponent.device))
        if data.requires_grad or _has_tangent(data):
            raise ValueError("BlockFP8: no backward pass, no forward derivative: detach the data, take the primal")
        ld, lde = _row_stride(data), _row_stride(exponent)
        if ld is None or lde is None or ld % 16 or lde % 4 or data.data_ptr() % 16 or exponent.data_ptr() % 4:
            raise ValueError("BlockFP8: contiguous columns, data rows 16-byte aligned, exponent rows 4-byte aligned")
        self._data, self._exponent, self._buf = data, exponent, None
        self.rows, self.cols, self._ld, self._lde = data.shape[0], cols, ld, lde

    @classmethod
    def empty(cls, rows, cols, device):
        """An operand to be written into: one allocation, values and exponents one behind the other."""
        self = cls.__new__(cls)
        blocks = (cols + 127) >> 7
        self.rows, self.cols, self._ld, self._lde = rows, cols, blocks << 7, (blocks + 3) & -4
        self._buf = torch.empty(rows * (self._ld + self._lde), dtype=torch.uint8, device=device)
        self._data = self._exponent = None
        return self

    def _pointers(self):
        if self._buf is None:
            return self._data.data_ptr(), self._exponent.data_ptr()
        p = self._buf.data_ptr()
        return p, p + self.rows * self._ld

    def _spans(self):
        """_span of the values and of the exponents."""
        d, e = self._pointers()
        return [(d, self._ld if self._buf is not None else self._data.shape[1], self._ld, self.rows),
                (e, self._lde if self._buf is not None else self._exponent.shape[1], self._lde, self.rows)]

    def _split(self):
        n = self.rows * self._ld
        self._data = self._buf[:n].view(torch.float8_e4m3fn).view(self.rows, self._ld)
        self._exponent = self._buf[n:].view(self.rows, self._lde)

    @property
    def data(self):
        if self._data is None:
            self._split()
        return self._data

    @property
    def exponent(self):
        if self._exponent is None:
            self._split()
        return self._exponent

    @property
    def device(self):
        return (self._data if self._buf is None else self._buf).device

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    def __getitem__(self, rows):
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise ValueError("BlockFP8: only slices of consecutive rows")
        return BlockFP8(self.data[rows], self.exponent[rows], self.cols)

    def dequantize(self, dtype=torch.float32, out=None):
        """The values, [rows, cols] float32 or bfloat16 (exact in both down to the type's subnormals: an e4m3 value has 4 bits)."""
        rows, cols = self.rows, self.cols
        dev = _gpu(self.device)
        if out is None:
            if dtype not in _DT:
                raise ValueError("dequantize: dtype %s not in %s" % (dtype, [str(d) for d in _DT]))
            out, ld = torch.empty(rows, cols, dtype=dtype, device=dev), cols
        else:
            ld = _out("dequantize", out, (rows, cols), _DT, dev)
            _apart("dequantize", _span(out, ld), self._spans())
        if rows:
            d, e = self._pointers()
            _call(dev, "sugar_fp8_dequant", d, self._ld, e, self._lde, rows, cols, out.data_ptr(), ld, _DT[out.dtype])
        return out


def _fp8_out(what, out, rows, cols, dev):
    if out is None:
        return BlockFP8.empty(rows, cols, dev)
    if not isinstance(out, BlockFP8) or out.rows != rows or out.cols != cols or out.device != dev:
        raise ValueError("%s: expected a BlockFP8 of [%d, %d] on %s" % (what, rows, cols, dev))
    if out._buf is None:
        data, exponent = out._spans()
        _apart(what, data, (exponent,))
    return out


def quantize_block_fp8(x, out=None):
    """
    [rows, cols] float32 / bfloat16 on the GPU -> BlockFP8.  Every block of 128 columns gets the smallest power of two that
    keeps its largest finite magnitude within 448; values go to the nearest e4m3, ties to the even one.  Infinities and NaN
    become NaN and do not move the scale of their block.
    """
    x, rows, cols, ld, dtype = _rows("quantize_block_fp8", x)
    dev = x.device
    _same_device(dev, (x,))
    q = _fp8_out("quantize_block_fp8", out, rows, cols, dev)
    if out is not None:
        _apart("quantize_block_fp8", _span(x, ld), q._spans())
    if rows:
        d, e = q._pointers()
        _call(dev, "sugar_fp8_quant", x.data_ptr(), ld, dtype, rows, cols, d, q._ld, e, q._lde)
    return q


def block_fp8_linear(a, w, scale=None, shift=None, relu=False, out_dtype=torch.bfloat16, out=None):
    """
    relu(a @ w.T) * scale + shift for BlockFP8 a [rows, k] and w [n, k], rounded once to `out_dtype` (bfloat16 or float32).
    float32 outputs are float32 sums of exact products.  bfloat16 outputs run twice as fast on the 8-bit matrix instruction:
    of every 8 neighbouring products it cuts off what lies 2^-13 below the largest of them, 1.5e-5 of the result in the 2-norm on
    random operands, more of a sum that cancels (include/sugar_amd.h); ask for float32 where that matters.  The order is that of
    the reference's layers, conv -> ReLU -> BatchNorm (sugar/models/dynamictdnn.py:183); scale, shift: float vectors [n], either
    may be missing.
    """
    if not isinstance(a, BlockFP8) or not isinstance(w, BlockFP8):
        raise ValueError("block_fp8_linear: operands must be BlockFP8 (quantize_block_fp8)")
    rows, n, k = a.rows, w.rows, a.cols
    if k != w.cols:
        raise ValueError("block_fp8_linear: a has %d columns, w %d" % (k, w.cols))
    if not 0 < n < MAX_COLS:
        raise ValueError("block_fp8_linear: w has %d rows, 1 .. %d are taken" % (n, MAX_COLS - 1))
    dev = a.device
    if w.device != dev:
        raise ValueError("tensors on %s and %s" % (dev, w.device))
    _gpu(dev)
    flags, sp, tp = _lib.EPI_RELU if relu else 0, None, None
    if scale is not None or shift is not None:
        _same_device(dev, [t for t in (scale, shift) if t is not None])
        flags |= _lib.EPI_AFFINE
        if scale is not None:
            scale = _vector("scale", scale, n)
            sp = scale.data_ptr()
        if shift is not None:
            shift = _vector("shift", shift, n)
            tp = shift.data_ptr()
    if out is None:
        if out_dtype not in _DT:
            raise ValueError("block_fp8_linear: out_dtype %s not in %s" % (out_dtype, [str(d) for d in _DT]))
        out, ld = torch.empty(rows, n, dtype=out_dtype, device=dev), n
    else:
        ld = _out("block_fp8_linear", out, (rows, n), _DT, dev)
        _apart("block_fp8_linear", _span(out, ld), a._spans() + w._spans() + [_span(t) for t in (scale, shift) if t is not None])
    if rows:
        (ap, aep), (wp, wep) = a._pointers(), w._pointers()
        _call(dev, "sugar_fp8_linear", ap, a._ld, aep, a._lde, rows, wp, w._ld, wep, w._lde, n, k, sp, tp, flags,
              out.data_ptr(), ld, _DT[out.dtype])
    return out


class RowNorm(object):
    """
    A norm over the channels of a row: kind "rms" (x / sqrt(mean x^2 + eps)), "layer" ((x - mean) / sqrt(var + eps)) or
    "affine" (x itself: a folded BatchNorm), times `weight`, plus `bias` (float vectors, or None).  The vectors are used as
    they are where they are contiguous float32 (later changes in place count), else converted once, here.
    """
    __slots__ = ("kind", "weight", "bias", "eps", "code", "cols")

    def __init__(self, kind, weight=None, bias=None, eps=1e-5):
        if kind not in NORMS:
            raise ValueError("RowNorm: kind %r not in %s" % (kind, sorted(NORMS)))
        if not 0 <= eps <= F32_MAX:
            raise ValueError("RowNorm: eps %r is no finite float32 >= 0" % (eps,))
        self.kind, self.eps, self.code, self.cols = kind, float(eps), NORMS[kind], None
        for v in (weight, bias):
            if v is not None:
                if v.dim() != 1 or self.cols not in (None, v.shape[0]):
                    raise ValueError("RowNorm: weight and bias must be vectors of one length, got %s"
                                     % [None if t is None else tuple(t.shape) for t in (weight, bias)])
                self.cols = v.shape[0]
        self.weight = None if weight is None else _vector("RowNorm: weight", weight, self.cols)
        self.bias = None if bias is None else _vector("RowNorm: bias", bias, self.cols)


JoinResult = collections.namedtuple("JoinResult", "stream normed quantized")


def block_join(u, residual, post=None, gate=None, row_off=None, alpha=1.0, dense=False, pre=None, normed=True,
               quantized=False, out_dtype=None, stream_out=None, normed_out=None, quantized_out=None):
    """
    The end of one block and the beginning of the next, in one pass over [rows, C]:

        v = post(u);  s = residual + alpha * gate * v;  stream = s  (residual + s when `dense`);  z = pre(s)

    u [rows, C] bfloat16 / float32, residual the same or, under a bfloat16 u, float32; post / pre: RowNorm or None;
    gate: None, [C], one row per utterance [B, C] with row_off (int32 [B + 1] on the GPU; the squeeze-excite gate of
    sugar/models/dynamictdnn.py:94-100), or [rows, C] in u's dtype.  Arithmetic is float32, each output is rounded once.
    `dense` is the running sum of DynamicTDNN.forward (:657-660).  Returns (stream, normed, quantized): stream in
    residual's dtype, normed = z in out_dtype (default u's) unless normed=False, quantized = z as BlockFP8 if asked for.
    Outputs may be passed in; stream_out may be `residual` or `u` itself, normed_out `u` (in place), any other shared memory
    is refused.  With row_off, rows in front of the first and behind the last utterance are left as they are (in outputs
    allocated here: undefined).  alpha is a number of the host, passed by value (a captured graph keeps it).
    """
    u, rows, cols, ldu, u_dtype = _rows("block_join: u", u)
    residual, r_rows, r_cols, ldr, r_dtype = _rows("block_join: residual", residual)
    if r_rows != rows or r_cols != cols:
        raise ValueError("block_join: u %s, residual %s" % (tuple(u.shape), tuple(residual.shape)))
    if cols > MAX_JOIN_COLS:
        raise ValueError("block_join: %d columns, at most %d" % (cols, MAX_JOIN_COLS))
    if u_dtype == _lib.SUGAR_F32 != r_dtype:
        raise ValueError("block_join: a float32 u needs a float32 residual")
    if isinstance(alpha, torch.Tensor) or (abs(alpha) > F32_MAX and abs(alpha) != INF):
        raise ValueError("block_join: alpha %r is no float32 number" % (alpha,))
    dev = u.device
    inputs = [residual, u]                             # and the norms' vectors, then what else comes in
    post_kind = pre_kind = post_w = post_b = pre_w = pre_b = 0
    post_eps = pre_eps = 0.0
    if post is not None:
        post_kind, post_eps, post_w, post_b = _norm("post", post, cols, inputs)
    if pre is not None:
        pre_kind, pre_eps, pre_w, pre_b = _norm("pre", pre, cols, inputs)
    n_vectors = len(inputs)
    if gate is not None:
        inputs.append(gate)
    if row_off is not None:
        inputs.append(row_off)
    _same_device(dev, inputs)
    utts = off_ptr = gate_kind = ldg = gate_ptr = 0
    if row_off is not None:
        if row_off.dim() != 1 or row_off.shape[0] < 2 or row_off.dtype != torch.int32:
            raise ValueError("block_join: row_off must be int32 [B + 1], got %s %s" % (row_off.dtype, tuple(row_off.shape)))
        row_off = row_off.contiguous()
        utts, off_ptr = row_off.shape[0] - 1, row_off.data_ptr()
    if gate is not None:
        if gate.dim() == 1:
            gate, gate_kind, ldg = _vector("gate", gate, cols), 1, cols
        elif row_off is not None and tuple(gate.shape) == (utts, cols):
            gate, _, _, ldg, _ = _rows("block_join: gate", gate if gate.dtype == torch.float32 else gate.float())
            gate_kind = 2
        elif row_off is None and gate.shape == u.shape and gate.dtype == u.dtype:
            gate, _, _, ldg, _ = _rows("block_join: gate", gate)
            gate_kind = 3
        else:
            raise ValueError("block_join: gate %s %s is neither [C], [B, C] with row_off, nor [rows, C] of u's dtype without it"
                             % (gate.dtype, tuple(gate.shape)))
        gate_ptr = gate.data_ptr()
    if stream_out is None:
        stream, lds = _like(residual, residual.dtype, rows, cols, dev), cols
    else:
        stream, lds = stream_out, _out("block_join: stream_out", stream_out, (rows, cols), (residual.dtype,), dev)
    z = q = None
    z_ptr = ldz = z_dtype = q_ptr = e_ptr = ldq = lde = 0
    if normed_out is not None:
        z, ldz = normed_out, _out("block_join: normed_out", normed_out, (rows, cols), _DT, dev)
    elif normed:
        out_dtype = u.dtype if out_dtype is None else out_dtype
        if out_dtype not in _DT:
            raise ValueError("block_join: out_dtype %s not in %s" % (out_dtype, [str(t) for t in _DT]))
        z, ldz = _like(u, out_dtype, rows, cols, dev), cols
    if z is not None:
        z_ptr, z_dtype = z.data_ptr(), _DT[z.dtype]
    if quantized or quantized_out is not None:
        q = _fp8_out("block_join: quantized_out", quantized_out, rows, cols, dev)
        (q_ptr, e_ptr), ldq, lde = q._pointers(), q._ld, q._lde
    if stream_out is not None or normed_out is not None or quantized_out is not None:
        su, sr, out = _span(u, ldu), _span(residual, ldr), _span(stream, lds)
        # read where they are written (an output may be u or residual itself), or by rows that others write
        own, shared = [su, sr], [_span(t) for t in [row_off] + inputs[2:n_vectors] if t is not None]
        if gate is not None:
            (own if gate_kind == 3 else shared).append(_span(gate, ldg))
        parts = [] if q is None else q._spans()
        _apart("block_join: stream_out", out, shared + parts)
        _apart("block_join: stream_out", out, own, (sr, su) if u_dtype == r_dtype else (sr,))
        if z is not None:
            sz = _span(z, ldz)
            _apart("block_join: normed_out", sz, [out] + shared + parts)
            _apart("block_join: normed_out", sz, own, (su,) if z_dtype == u_dtype else ())
        for span in parts:
            _apart("block_join: quantized_out", span, own + shared)
    if rows:
        _call(dev, "sugar_block_join", _JOIN.pack(
            rows, cols, utts, u_dtype, r_dtype, z_dtype, post_kind, pre_kind, gate_kind, 1 if dense else 0, alpha, post_eps, pre_eps,
            ldu, ldr, ldg, lds, ldz, ldq, lde, u.data_ptr(), residual.data_ptr(), post_w, post_b, pre_w, pre_b, gate_ptr, off_ptr,
            stream.data_ptr(), z_ptr, q_ptr, e_ptr))
    return JoinResult(stream, z, q)


# SugarBlockJoin of include/sugar_amd.h (_lib.SugarBlockJoin) as one packing: 30 attribute writes of a ctypes structure
# cost 5 us a call
_JOIN = struct.Struct("@q9i3f7q12P")


def _norm(side, p, cols, inputs):
    """(kind, eps, weight pointer, bias pointer) of a RowNorm, whose vectors join the inputs to be checked."""
    if not isinstance(p, RowNorm):
        raise ValueError("block_join: %s must be a RowNorm, got %r" % (side, p))
    if p.cols is not None and p.cols != cols:
        raise ValueError("block_join: the vectors of %s have %d entries, rows %d" % (side, p.cols, cols))
    w, b = p.weight, p.bias
    if w is not None:
        inputs.append(w)
    if b is not None:
        inputs.append(b)
    return p.code, p.eps, 0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr()


def _like(x, dtype, rows, cols, dev):
    """A new contiguous [rows, cols] (empty_like is the cheaper call)."""
    return torch.empty_like(x) if x.dtype == dtype and x.is_contiguous() else torch.empty(rows, cols, dtype=dtype, device=dev)
