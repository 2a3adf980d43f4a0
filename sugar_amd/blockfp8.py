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
graph; there is no backward pass: tensors that require a gradient are refused while gradients are recorded.
"""
import collections
import ctypes as C

import torch

from . import _lib

_DT = {torch.float32: _lib.SUGAR_F32, torch.bfloat16: _lib.SUGAR_BF16}
NORMS = {None: 0, "affine": 1, "rms": 2, "layer": 3}
MAX_JOIN_COLS = 8192


def _up(v, m):
    return (v + m - 1) // m * m


def _need_cuda(*tensors):
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise _lib.SugarError("sugar_amd runs on an MI355X only: tensors must be CUDA tensors (no CPU fallback)")
        if t.device != dev:
            raise ValueError("tensors on %s and %s" % (dev, t.device))
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("no backward pass: call under torch.no_grad() or detach the inputs")
    return dev


def _call(dev, name, *args):
    """One library call on the current stream of `dev`, with that device current."""
    fn = getattr(_lib.lib(), name)
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc < 0:
        _lib.check(rc, name)


def _rows(what, x, dtypes=_DT):
    """x as a matrix whose columns lie next to each other (a copy when they do not)."""
    if x.dim() != 2:
        raise ValueError("%s: expected [rows, columns], got %s" % (what, tuple(x.shape)))
    if x.dtype not in dtypes:
        raise ValueError("%s: dtype %s not in %s" % (what, x.dtype, [str(d) for d in dtypes]))
    if x.shape[1] == 0:
        raise ValueError("%s: no columns" % what)
    return x if _plain(x) else x.contiguous()


def _plain(x):
    return (x.stride(1) == 1 or x.shape[1] == 1) and (x.stride(0) >= x.shape[1] or x.shape[0] <= 1)


def _ld(x):
    """Row stride (a single row has none of its own: torch leaves any number there)."""
    return x.stride(0) if x.shape[0] > 1 else max(x.shape[1], x.stride(0))


def _out(what, out, shape, dtypes, dev):
    if tuple(out.shape) != tuple(shape) or out.dtype not in dtypes or out.device != dev:
        raise ValueError("%s: expected %s %s on %s, got %s %s on %s" % (what, tuple(shape), "/".join(str(d) for d in dtypes), dev,
                                                                        tuple(out.shape), out.dtype, out.device))
    if not _plain(out):
        raise ValueError("%s: the columns of an output must be contiguous" % what)
    return out


def _vector(what, v, n, dev):
    """A float32 vector of n on the device (other float types and strides are converted)."""
    if v is None:
        return None
    if v.dim() != 1 or v.shape[0] != n or not v.dtype.is_floating_point:
        raise ValueError("%s: expected a floating vector of %d, got %s %s" % (what, n, v.dtype, tuple(v.shape)))
    return v if v.dtype == torch.float32 and v.is_contiguous() else v.to(torch.float32).contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


class BlockFP8(object):
    """
    [rows, cols] in 8 bits: value[r, c] = data[r, c] * 2^(exponent[r, c // 128] - 127).
      data      float8_e4m3fn [rows, >= round_up(cols, 128)], zeros from column `cols` on; rows 16-byte aligned
      exponent  uint8 [rows, >= round_up(blocks, 4)], blocks = ceil(cols / 128); rows 4-byte aligned; 255 stands for NaN
    Row slices (`x[10:20]`) share the memory.  `BlockFP8(data, exponent, cols)` takes existing tensors as they are.
    """
    BLOCK = 128
    __slots__ = ("data", "exponent", "cols")

    def __init__(self, data, exponent, cols):
        cols = int(cols)
        blocks = -(-cols // self.BLOCK)
        if data.dim() != 2 or data.dtype != torch.float8_e4m3fn or exponent.dim() != 2 or exponent.dtype != torch.uint8:
            raise ValueError("BlockFP8: data float8_e4m3fn [rows, n], exponent uint8 [rows, n]; got %s %s, %s %s"
                             % (data.dtype, tuple(data.shape), exponent.dtype, tuple(exponent.shape)))
        if cols < 1 or data.shape[1] < blocks * self.BLOCK or exponent.shape[1] < _up(blocks, 4) or data.shape[0] != exponent.shape[0]:
            raise ValueError("BlockFP8: %d columns need data [rows, >= %d] and exponent [rows, >= %d], got %s and %s"
                             % (cols, blocks * self.BLOCK, _up(blocks, 4), tuple(data.shape), tuple(exponent.shape)))
        if data.device != exponent.device:
            raise ValueError("BlockFP8: data on %s, exponent on %s" % (data.device, exponent.device))
        if not (_plain(data) and _plain(exponent)) or _ld(data) % 16 or _ld(exponent) % 4 or data.data_ptr() % 16 or exponent.data_ptr() % 4:
            raise ValueError("BlockFP8: contiguous columns, data rows 16-byte aligned, exponent rows 4-byte aligned")
        self.data, self.exponent, self.cols = data, exponent, cols

    @classmethod
    def empty(cls, rows, cols, device):
        blocks = -(-int(cols) // cls.BLOCK)
        self = cls.__new__(cls)
        self.data = torch.empty((rows, blocks * cls.BLOCK), dtype=torch.float8_e4m3fn, device=device)
        self.exponent = torch.empty((rows, _up(blocks, 4)), dtype=torch.uint8, device=device)
        self.cols = int(cols)
        return self

    @property
    def rows(self):
        return self.data.shape[0]

    @property
    def shape(self):
        return torch.Size((self.data.shape[0], self.cols))

    @property
    def device(self):
        return self.data.device

    def __getitem__(self, rows):
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise ValueError("BlockFP8: only slices of consecutive rows")
        return BlockFP8(self.data[rows], self.exponent[rows], self.cols)

    def dequantize(self, dtype=torch.float32, out=None):
        """The values, [rows, cols] float32 or bfloat16 (exact in both)."""
        dev = _need_cuda(self.data, self.exponent)
        if out is None:
            if dtype not in _DT:
                raise ValueError("dequantize: dtype %s not in %s" % (dtype, [str(d) for d in _DT]))
            out = torch.empty((self.data.shape[0], self.cols), dtype=dtype, device=dev)
        else:
            _out("dequantize", out, self.shape, _DT, dev)
        if out.shape[0]:
            _call(dev, "sugar_fp8_dequant", self.data.data_ptr(), _ld(self.data), self.exponent.data_ptr(), _ld(self.exponent),
                  out.shape[0], self.cols, out.data_ptr(), _ld(out), _DT[out.dtype])
        return out


def _fp8_out(what, out, rows, cols, dev):
    if out is None:
        return BlockFP8.empty(rows, cols, dev)
    if not isinstance(out, BlockFP8) or out.rows != rows or out.cols != cols or out.device != dev:
        raise ValueError("%s: expected a BlockFP8 of [%d, %d] on %s" % (what, rows, cols, dev))
    return out


def quantize_block_fp8(x, out=None):
    """
    [rows, cols] float32 / bfloat16 on the GPU -> BlockFP8.  Every block of 128 columns gets the smallest power of two that
    keeps its largest finite magnitude within 448; values go to the nearest e4m3, ties to the even one.  Infinities and NaN
    become NaN and do not move the scale of their block.
    """
    x = _rows("quantize_block_fp8", x)
    dev = _need_cuda(x)
    q = _fp8_out("quantize_block_fp8", out, x.shape[0], x.shape[1], dev)
    if x.shape[0]:
        _call(dev, "sugar_fp8_quant", x.data_ptr(), _ld(x), _DT[x.dtype], x.shape[0], x.shape[1], q.data.data_ptr(),
              _ld(q.data), q.exponent.data_ptr(), _ld(q.exponent))
    return q


def block_fp8_linear(a, w, scale=None, shift=None, relu=False, out_dtype=torch.bfloat16, out=None):
    """
    relu(a @ w.T) * scale + shift for BlockFP8 a [rows, k] and w [n, k], rounded once to `out_dtype` (bfloat16 or float32).
    float32 outputs are float32 sums of exact products; bfloat16 outputs run twice as fast on the 8-bit matrix
    instruction, whose sums are good to about 1.5e-5 (include/sugar_amd.h).  The order is that of the reference's layers, conv -> ReLU -> BatchNorm
    (sugar/models/dynamictdnn.py:183); scale, shift: float vectors [n], either may be missing.
    """
    if not isinstance(a, BlockFP8) or not isinstance(w, BlockFP8):
        raise ValueError("block_fp8_linear: operands must be BlockFP8 (quantize_block_fp8)")
    rows, n, k = a.data.shape[0], w.data.shape[0], a.cols
    if k != w.cols:
        raise ValueError("block_fp8_linear: a has %d columns, w %d" % (k, w.cols))
    if n == 0:
        raise ValueError("block_fp8_linear: w has no rows")
    dev = _need_cuda(a.data, a.exponent, w.data, w.exponent, *[v for v in (scale, shift) if v is not None])
    scale, shift = _vector("scale", scale, n, dev), _vector("shift", shift, n, dev)
    flags = _lib.EPI_RELU if relu else 0
    if scale is not None or shift is not None:
        flags |= _lib.EPI_AFFINE
        scale = torch.ones(n, device=dev) if scale is None else scale
        shift = torch.zeros(n, device=dev) if shift is None else shift
    if out is None:
        if out_dtype not in _DT:
            raise ValueError("block_fp8_linear: out_dtype %s not in %s" % (out_dtype, [str(d) for d in _DT]))
        out = torch.empty((rows, n), dtype=out_dtype, device=dev)
    else:
        _out("block_fp8_linear", out, (rows, n), _DT, dev)
    if rows:
        _call(dev, "sugar_fp8_linear", a.data.data_ptr(), _ld(a.data), a.exponent.data_ptr(), _ld(a.exponent), rows,
              w.data.data_ptr(), _ld(w.data), w.exponent.data_ptr(), _ld(w.exponent), n, k, _ptr(scale), _ptr(shift), flags,
              out.data_ptr(), _ld(out), _DT[out.dtype])
    return out


RowNorm = collections.namedtuple("RowNorm", "kind weight bias eps")
RowNorm.__new__.__defaults__ = (None, None, 1e-5)
RowNorm.__doc__ = """A norm over the channels of a row: kind "rms" (x / sqrt(mean x^2 + eps)), "layer" ((x - mean) /
sqrt(var + eps)) or "affine" (x itself: a folded BatchNorm); times `weight`, plus `bias` (float vectors, or None)."""

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
    Outputs may be passed in; stream_out may be `residual` or `u` itself, normed_out `u` (in place).  With row_off, rows in
    front of the first and behind the last utterance are left as they are (in outputs allocated here: undefined).
    """
    u = _rows("block_join: u", u)
    residual = _rows("block_join: residual", residual)
    rows, cols = u.shape
    if residual.shape != u.shape:
        raise ValueError("block_join: u %s, residual %s" % (tuple(u.shape), tuple(residual.shape)))
    if cols > MAX_JOIN_COLS:
        raise ValueError("block_join: %d columns, at most %d" % (cols, MAX_JOIN_COLS))
    if u.dtype == torch.float32 and residual.dtype != torch.float32:
        raise ValueError("block_join: a float32 u needs a float32 residual")
    vecs = [t for p in (post, pre) if p is not None for t in (p.weight, p.bias) if t is not None]
    dev = _need_cuda(u, residual, *vecs, *[t for t in (gate, row_off) if t is not None])
    d = _lib.SugarBlockJoin()
    keep = []
    for side, p in (("post", post), ("pre", pre)):
        if p is None:
            continue
        if p.kind not in NORMS or p.kind is None or not p.eps >= 0:
            raise ValueError("block_join: %s kind %r not in %s, or eps %r negative" % (side, p.kind, [k for k in NORMS if k], p.eps))
        wt, bs = _vector(side + " weight", p.weight, cols, dev), _vector(side + " bias", p.bias, cols, dev)
        keep += [wt, bs]
        setattr(d, side + "_kind", NORMS[p.kind])
        setattr(d, side + "_eps", p.eps)
        setattr(d, "d_%s_w" % side, _ptr(wt))
        setattr(d, "d_%s_b" % side, _ptr(bs))
    if row_off is not None:
        if row_off.dim() != 1 or row_off.shape[0] < 2 or row_off.dtype != torch.int32:
            raise ValueError("block_join: row_off must be int32 [B + 1], got %s %s" % (row_off.dtype, tuple(row_off.shape)))
        row_off = row_off.contiguous()
        d.d_row_off, d.n_utts = row_off.data_ptr(), row_off.shape[0] - 1
    if gate is not None:
        if gate.dim() == 1:
            gate = _vector("gate", gate, cols, dev)
            d.gate_kind, d.ldg = 1, cols
        elif row_off is not None and tuple(gate.shape) == (d.n_utts, cols):
            gate = _rows("block_join: gate", gate if gate.dtype == torch.float32 else gate.float())
            d.gate_kind, d.ldg = 2, _ld(gate)
        elif row_off is None and gate.shape == u.shape and gate.dtype == u.dtype:
            gate = _rows("block_join: gate", gate)
            d.gate_kind, d.ldg = 3, _ld(gate)
        else:
            raise ValueError("block_join: gate %s %s is neither [C], [B, C] with row_off, nor [rows, C] of u's dtype without it"
                             % (gate.dtype, tuple(gate.shape)))
        d.d_gate = gate.data_ptr()
    d.rows, d.cols, d.alpha, d.dense = rows, cols, alpha, int(bool(dense))
    d.u_dtype, d.stream_dtype = _DT[u.dtype], _DT[residual.dtype]
    stream = torch.empty((rows, cols), dtype=residual.dtype, device=dev) if stream_out is None else \
        _out("block_join: stream_out", stream_out, (rows, cols), (residual.dtype,), dev)
    d.d_u, d.ldu, d.d_residual, d.ldr = u.data_ptr(), _ld(u), residual.data_ptr(), _ld(residual)
    d.d_stream, d.lds = stream.data_ptr(), _ld(stream)
    z = q = None
    if normed or normed_out is not None:
        out_dtype = u.dtype if out_dtype is None else out_dtype
        if out_dtype not in _DT:
            raise ValueError("block_join: out_dtype %s not in %s" % (out_dtype, [str(t) for t in _DT]))
        z = torch.empty((rows, cols), dtype=out_dtype, device=dev) if normed_out is None else \
            _out("block_join: normed_out", normed_out, (rows, cols), _DT, dev)
        d.d_z, d.ldz, d.z_dtype = z.data_ptr(), _ld(z), _DT[z.dtype]
    if quantized or quantized_out is not None:
        q = _fp8_out("block_join: quantized_out", quantized_out, rows, cols, dev)
        d.d_q, d.ldq, d.d_e, d.lde = q.data.data_ptr(), _ld(q.data), q.exponent.data_ptr(), _ld(q.exponent)
    if rows:
        _call(dev, "sugar_block_join", C.byref(d))
    del keep
    return JoinResult(stream, z, q)
