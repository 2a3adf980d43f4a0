"""
8-bit operands with block scales, their matrix product, and the block join (sugar_amd/blockfp8.py) against plain
implementations in 64 bits.  Tolerances are bounds, not measurements: half a step of the output type, plus the rounding of
float32 sums of n terms, n 2^-24 times the sum of the terms' magnitudes (products of two e4m3 values are exact in float32).
"""
import ctypes as C

import pytest
import torch

import sugar_amd
from sugar_amd import BlockFP8, RowNorm, _lib, block_fp8_linear, block_join, quantize_block_fp8

gpu = pytest.mark.gpu
U32 = 2.0 ** -24                                   # half a step of float32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


# ------------------------------------------------------------------------------------------------ 64-bit forms
def e4m3_table():
    """All finite non-negative e4m3 values, in order (index = bits)."""
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quant64(x):
    """(e4m3 bits [R, padded], exponent byte [R, blocks]) of float rows on the CPU, by search in the table."""
    x = x.detach().cpu().double()
    R, Cc = x.shape
    nb = -(-Cc // 128)
    p = torch.zeros(R, nb * 128, dtype=torch.float64)
    p[:, :Cc] = x
    p = p.view(R, nb, 128)
    fin = torch.isfinite(p)
    amax = torch.where(fin, p.abs(), torch.zeros_like(p)).amax(2)
    powers = torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64)
    byte = torch.searchsorted(powers, amax / 448.0)            # smallest power >= amax / 448, from 2^-127 on
    v = p / powers[byte][:, :, None]
    t = e4m3_table()
    mid = (t[1:] + t[:-1]) / 2
    a = torch.where(fin, v.abs(), torch.zeros_like(v))
    lo = torch.searchsorted(mid, a)                            # ties land on the lower neighbour ...
    tie = (lo < 126) & (a == mid[lo.clamp(max=125)]) & (lo % 2 == 1)
    bits = lo + tie.long()                                     # ... and move up when that one is odd
    bits = torch.where(torch.signbit(v), bits + 128, bits)
    bits = torch.where(fin, bits, torch.full_like(bits, 127))
    return bits.view(R, nb * 128).to(torch.uint8), byte.to(torch.uint8)


def values64(q):
    """The float64 values of a BlockFP8."""
    nb = -(-q.cols // 128)
    v = q.data.cpu().float().double()[:, :nb * 128].view(q.rows, nb, 128)
    e = q.exponent.cpu()[:, :nb].long()
    powers = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [float("nan")], dtype=torch.float64)
    return (v * powers[e][:, :, None]).view(q.rows, -1)[:, :q.cols]


def rows_of(seed, r, c, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(r, c, generator=g) * torch.exp(spread * torch.randn(r, 1, generator=g)) * torch.exp(spread * torch.randn(c, generator=g))
    return x.to(dtype)


def check_quantised(q, x, exact=True):
    bits, byte = quant64(x)
    nb = byte.shape[1]
    assert torch.equal(q.exponent.cpu()[:, :nb], byte)
    assert (q.exponent.cpu()[:, nb:(nb + 3) // 4 * 4] == 127).all()
    got = q.data.cpu().view(torch.uint8)[:, :nb * 128]
    nan = (bits & 127) == 127
    assert torch.equal(got[~nan], bits[~nan])
    assert ((got[nan] & 127) == 127).all()


def linear64(a, w, scale, shift, relu):
    va, vw = values64(a), values64(w)
    y, mag = va @ vw.T, va.abs() @ vw.abs().T
    if relu:
        y = y.clamp(min=0)
    if scale is not None:
        y, mag = y * scale.cpu().double(), mag * scale.cpu().double().abs()
    if shift is not None:
        y, mag = y + shift.cpu().double(), mag + shift.cpu().double().abs()
    return y, mag


def cut64(a, w):
    """Bound of what the 8-bit matrix instruction cuts off: of 8 neighbouring products each loses less than 2^-13 of the
    largest one (taken as largest |a| x largest |w| of the eight)."""
    top = [torch.nn.functional.pad(values64(q).abs(), (0, -q.cols % 8)).view(q.rows, -1, 8).amax(2) for q in (a, w)]
    return 8 * 2.0 ** -13 * (top[0] @ top[1].T)


def check_linear(a, w, scale=None, shift=None, relu=False, dtype=torch.bfloat16, out=None):
    y, mag = linear64(a, w, scale, shift, relu)
    got = block_fp8_linear(a, w, scale=scale, shift=shift, relu=relu, out_dtype=dtype, out=out)
    assert got.dtype == dtype and got.shape == y.shape
    tol = (a.cols + 4) * U32 * mag
    if dtype == torch.bfloat16:
        tol = tol + cut64(a, w) * (1.0 if scale is None else scale.cpu().double().abs())
    tol = tol * (1 + HALF[dtype]) + HALF[dtype] * y.abs() + 1e-38
    bad = (got.cpu().double() - y).abs() > tol
    assert not bad.any(), ((got.cpu().double() - y).abs().max(), bad.sum(), bad.nonzero()[:4])
    return got


def norm64(p, x, mag):
    """(norm of x, magnitude its float32 rounding errors are relative to)."""
    if p is None:
        return x, mag
    w = torch.ones(x.shape[1], dtype=torch.float64) if p.weight is None else p.weight.cpu().double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if p.bias is None else p.bias.cpu().double()
    d, mul = x, torch.ones(x.shape[0], 1, dtype=torch.float64)
    if p.kind == "layer":
        d = x - x.mean(1, keepdim=True)
        mag = mag + mag.mean(1, keepdim=True)
    if p.kind in ("rms", "layer"):
        mul = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + p.eps)
        # an error of the row moves every value through mul as well: relative to it, at most mean |d err| mul^2
        mag = mag + d.abs() * (mul * mul) * (d.abs() * mag).mean(1, keepdim=True) + d.abs()
    return d * mul * w + b, mag * mul * w.abs() + b.abs()


def join64(u, residual, post, gate, row_off, alpha, dense, pre):
    u, r = u.cpu().double(), residual.cpu().double()
    v, mv = norm64(post, u, u.abs())
    g = torch.ones_like(u)
    if gate is not None:
        g = gate.cpu().double()
        if row_off is not None and gate.dim() == 2:
            off = row_off.cpu().long()
            rows = torch.bucketize(torch.arange(u.shape[0]), off, right=True) - 1
            g = g[rows.clamp(0, g.shape[0] - 1)]
    s, ms = r + alpha * g * v, r.abs() + abs(alpha) * g.abs() * mv
    z, mz = norm64(pre, s, ms + s.abs())
    return (r + s if dense else s), (ms + r.abs()), z, mz


ROUNDINGS = 64       # float32 roundings on the longest way to a value: sums of at most 8 x 4 + 8 terms a lane, and the products


def check_join(j, u, residual, post=None, gate=None, row_off=None, alpha=1.0, dense=False, pre=None, rows=slice(None)):
    s, ms, z, mz = join64(u, residual, post, gate, row_off, alpha, dense, pre)
    for got, want, mag in ((j.stream, s, ms), (j.normed, z, mz)):
        if got is None:
            continue
        tol = ROUNDINGS * U32 * mag * (1 + HALF[got.dtype]) + HALF[got.dtype] * want.abs()
        err = (got.cpu().double() - want).abs()[rows]
        assert (err <= tol[rows]).all(), (err.max(), (err > tol[rows]).nonzero()[:4])
    if j.quantized is not None:
        got = values64(j.quantized)
        nb = -(-u.shape[1] // 128)
        pad = torch.zeros(z.shape[0], nb * 128, dtype=torch.float64)
        pad[:, :u.shape[1]] = z.abs() + ROUNDINGS * U32 * mz
        unit = (pad.view(-1, nb, 128).amax(2) / 224.0).repeat_interleave(128, 1)[:, :u.shape[1]]     # 2^e < 2 amax / 448
        tol = 2.0 ** -4 * (z.abs() + ROUNDINGS * U32 * mz) + 2.0 ** -10 * unit + ROUNDINGS * U32 * mz
        err = (got - z).abs()[rows]
        assert (err <= tol[rows]).all(), (err.max(), (err > tol[rows]).nonzero()[:4])
        # and exactly the quantisation of a float32 z where that one was asked for as well
        if j.normed is not None and j.normed.dtype == torch.float32:
            check_quantised(j.quantized[rows], j.normed[rows])


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def parts(r, c):
    nb = -(-c // 128)
    return torch.zeros(r, nb * 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.full((r, (nb + 3) // 4 * 4), 127, dtype=torch.uint8)


def test_no_cpu_fallback_of_the_8_bit_operators():
    x = torch.zeros(3, 8)
    q = BlockFP8(*parts(3, 8), 8)
    for call in (lambda: quantize_block_fp8(x), lambda: q.dequantize(), lambda: block_fp8_linear(q, q), lambda: block_join(x, x)):
        with pytest.raises(_lib.SugarError, match="no CPU fallback"):
            call()


def test_blockfp8_refuses_what_it_cannot_hold():
    d, e = parts(4, 200)
    assert BlockFP8(d, e, 200).shape == (4, 200) and BlockFP8(d, e, 256).cols == 256
    assert BlockFP8(d, e, 200)[1:3].rows == 2
    for bad in (lambda: BlockFP8(d, e, 0), lambda: BlockFP8(d, e, 257), lambda: BlockFP8(d, e[:3], 200),
                lambda: BlockFP8(d.view(torch.uint8), e, 200), lambda: BlockFP8(d, e.to(torch.int32), 200),
                lambda: BlockFP8(d, e[:, :2], 200), lambda: BlockFP8(d.T, e, 4), lambda: BlockFP8(d[0], e, 200),
                lambda: BlockFP8(d, e, 200)[1], lambda: BlockFP8(d, e, 200)[::2]):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(4, 272, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert BlockFP8(wide[:, :256], e, 200).rows == 4                    # a row stride of its own
    with pytest.raises(ValueError):
        BlockFP8(wide[:, 8:264], e, 200)                                # not 16-byte aligned


def test_argument_checks_without_a_gpu():
    x = torch.zeros(3, 8)
    q = BlockFP8(*parts(3, 8), 8)
    p = BlockFP8(*parts(3, 16), 16)
    for call in (lambda: quantize_block_fp8(x[0]), lambda: quantize_block_fp8(x.half()), lambda: quantize_block_fp8(x.long()),
                 lambda: quantize_block_fp8(x[:, :0]), lambda: block_fp8_linear(q, p), lambda: block_fp8_linear(x, q),
                 lambda: block_fp8_linear(q, q[:0]), lambda: block_join(x, x[:2]), lambda: block_join(x, x.bfloat16()),
                 lambda: block_join(x[0], x[0]), lambda: block_join(x.half(), x)):
        with pytest.raises(ValueError):
            call()


def test_numbers_and_sizes_beyond_the_c_types_are_refused():
    x = torch.zeros(3, 8)
    wide = torch.empty(1, 1 << 24, dtype=torch.bfloat16, device="meta")
    d, e = (t.to("meta") for t in parts(1, 128))
    for call in (lambda: block_join(x, x, alpha=1e39), lambda: block_join(x, x, alpha=torch.ones(())), lambda: RowNorm("rms", eps=1e39),
                 lambda: RowNorm("rms", eps=float("nan")), lambda: RowNorm("rms", eps=float("inf")), lambda: quantize_block_fp8(wide),
                 lambda: BlockFP8(d.expand(1, 128), e, 1 << 24), lambda: block_fp8_linear(BlockFP8(*parts(3, 8), 8), BlockFP8.empty(1 << 24, 8, "meta"))):
        with pytest.raises(ValueError):
            call()


def test_c_entries_check_their_arguments_before_any_launch():
    lib, p = _lib.lib(), 4096                                            # an address no call may follow
    fails = [
        lib.sugar_fp8_quant(None, 8, 0, 1, 8, p, 128, p, 4, None),
        lib.sugar_fp8_quant(p, 8, 7, 1, 8, p, 128, p, 4, None),
        lib.sugar_fp8_quant(p, 7, 0, 1, 8, p, 128, p, 4, None),          # stride shorter than the row
        lib.sugar_fp8_quant(p + 2, 8, 0, 1, 8, p, 128, p, 4, None),      # float32 off its alignment
        lib.sugar_fp8_quant(p, 8, 0, -1, 8, p, 128, p, 4, None),
        lib.sugar_fp8_quant(p, 8, 0, 1, 8, p + 8, 128, p, 4, None),
        lib.sugar_fp8_quant(p, 8, 0, 1, 8, p, 120, p, 4, None),
        lib.sugar_fp8_quant(p, 8, 0, 1, 8, p, 128, p, 2, None),
        lib.sugar_fp8_quant(p, 1 << 24, 1, 1, 1 << 24, p, 1 << 24, p, 1 << 17, None),
        lib.sugar_fp8_dequant(p, 1 << 24, p, 1 << 17, 1, 1 << 24, p, 1 << 24, 1, None),
        lib.sugar_fp8_dequant(p, 128, p + 1, 4, 1, 8, p, 8, 0, None),
        lib.sugar_fp8_dequant(p, 128, p, 4, 1, 8, p, 7, 0, None),
        lib.sugar_fp8_linear(p, 128, p, 4, 1, p, 128, p, 4, 0, 8, None, None, 0, p, 8, 0, None),
        lib.sugar_fp8_linear(p, 128, p, 4, 1, p, 128, p, 4, 8, 8, None, None, 2, p, 8, 0, None),   # affine without vectors
        lib.sugar_fp8_linear(p, 128, p, 4, 1, p, 128, p, 4, 8, 8, None, None, 4, p, 8, 0, None),   # unknown flag
        lib.sugar_fp8_linear(p, 128, p, 4, 1, p, 128, p, 4, 8, 129, None, None, 0, p, 8, 0, None),
        lib.sugar_fp8_linear(p, 128, p, 4, 1, p, 128, p, 4, 8, 8, None, None, 0, p, 7, 0, None),
        lib.sugar_fp8_linear(p, 128, p, 4, 1 << 27, p, 128, p, 4, 8, 8, None, None, 0, p, 8, 0, None),
        lib.sugar_block_join(None, None),
    ]
    assert all(rc == -1 for rc in fails), fails

    def join(**kw):
        d = _lib.SugarBlockJoin()
        d.rows, d.cols, d.u_dtype, d.stream_dtype, d.z_dtype = 4, 8, 1, 1, 1
        d.d_u = d.d_residual = d.d_stream = p
        d.ldu = d.ldr = d.lds = 8
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.sugar_block_join(C.byref(d), None)
    for kw in (dict(rows=-1), dict(rows=1 << 33), dict(cols=0), dict(cols=8193), dict(u_dtype=2), dict(u_dtype=0), dict(d_u=None), dict(d_stream=None),
               dict(post_kind=4), dict(pre_kind=-1), dict(post_eps=-1.0), dict(gate_kind=1), dict(d_gate=p), dict(gate_kind=4, d_gate=p),
               dict(gate_kind=2, d_gate=p, ldg=8), dict(d_row_off=p), dict(ldu=7), dict(ldr=4), dict(d_z=p, ldz=7), dict(d_u=p + 1),
               dict(d_q=p, ldq=128, lde=4), dict(d_q=p, d_e=p, ldq=64, lde=4), dict(d_q=p, d_e=p, ldq=128, lde=1),
               dict(d_pre_w=p + 2), dict(gate_kind=3, d_gate=p, ldg=4)):
        assert join(**kw) == -1, kw
    assert join(rows=0) == 0


def test_join_struct_layout_matches_header():
    from sugar_amd import blockfp8
    assert C.sizeof(_lib.SugarBlockJoin) == 8 + 9 * 4 + 3 * 4 + 7 * 8 + 12 * 8 == blockfp8._JOIN.size
    values = tuple(range(1, 11)) + (0.5, 0.25, 0.125) + tuple(range(20, 39))
    d = _lib.SugarBlockJoin.from_buffer_copy(blockfp8._JOIN.pack(*values))
    assert tuple(getattr(d, name) for name, _ in d._fields_) == values


# ------------------------------------------------------------------------------------------------ quantisation
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("r,c", [(1, 1), (1, 7), (3, 127), (5, 128), (2, 129), (301, 512), (17, 536), (64, 80), (1000, 1536), (3, 4001)])
def test_quantise_and_read_back(dtype, r, c):
    x = rows_of(r * 7 + c, r, c, dtype)
    q = quantize_block_fp8(x.cuda())
    check_quantised(q, x)
    for out_dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(q.dequantize(out_dtype).cpu().double(), values64(q))


@gpu
def test_quantise_extremes():
    t = e4m3_table().float()
    mids = ((t[1:] + t[:-1]) / 2).float()
    rows = [torch.cat([t, torch.tensor([448.0])]),                                    # every e4m3 value, scale 1
            torch.cat([mids, torch.tensor([448.0, 448.0])]), -torch.cat([mids, torch.tensor([448.0, 0.0])]),
            torch.full((128,), 448.0), torch.full((128,), 448.00003), torch.full((128,), torch.finfo(torch.float32).max),
            torch.zeros(128), -torch.zeros(128), torch.full((128,), 1e-45), torch.full((128,), 1.1754944e-38),
            torch.full((128,), 2.0 ** -119 * 1.75), torch.full((128,), 2.0 ** -119 * 1.7500001), torch.linspace(-1e-38, 1e-38, 128)]
    inf = torch.linspace(-3, 3, 128)
    inf[5], inf[77], inf[100] = float("inf"), float("-inf"), float("nan")
    rows += [inf, torch.full((128,), float("nan")), torch.full((128,), float("inf"))]
    for x in (torch.stack(rows), torch.stack(rows).bfloat16()):
        q = quantize_block_fp8(x.cuda())
        check_quantised(q, x)
        # (the largest float32 rounds up to 256 * 2^120 = 2^128, which float32 holds as infinity)
        got, want = q.dequantize(torch.float32).cpu().double(), values64(q).float().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = want.abs() >= 2.0 ** -126                                             # below: float32 subnormals, rounded
        assert torch.equal(got[fine], want[fine])
        assert ((got - want).abs()[~fine & ~torch.isnan(want)] <= 2.0 ** -150).all()


@gpu
def test_quantise_strides_offsets_and_preallocated_outputs():
    base = rows_of(3, 40, 700)
    dev = base.cuda()
    for view, cpu in ((dev[:, 3:523], base[:, 3:523]), (dev[::3, 8:520], base[::3, 8:520]), (dev.T, base.T), (dev[5:6, 1:], base[5:6, 1:]),
                      (dev[:1].expand(9, 700), base[:1].expand(9, 700)), (dev.bfloat16()[:, 1:130], base.bfloat16()[:, 1:130])):
        check_quantised(quantize_block_fp8(view), cpu)
    big = BlockFP8.empty(50, 700, "cuda")
    big.data.view(torch.uint8).fill_(0x55)
    big.exponent.fill_(9)
    q = quantize_block_fp8(dev, out=big[5:45])
    check_quantised(q, base)
    for rows in (slice(0, 5), slice(45, 50)):                                        # rows of the operand around it
        assert (big.data[rows].view(torch.uint8) == 0x55).all() and (big.exponent[rows] == 9).all()
    out = torch.full((40, 720), 7.0, device="cuda")
    q.dequantize(out=out[:, 4:704])
    assert torch.equal(out[:, 4:704].cpu().double(), values64(q)) and (out[:, :4] == 7).all() and (out[:, 704:] == 7).all()
    assert quantize_block_fp8(dev[:0]).dequantize().shape == (0, 700)
    for bad in (lambda: quantize_block_fp8(dev, out=big), lambda: quantize_block_fp8(dev, out=out), lambda: q.dequantize(out=out),
                lambda: q.dequantize(torch.float16), lambda: quantize_block_fp8(dev.clone().requires_grad_())):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------ product
def operands(seed, r, n, k):
    a = quantize_block_fp8(rows_of(seed, r, k).cuda())
    w = quantize_block_fp8(rows_of(seed + 1, n, k, spread=0.3).cuda() / k ** 0.5)
    return a, w


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,n,k", [(1, 1, 1), (1, 192, 1536), (2, 16, 128), (7, 33, 129), (16, 512, 512), (17, 17, 17), (63, 512, 512),
                                   (64, 64, 256), (65, 65, 300), (128, 128, 640), (129, 255, 384), (255, 257, 2048), (300, 536, 528),
                                   (301, 1536, 1536), (513, 8, 80)])
def test_linear_sizes(dtype, r, n, k):
    a, w = operands(r + n + k, r, n, k)
    check_linear(a, w, dtype=dtype)


@gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("scale,shift", [(True, True), (True, False), (False, True)])
def test_linear_epilogue(relu, scale, shift):
    a, w = operands(5, 70, 200, 384)
    s = rows_of(8, 1, 200)[0].cuda() if scale else None
    t = rows_of(9, 1, 200)[0].cuda() if shift else None
    for dtype in (torch.bfloat16, torch.float32):
        check_linear(a, w, s, t, relu, dtype)


@gpu
@pytest.mark.parametrize("r,n,k", [(20011, 512, 512), (9001, 1536, 1536), (4097, 536, 528), (33000, 264, 1152), (8200, 2048, 640)])
def test_linear_large(r, n, k):
    a, w = operands(r, r, n, k)
    s = rows_of(8, 1, n)[0].cuda()
    got = block_fp8_linear(a, w, scale=s, relu=True, out_dtype=torch.float32)
    for lo in range(0, r, max(1, r // 3)):                               # the 64-bit form in parts: rows do not depend on others
        y, mag = linear64(a[lo:lo + 700], w, s, None, True)
        err = (got[lo:lo + 700].cpu().double() - y).abs()
        assert (err <= (k + 4) * U32 * mag).all(), err.max()
    last = r - 300
    y, mag = linear64(a[last:], w, s, None, True)
    assert ((got[last:].cpu().double() - y).abs() <= (k + 4) * U32 * mag).all()
    b16 = block_fp8_linear(a, w, scale=s, relu=True)
    for rows in (slice(0, 300), slice(r // 2, r // 2 + 300), slice(r - 300, r)):
        y, mag = linear64(a[rows], w, s, None, True)
        tol = ((k + 4) * U32 * mag + cut64(a[rows], w) * s.cpu().double().abs()) * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()
        assert ((b16[rows].cpu().double() - y).abs() <= tol).all()


@gpu
def test_linear_scales_reach_every_block():
    """Blocks of unlike exponents: a block scaled by the wrong byte would change the result by a power of two."""
    k, n = 128 * 13 + 5, 40
    x = rows_of(1, 300, k)
    x *= torch.pow(2.0, torch.randint(-20, 21, (300, (k + 127) // 128), generator=torch.Generator().manual_seed(2)).float()).repeat_interleave(128, 1)[:, :k]
    wt = rows_of(2, n, k)
    wt *= torch.pow(2.0, torch.randint(-20, 21, (n, (k + 127) // 128), generator=torch.Generator().manual_seed(3)).float()).repeat_interleave(128, 1)[:, :k]
    a, w = quantize_block_fp8(x.cuda()), quantize_block_fp8(wt.cuda())
    assert len(set(a.exponent.cpu().flatten().tolist())) > 20
    check_linear(a, w, dtype=torch.float32)
    check_linear(a[:3], w, dtype=torch.float32)


@gpu
@pytest.mark.parametrize("r", [3, 300])
def test_linear_tiny_times_huge(r):
    """Blocks at the lower end of the exponents (values down to e4m3's smallest times 2^-127) against blocks near the upper
    end.  float32 outputs take the values as bfloat16 numbers: what lies below that type's subnormals is off by at most half
    of the smallest, 2^-134, each; the 8-bit instruction scales behind the product and loses nothing there."""
    k, n = 300, 72
    x, wt = rows_of(1, r, k, spread=0.5) * 2.0 ** -122, rows_of(2, n, k, spread=0.3) * 2.0 ** 100
    a, w = quantize_block_fp8(x.cuda()), quantize_block_fp8(wt.cuda())
    assert a.exponent[:, :3].min() == 0 and 215 < w.exponent[:, :3].max() < 247
    check_linear(a, w, dtype=torch.bfloat16)
    y, mag = linear64(a, w, None, None, False)
    got = block_fp8_linear(a, w, out_dtype=torch.float32).cpu().double()
    lost = 2.0 ** -134 * values64(w).abs().sum(1)
    assert ((got - y).abs() <= (k + 4) * U32 * mag + lost).all()


@gpu
def test_linear_strides_slices_and_untouched_surroundings():
    a, w = operands(11, 90, 60, 600)
    full = block_fp8_linear(a, w)
    assert torch.equal(block_fp8_linear(a[13:77], w[5:55]), full[13:77, 5:55])
    for dtype, lo in ((torch.bfloat16, 8), (torch.bfloat16, 3), (torch.float32, 1), (torch.float32, 4)):
        out = torch.full((94, 90), 7.0, dtype=dtype, device="cuda")
        check_linear(a, w, dtype=dtype, out=out[2:92, lo:lo + 60])
        edge = out.clone()
        edge[2:92, lo:lo + 60] = 7.0
        assert (edge == 7.0).all()
    # columns of a wider operand: block 1 .. of `a` (exponent rows start on a dword: blocks 4 ..)
    big_a, big_w = operands(12, 33, 20, 1024)
    sub = BlockFP8(big_a.data[:, 512:], big_a.exponent[:, 4:], 512)
    check_linear(sub, BlockFP8(big_w.data[:, 512:], big_w.exponent[:, 4:], 512), dtype=torch.float32)
    assert block_fp8_linear(a[:0], w).shape == (0, 60)


@gpu
def test_linear_nan_stays_in_its_row():
    x = rows_of(4, 40, 300)
    x[7, 100], x[20, 299] = float("nan"), float("inf")
    a, w = quantize_block_fp8(x.cuda()), quantize_block_fp8(rows_of(5, 30, 300).cuda())
    for relu, dtype in ((False, torch.bfloat16), (True, torch.bfloat16), (True, torch.float32)):
        y = block_fp8_linear(a, w, relu=relu, out_dtype=dtype).cpu()
        assert torch.isnan(y[[7, 20]]).all() and torch.isfinite(y[[i for i in range(40) if i not in (7, 20)]]).all()
    w.exponent[3, 1] = 255                                               # the byte that stands for NaN
    for dtype in (torch.bfloat16, torch.float32):
        y = block_fp8_linear(a[:7], w, out_dtype=dtype).cpu()
        assert torch.isnan(y[:, 3]).all() and torch.isfinite(y[:, :3]).all() and torch.isfinite(y[:, 4:]).all()


# ------------------------------------------------------------------------------------------------ join
def norm_of(kind, c, seed, bias=True, eps=1e-5):
    if kind is None:
        return None
    return RowNorm(kind, 1 + 0.3 * rows_of(seed, 1, c, spread=0.1)[0].cuda(), rows_of(seed + 1, 1, c, spread=0.1)[0].cuda() if bias else None, eps)


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


@gpu
@pytest.mark.parametrize("tu,ts", TYPES)
@pytest.mark.parametrize("post", [None, "affine", "rms", "layer"])
@pytest.mark.parametrize("pre", [None, "affine", "rms", "layer"])
def test_join_norms(tu, ts, post, pre):
    r, c = 37, 264
    u, res = rows_of(1, r, c, tu).cuda(), rows_of(2, r, c, ts).cuda()
    kw = dict(post=norm_of(post, c, 3), pre=norm_of(pre, c, 5, bias=pre != "rms"), gate=torch.rand(c).cuda(), alpha=0.7)
    check_join(block_join(u, res, quantized=True, **kw), u, res, **kw)
    check_join(block_join(u, res, quantized=True, out_dtype=torch.float32, dense=True, **kw), u, res, dense=True, **kw)


@gpu
@pytest.mark.parametrize("tu,ts", TYPES)
@pytest.mark.parametrize("r,c", [(1, 1), (1, 512), (2, 7), (3, 129), (5, 511), (4, 513), (700, 512), (9, 1024), (6, 1536), (3, 2048),
                                 (3, 2049), (2, 4096), (2, 4100), (2, 8192), (3, 8190)])
def test_join_sizes(tu, ts, r, c):
    u, res = rows_of(r, r, c, tu).cuda(), rows_of(c, r, c, ts).cuda()
    kw = dict(post=norm_of("layer", c, 3), pre=norm_of("rms", c, 5), alpha=-1.5)
    check_join(block_join(u, res, quantized=True, **kw), u, res, **kw)
    kw = dict(gate=torch.rand(r, c).to(tu).cuda())
    check_join(block_join(u, res, quantized=True, out_dtype=torch.float32, **kw), u, res, **kw)


@gpu
@pytest.mark.parametrize("c", [512, 40, 1000])
def test_join_gate_per_utterance(c):
    off = [0, 1, 1, 5, 105, 105, 405, 406, 700]                          # empty and single-row utterances
    r = off[-1]
    row_off = torch.tensor(off, dtype=torch.int32).cuda()
    u, res, gate = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(2, r, c, torch.bfloat16).cuda(), torch.rand(8, c).cuda()
    for dense in (False, True):
        kw = dict(gate=gate, row_off=row_off, dense=dense, pre=norm_of("layer", c, 9))
        check_join(block_join(u, res, quantized=True, **kw), u, res, **kw)


@gpu
def test_join_rows_outside_the_utterances_are_left_alone():
    c, r = 136, 90
    row_off = torch.tensor([4, 4, 30, 80], dtype=torch.int32).cuda()
    u, res, gate = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(2, r, c).cuda(), torch.rand(3, c).cuda()
    stream, z, q = torch.full((r, c), 7.0).cuda(), torch.full((r, c), 7.0).cuda().bfloat16(), BlockFP8.empty(r, c, "cuda")
    q.data.view(torch.uint8).fill_(0x55)
    q.exponent.fill_(9)
    kw = dict(gate=gate, row_off=row_off, pre=norm_of("rms", c, 9))
    j = block_join(u, res, stream_out=stream, normed_out=z, quantized_out=q, **kw)
    assert j.stream is stream and j.normed is z and j.quantized is q
    check_join(j, u, res, rows=slice(4, 80), **kw)
    for rows in (slice(0, 4), slice(80, 90)):
        assert (stream[rows] == 7).all() and (z[rows] == 7).all()
        assert (q.data[rows].view(torch.uint8) == 0x55).all() and (q.exponent[rows] == 9).all()


@gpu
def test_join_in_place_strides_and_single_outputs():
    c, r = 200, 33
    big_u, big_r = rows_of(1, r, 300, torch.bfloat16).cuda(), rows_of(2, r, 301, torch.bfloat16).cuda()
    u, res = big_u[:, 8:208], big_r[:, 1:201]
    kw = dict(post=norm_of("rms", c, 3, bias=False), pre=norm_of("layer", c, 5), dense=True)
    want = block_join(u, res, quantized=True, **kw)
    check_join(want, u, res, **kw)
    only = block_join(u, res, normed=False, **kw)
    assert only.normed is None and only.quantized is None and torch.equal(only.stream, want.stream)
    u2, r2 = u.clone(), big_r.clone()
    got = block_join(u2, r2[:, 1:201], stream_out=r2[:, 1:201], normed_out=u2, **kw)
    assert torch.equal(got.stream, want.stream) and torch.equal(u2, want.normed)
    assert torch.equal(r2[:, 0], big_r[:, 0]) and torch.equal(r2[:, 201:], big_r[:, 201:])
    for bad in (lambda: block_join(u, res, gate=torch.rand(7, c).cuda()), lambda: block_join(u, res, gate=torch.rand(r, c).cuda()),
                lambda: block_join(u, res, post=RowNorm("batch")), lambda: block_join(u, res, post="rms"), lambda: block_join(u, res, post=RowNorm("rms", torch.ones(3).cuda())),
                lambda: block_join(u, res, pre=RowNorm("rms", None, None, -1.0)), lambda: block_join(u, res, out_dtype=torch.float16),
                lambda: block_join(u, res, row_off=torch.zeros(3).cuda()), lambda: block_join(u, res, stream_out=u2[:5]),
                lambda: block_join(u, res, gate=torch.rand(c)), lambda: block_join(u, res, quantized_out=stream_like(u2))):
        with pytest.raises((ValueError, _lib.SugarError)):
            bad()


@gpu
def test_outputs_that_share_memory_are_refused():
    c, r = 128, 16
    big = rows_of(1, r, 3 * c, torch.bfloat16).cuda()
    u, res, out = big[:, :c], big[:, c:2 * c], big[:, 2 * c:]            # columns of one buffer are apart
    want = block_join(u, res)
    got = block_join(u, res, stream_out=out)
    assert torch.equal(got.stream, want.stream) and torch.equal(got.normed, want.normed)
    flat = torch.zeros(r * c + 8, dtype=torch.bfloat16, device="cuda")
    x, y = flat[:r * c].view(r, c), flat[8:].view(r, c)
    q = quantize_block_fp8(x)
    raw = q.data.view(torch.uint8).view(-1)[:r * 64].view(torch.bfloat16).view(r, 32)
    for bad in (lambda: block_join(x, x.clone(), stream_out=y), lambda: block_join(x.clone(), x, normed_out=y),
                lambda: block_join(x.clone(), x, normed_out=x), lambda: block_join(u, res, stream_out=x, normed_out=x),
                lambda: block_join(x.clone(), x.clone(), stream_out=x, normed_out=y),
                lambda: block_join(big[:, :c], big[:, c:2 * c], stream_out=big[:, 8:c + 8]),
                lambda: block_fp8_linear(q, q[:16], out=q.data.view(torch.uint8).view(torch.bfloat16)[:, :16]),
                lambda: quantize_block_fp8(raw, out=BlockFP8(q.data, q.exponent, 32)),
                lambda: block_join(x, x.clone(), stream_out=x, normed_out=x)):   # (each alone may be u itself)
        with pytest.raises(ValueError, match="shares memory"):
            bad()


@gpu
def test_outputs_passed_in_with_any_form_of_the_gate():
    """Gates and row offsets that are no plain matrix or vector (transposed, other types, every second entry) next to outputs
    of the caller's; an output that requires a gradient; an operand whose parts lie in each other."""
    c, r = 136, 24
    u, res = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(2, r, c, torch.bfloat16).cuda()
    off = torch.tensor([0, 7, 10, 3, 24, 9], dtype=torch.int32).cuda()[::2]
    gate = torch.rand(c, 2).cuda()
    for kw in (dict(gate=gate.T, row_off=off), dict(gate=gate.T.bfloat16(), row_off=off), dict(gate=torch.rand(c, r).cuda().bfloat16().T),
               dict(gate=torch.rand(2 * c).cuda()[::2]), dict(gate=torch.rand(c).cuda().double())):
        want = block_join(u, res, **kw)
        out = torch.empty_like(u)
        got = block_join(u, res, stream_out=out, **kw)
        assert got.stream is out and torch.equal(out, want.stream) and torch.equal(got.normed, want.normed)
        check_join(want, u, res, **kw)
    leaf = torch.zeros(r, c, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q = quantize_block_fp8(u)
    raw = torch.zeros(r, 1024, dtype=torch.uint8, device="cuda")
    inside = BlockFP8(raw[:, :256].view(torch.float8_e4m3fn), raw[:, 128:132], c)
    for bad in (lambda: block_join(u, res, stream_out=leaf), lambda: block_fp8_linear(q, q, out=leaf[:, :r]), lambda: q.dequantize(out=leaf),
                lambda: quantize_block_fp8(u, out=inside)):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        assert torch.equal(q.dequantize(out=leaf), q.dequantize(torch.bfloat16))


def stream_like(x):
    return torch.empty_like(x)


@gpu
def test_join_non_finite_rows_do_not_spread():
    c = 512
    u, res = rows_of(1, 20, c, torch.bfloat16), rows_of(2, 20, c, torch.bfloat16)
    u[3, 17], res[9, 500] = float("inf"), float("nan")
    j = block_join(u.cuda(), res.cuda(), post=norm_of("layer", c, 3), pre=norm_of("rms", c, 5), quantized=True)
    good = [i for i in range(20) if i not in (3, 9)]
    assert torch.isfinite(j.normed.cpu()[good]).all() and torch.isnan(j.normed.cpu()[[3, 9]]).any(1).all()
    assert torch.isfinite(values64(j.quantized)[good]).all() and torch.isnan(values64(j.quantized)[[3, 9]]).any(1).all()
    zero = torch.zeros(4, c).cuda()                                      # rows of zeros: eps keeps the norm finite
    j = block_join(zero, zero, post=RowNorm("rms"), pre=RowNorm("layer"), quantized=True)
    assert (j.normed == 0).all() and (values64(j.quantized) == 0).all()


@gpu
@pytest.mark.parametrize("c", [200, 520, 1100])
def test_join_pads_bad_rows_with_zeros(c):
    """Rows that a norm makes NaN throughout, an infinite factor: the padding columns of the 8-bit output stay 0 and the rest
    is the quantisation of the float32 output."""
    u, res = rows_of(1, 9, c), rows_of(2, 9, c)
    u[3, 17], res[5, c - 1], u[6] = float("inf"), float("nan"), 0.0
    for kw in (dict(post=norm_of("layer", c, 3), pre=norm_of("layer", c, 5)), dict(alpha=float("inf")), dict(alpha=float("nan")),
               dict(gate=torch.rand(c).cuda(), alpha=float("-inf"), pre=norm_of("affine", c, 5))):
        j = block_join(u.cuda(), res.cuda(), quantized=True, **kw)
        check_quantised(j.quantized, j.normed)
        assert (j.quantized.data.view(torch.uint8)[:, c:(c + 127) // 128 * 128] == 0).all()


# ------------------------------------------------------------------------------------------------ together, streams, graphs
@gpu
def test_two_blocks_of_products_and_joins():
    """quantise -> product -> join (norms, gate per utterance, 8-bit output) -> product -> join, every step against the 64-bit
    form of the step on what the kernels handed over."""
    c, mid = 256, 384
    off = torch.tensor([0, 40, 40, 193], dtype=torch.int32).cuda()
    x = rows_of(1, 193, c, torch.bfloat16, spread=0.4).cuda()
    ws = [quantize_block_fp8(rows_of(10 + i, n, k, spread=0.2).cuda() / k ** 0.5) for i, (n, k) in enumerate([(mid, c), (c, mid), (mid, c), (c, mid)])]
    gate = torch.rand(3, c).cuda()
    stream, q = x, quantize_block_fp8(x)
    for blk in range(2):
        h = check_linear(q, ws[2 * blk], relu=True)
        qh = quantize_block_fp8(h)
        check_quantised(qh, h)
        y = check_linear(qh, ws[2 * blk + 1])
        kw = dict(post=norm_of("rms", c, 20 + blk), gate=gate, row_off=off, alpha=0.5, pre=norm_of("layer", c, 30 + blk))
        j = block_join(y, stream, quantized=True, **kw)
        check_join(j, y, stream, **kw)
        stream, q = j.stream, j.quantized


@gpu
def test_streams_and_graph_replays():
    c, n, r = 512, 536, 300
    w = quantize_block_fp8(rows_of(2, n, c).cuda() / 20)
    x, res = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(3, r, c, torch.bfloat16).cuda()
    norm = norm_of("rms", c, 5)

    def step():
        j = block_join(x, res, post=norm, quantized=True)
        return j.stream, j.normed, quantize_block_fp8(j.normed).dequantize(), block_fp8_linear(j.quantized, w, relu=True)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 7, 9):
        x.copy_(rows_of(seed, r, c, torch.bfloat16))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(held, want)), seed


@gpu
def test_results_do_not_depend_on_the_other_rows():
    """A row's result is the same alone and in a batch only where the same kernel serves both; its values always agree to
    rounding, and calls repeat bit for bit."""
    a, w = operands(21, 5000, 512, 512)
    y = block_fp8_linear(a, w, out_dtype=torch.float32)
    assert torch.equal(y, block_fp8_linear(a, w, out_dtype=torch.float32))
    one = block_fp8_linear(a[100:101], w, out_dtype=torch.float32)
    _, mag = linear64(a[100:101], w, None, None, False)
    assert ((one.cpu().double() - y[100:101].cpu().double()).abs() <= 2 * 516 * U32 * mag).all()
    u, res = rows_of(1, 3000, 512, torch.bfloat16).cuda(), rows_of(2, 3000, 512, torch.bfloat16).cuda()
    j = block_join(u, res, pre=norm_of("rms", 512, 5))
    k = block_join(u[7:9], res[7:9], pre=norm_of("rms", 512, 5))
    assert torch.equal(j.normed[7:9], k.normed)


@gpu
@pytest.mark.parametrize("r,n,k", [(23000, 1536, 1152), (44000, 776, 1400), (100001, 264, 1024), (35000, 1024, 2100)])
def test_linear_persistent_tiles(r, n, k):
    """Products of two rounds of 256 x 256 tiles and more: odd numbers of k-tiles, channels and rows that end inside a tile,
    one tile of channels, tails; with and without the affine vectors, and rows around the output left alone."""
    check_many_rows(r, n, k)


@gpu
@pytest.mark.parametrize("r,n,k", [(60000, 512, 512), (35001, 776, 384), (52007, 456, 100), (52016, 1000, 200)])
def test_linear_weights_in_registers(r, n, k):
    """Products of up to 4 blocks over many rows: every number of blocks, slabs that are not full, runs of uneven length."""
    check_many_rows(r, n, k)


def check_many_rows(r, n, k):
    a, w = operands(r, r, n, k)
    s, t = rows_of(8, 1, n)[0].cuda(), rows_of(9, 1, n)[0].cuda()
    out = torch.full((r + 2, n + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    for scale, shift, relu in ((s, t, True), (None, None, False)):
        got = block_fp8_linear(a, w, scale=scale, shift=shift, relu=relu, out=out[1:r + 1, :n])
        wide = block_fp8_linear(a, w, scale=scale, shift=shift, relu=relu, out_dtype=torch.float32)
        for lo in (0, 200, r // 2, r - 333):
            rows = slice(lo, lo + 333)
            y, mag = linear64(a[rows], w, scale, shift, relu)
            assert ((wide[rows].cpu().double() - y).abs() <= (k + 4) * U32 * mag).all()
            f = 1.0 if scale is None else scale.cpu().double().abs()
            tol = ((k + 4) * U32 * mag + cut64(a[rows], w) * f) * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()
            assert ((got[rows].cpu().double() - y).abs() <= tol).all()
        # everywhere, against the float32 output: cut-offs and roundings of both
        top = a.data.float().abs().amax(1)
        assert torch.isfinite(top).all()
        assert ((got.float() - wide).norm() / wide.norm()).item() <= 2.0 ** -8
        worst = (got.float() - wide).abs().amax(1) / wide.abs().amax(1).clamp(min=1e-30)
        assert (worst <= 2.0 ** -7).all()
    assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[:, n:] == 7).all()


@gpu
def test_linear_huge_operand_offsets():
    """Rows whose byte offsets pass 32 bits: the left operand is cut into launches."""
    r, k, n = 2_200_000, 2048, 8
    a = BlockFP8.empty(r, k, "cuda")
    a.data.view(torch.uint8).fill_(0x38)                                # 1.0
    a.exponent.fill_(127)
    w = quantize_block_fp8(rows_of(1, n, k).cuda())
    probe = [0, 1, 2_000_000, 2_097_000, 2_097_151, 2_097_152, 2_100_000, r - 1]
    x = rows_of(2, len(probe), k, spread=0.2).cuda()
    q = quantize_block_fp8(x)
    for i, row in enumerate(probe):
        a.data[row:row + 1].view(torch.uint8).copy_(q.data[i:i + 1].view(torch.uint8))
        a.exponent[row:row + 1].copy_(q.exponent[i:i + 1])
    y = block_fp8_linear(a, w, out_dtype=torch.float32)
    want, mag = linear64(q, w, None, None, False)
    assert ((y[probe].cpu().double() - want).abs() <= (k + 4) * U32 * mag).all()
    ones, mag = values64(w).sum(1), values64(w).abs().sum(1)
    keep = torch.ones(r, dtype=torch.bool, device="cuda")
    keep[probe] = False
    bad = ((y.double() - ones.cuda()).abs() > ((k + 4) * U32 * mag).cuda()).any(1) & keep
    assert not bad.any()


@gpu
@pytest.mark.parametrize("c", [8, 9, 15, 121, 127, 130, 253, 519, 1027])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_end_of_a_row(c, dtype):
    """Rows whose last 1 .. 7 columns are no whole group of eight, inside a wider buffer whose other columns are NaN (nothing of
    them may come in) or 7 (nothing may be written there)."""
    r = 21
    big = torch.full((r, c + 11), float("nan"), dtype=dtype)
    big[:, 3:3 + c] = rows_of(c, r, c, dtype)
    x = big.cuda()[:, 3:3 + c]
    q = quantize_block_fp8(x)
    check_quantised(q, big[:, 3:3 + c])
    out = torch.full((r, c + 11), 7.0, dtype=dtype, device="cuda")
    q.dequantize(out=out[:, 5:5 + c])
    assert torch.equal(out[:, 5:5 + c].cpu().double(), values64(q)) and (out[:, :5] == 7).all() and (out[:, 5 + c:] == 7).all()
    gate, res = torch.full((r, c + 4), float("nan"), dtype=dtype, device="cuda"), rows_of(c + 1, r, c, dtype).cuda()
    gate[:, 1:1 + c] = torch.rand(r, c).to(dtype)
    kw = dict(post=norm_of("layer", c, 3), pre=norm_of("rms", c, 5), gate=gate[:, 1:1 + c])
    stream, z = (torch.full((r, c + 11), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    check_join(block_join(x, res, stream_out=stream[:, 1:1 + c], normed_out=z[:, 4:4 + c], quantized=True, **kw), x, res, **kw)
    for t, lo in ((stream, 1), (z, 4)):
        assert (t[:, :lo] == 7).all() and (t[:, lo + c:] == 7).all()
    w = quantize_block_fp8(rows_of(c + 2, c, 200, spread=0.2).cuda() / 14)
    a = quantize_block_fp8(rows_of(c + 3, 900, 200).cuda())
    for rows in (3, 900):                                                 # the direct kernel's and the tiles' stores
        out = torch.full((rows, c + 11), 7.0, dtype=dtype, device="cuda")
        check_linear(a[:rows], w, dtype=dtype, out=out[:, 2:2 + c])
        assert (out[:, :2] == 7).all() and (out[:, 2 + c:] == 7).all()


@gpu
def test_quantise_more_rows_than_one_launch_takes():
    r = (1 << 27) + 77
    x = torch.ones(r, 1, dtype=torch.bfloat16, device="cuda")
    probe = [0, 1, (1 << 27) - 1, 1 << 27, (1 << 27) + 1, r - 1]
    x[probe] = torch.tensor([[3.0], [-0.3], [500.0], [-7.0], [1e-30], [0.11]], dtype=torch.bfloat16, device="cuda")
    q = quantize_block_fp8(x)
    for i in probe:
        check_quantised(q[i:i + 1], x[i:i + 1])
    y = q.dequantize(torch.bfloat16)
    assert (y[probe] != 1).all() and int((y == 1).sum()) == r - len(probe)
    assert bool((q.exponent[:, 0] == 119).sum() == r - len(probe)) and bool((q.exponent[:, 1:] == 127).all())


@gpu
@pytest.mark.parametrize("c", [5, 20, 128, 150, 256, 300])
def test_join_many_utterances_in_narrow_rows(c):
    """Several rows a wave, each with an utterance of its own: more utterances than one step of the search tells apart, empty
    ones among them, rows in front of the first and behind the last."""
    g = torch.Generator().manual_seed(c)
    sizes = torch.randint(0, 5, (1500,), generator=g)
    off = torch.cat([torch.tensor([3]), 3 + sizes.cumsum(0)]).to(torch.int32)
    n = int(off[-1])
    r = n + 6
    u, res, gate = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(2, r, c).cuda(), torch.rand(1500, c).cuda()
    for post, pre in ((None, None), ("rms", "layer")):
        out = torch.full((r, c), 7.0).cuda()
        kw = dict(gate=gate, row_off=off.cuda(), post=norm_of(post, c, 3), pre=norm_of(pre, c, 5))
        j = block_join(u, res, stream_out=out, quantized=True, **kw)
        check_join(j, u, res, rows=slice(3, n), **kw)
        assert (out[:3] == 7).all() and (out[n:] == 7).all()


@gpu
@pytest.mark.parametrize("r,c", [(9000, 100), (9001, 256), (7003, 513), (4099, 1025), (3001, 1536), (2003, 2047), (1001, 3000), (70001, 16)])
def test_join_runs_of_rows(r, c):
    """Rows enough that a group of lanes takes several, over every number of lanes and waves a row."""
    u, res = rows_of(1, r, c, torch.bfloat16).cuda(), rows_of(2, r, c, torch.bfloat16).cuda()
    kw = dict(post=norm_of("layer", c, 3), pre=norm_of("rms", c, 5), gate=torch.rand(c).cuda())
    check_join(block_join(u, res, quantized=True, **kw), u, res, **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,n,k", [(1492, 1088, 567), (9619, 72, 850), (13446, 373, 704), (2100, 1000, 130), (9000, 1400, 100), (12001, 300, 1030)])
def test_linear_every_tile(dtype, r, n, k):
    """Sizes between a few rows and many: each tile and number of waves, rows and channels that end inside one."""
    a, w = operands(r, r, n, k)
    s, t = rows_of(8, 1, n)[0].cuda(), rows_of(9, 1, n)[0].cuda()
    got = block_fp8_linear(a, w, scale=s, shift=t, relu=True, out_dtype=dtype)
    for lo in (0, r // 2, r - 200):
        rows = slice(lo, lo + 200)
        y, mag = linear64(a[rows], w, s, t, True)
        tol = (k + 4) * U32 * mag
        if dtype == torch.bfloat16:
            tol = (tol + cut64(a[rows], w) * s.cpu().double().abs()) * (1 + HALF[dtype]) + HALF[dtype] * y.abs()
        assert ((got[rows].cpu().double() - y).abs() <= tol).all()
    # everywhere: the same products by the 64-bit form's inputs in float32, 64 rows of every 500
    for lo in range(0, r - 64, 500):
        part = block_fp8_linear(a[lo:lo + 64], w, scale=s, shift=t, relu=True, out_dtype=torch.float32)
        err = (got[lo:lo + 64].float() - part).abs().amax(1) / part.abs().amax(1).clamp(min=1e-30)
        assert (err <= (2.0 ** -7 if dtype == torch.bfloat16 else 1e-5)).all()


@gpu
def test_join_more_rows_than_short_runs_cover():
    """A launch has fewer than 2^32 threads: runs of rows get longer."""
    r = (1 << 29) + 4321
    u, res = torch.ones(r, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(r, 1, dtype=torch.bfloat16, device="cuda")
    probe = torch.tensor([0, 1, 12345, (1 << 29) - 1, 1 << 29, r - 2, r - 1], device="cuda")
    u[probe, 0] = torch.arange(2, 9, device="cuda").bfloat16()
    out = block_join(u, res, alpha=2.0, normed=False, stream_out=res).stream
    assert out[probe, 0].tolist() == [2.0 * i for i in range(2, 9)]
    assert int((out == 2).sum()) == r - len(probe)


@gpu
@pytest.mark.parametrize("tu,ts", TYPES)
@pytest.mark.parametrize("r,c", [(12000, 512), (20011, 200), (40003, 100), (9001, 600), (5003, 1500), (3001, 3000), (40003, 5)])
def test_join_utterances_begin_inside_runs_of_rows(tu, ts, r, c):
    """Rows enough that a group of lanes takes 2 .. 4 of them one after the other (share of launch_join >= 2 on 256 CUs).  Utterances
    of 0 .. 6 rows begin inside those runs: the gate changes within them, rows of no utterance end them."""
    g = torch.Generator().manual_seed(r + c)
    sizes = torch.randint(0, 7, (r // 3,), generator=g)
    sizes = sizes[sizes.cumsum(0) < r - 9]
    off = torch.cat([torch.tensor([3]), 3 + sizes.cumsum(0)]).to(torch.int32)
    n, b = int(off[-1]), len(sizes)
    u, res, gate = rows_of(1, r, c, tu).cuda(), rows_of(2, r, c, ts).cuda(), torch.rand(b, c, generator=g).cuda()
    for kw in (dict(dense=True), dict(post=norm_of("rms", c, 3), pre=norm_of("layer", c, 5), alpha=0.7)):
        kw.update(gate=gate, row_off=off.cuda())
        stream, z, q = torch.full((r, c), 7.0, dtype=ts).cuda(), torch.full((r, c), 7.0).cuda(), BlockFP8.empty(r, c, "cuda")
        q.data.view(torch.uint8).fill_(0x55)
        q.exponent.fill_(9)
        j = block_join(u, res, stream_out=stream, normed_out=z, quantized_out=q, **kw)
        check_join(j, u, res, rows=slice(3, n), **kw)
        for rows in (slice(0, 3), slice(n, r)):
            assert (stream[rows] == 7).all() and (z[rows] == 7).all()
            assert (q.data[rows].view(torch.uint8) == 0x55).all() and (q.exponent[rows] == 9).all()


@gpu
@pytest.mark.parametrize("tu,ts", TYPES)
@pytest.mark.parametrize("r,c", [(12000, 512), (20011, 200), (40003, 100), (9001, 600), (5003, 1500), (40003, 5)])
def test_join_runs_of_rows_with_gates_and_in_place(tu, ts, r, c):
    """The same runs with a gate per row, fetched with the row ahead, with one per channel and with none; outputs in place of the
    inputs, whose next row has been fetched by then."""
    u, res = rows_of(1, r, c, tu).cuda(), rows_of(2, r, c, ts).cuda()
    norms = dict(post=norm_of("layer", c, 3), pre=norm_of("rms", c, 5))
    row_gate, channel_gate = torch.rand(r, c).to(tu).cuda(), torch.rand(c).cuda()
    for kw in (dict(gate=row_gate), dict(gate=row_gate, **norms), dict(gate=channel_gate), dict(gate=channel_gate, **norms), dict(alpha=-2.0)):
        want = block_join(u, res, quantized=True, **kw)
        check_join(want, u, res, **kw)
        u2, res2 = u.clone(), res.clone()
        got = block_join(u2, res2, stream_out=res2, normed_out=u2, quantized=True, **kw)
        assert torch.equal(res2, want.stream) and torch.equal(u2, want.normed) and torch.equal(got.quantized.exponent, want.quantized.exponent)
        assert torch.equal(got.quantized.data.view(torch.uint8), want.quantized.data.view(torch.uint8))
        if tu == ts:
            u2 = u.clone()
            assert block_join(u2, res, stream_out=u2, **kw).stream is u2 and torch.equal(u2, want.stream)


@gpu
@pytest.mark.parametrize("r,n,k", [(52007, 457, 100), (52016, 1001, 200), (35001, 779, 384), (60000, 511, 512),          # weights in registers
                                   (23000, 1531, 1152), (44000, 773, 1400), (100001, 261, 1024),                     # persistent, each tail
                                   (9000, 1399, 100), (4816, 1533, 640)])                                                # 128 x 128 tiles
def test_linear_many_rows_of_odd_widths(r, n, k):
    """Output widths that are no multiple of 8 over many rows: every kernel's stores of the last 1 .. 7 channels, and the half
    tile of float32 outputs (773)."""
    check_many_rows(r, n, k)
