"""
What the 8-bit operators hand to the library and what they refuse.  On the CPU the check for a GPU is taken out and the library
call is replaced by a record of its arguments, so nothing is launched; what the kernels make of such calls is tested on a GPU.
"""
import pytest
import torch
from torch.autograd import forward_ad

import sugar_amd
from sugar_amd import BlockFP8, RowNorm, block_fp8_linear, block_join, blockfp8, quantize_block_fp8

gpu = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    """The library calls a test makes, [(name, arguments)]; CPU tensors stand for the GPU's."""
    made = []
    monkeypatch.setattr(blockfp8, "_gpu", lambda dev: dev)
    monkeypatch.setattr(blockfp8, "_call", lambda dev, name, *args: made.append((name, args)))
    return made


def operand(rows, cols):
    q = BlockFP8.empty(rows, cols, "cpu")
    q.data.view(torch.uint8).zero_()
    q.exponent.fill_(127)
    return q


def join_args(call):
    """The descriptor of a recorded join."""
    name, (packed,) = call
    assert name == "sugar_block_join"
    return sugar_amd._lib.SugarBlockJoin.from_buffer_copy(packed)


def test_dual_tensors_are_refused(calls):
    """Forward-mode differentiation: a dual tensor does not require a gradient, its tangent would be dropped silently."""
    c, r = 128, 4
    x, res, vec, gate = torch.randn(r, c), torch.randn(r, c), torch.randn(c), torch.rand(r, c)
    q = operand(r, c)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        bad = (lambda: quantize_block_fp8(dual(x)), lambda: block_fp8_linear(q, q, scale=dual(torch.randn(r))),
               lambda: block_fp8_linear(q, q, shift=dual(torch.randn(r))), lambda: block_join(dual(x), res),
               lambda: block_join(x, dual(res)), lambda: block_join(x, res, gate=dual(gate)), lambda: block_join(x, res, gate=dual(vec)),
               lambda: block_join(x, res, post=RowNorm("rms", dual(vec))), lambda: block_join(x, res, pre=RowNorm("layer", None, dual(vec))),
               lambda: block_join(x, res, pre=RowNorm("layer", dual(vec.double()))),
               lambda: block_join(x, res, stream_out=dual(x.clone())), lambda: q.dequantize(out=dual(x.clone())),
               lambda: block_fp8_linear(q, q, out_dtype=torch.float32, out=dual(torch.zeros(r, r))))
        for grad in (True, False):                      # torch.no_grad() records no gradients, but forward derivatives all the same
            with torch.set_grad_enabled(grad):
                for call in bad:
                    with pytest.raises(ValueError, match="dual"):
                        call()
        with pytest.raises(ValueError, match="forward derivative"):
            BlockFP8(dual(q.data), q.exponent, c)
        assert not calls
        quantize_block_fp8(x)                            # plain tensors at a level, and what a dual tensor stands for
        block_join(forward_ad.unpack_dual(dual(x)).primal, res, gate=gate)
    block_join(x, res)
    assert [name for name, _ in calls] == ["sugar_fp8_quant", "sugar_block_join", "sugar_block_join"]


def test_views_whose_memory_holds_the_negated_values(calls):
    """The imaginary part of a conjugate is a view with the sign still to be applied; one column of it passes for a plain matrix."""
    view = torch.randn(6, 1, dtype=torch.complex64).conj().imag
    vec = torch.randn(1, dtype=torch.complex64).conj().imag
    assert view.is_neg() and vec.is_neg() and vec.is_contiguous()
    x = torch.randn(6, 1)
    quantize_block_fp8(view)
    assert calls[-1][1][0] != view.data_ptr()
    block_join(view, x, gate=vec)
    j = join_args(calls[-1])
    assert j.d_u != view.data_ptr() and j.d_gate != vec.data_ptr()
    assert torch.equal(RowNorm("affine", vec).weight, vec) and not RowNorm("affine", vec).weight.is_neg()
    n = len(calls)
    for call in (lambda: operand(6, 1).dequantize(out=view), lambda: block_join(x, x.clone(), stream_out=view)):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert len(calls) == n


def test_an_output_that_is_the_gate_of_other_rows(calls):
    """stream_out = u and normed_out = u are allowed because every value is read by the lane that writes it.  A gate per utterance
    that is u as well is read for other rows too, by workgroups that may run later."""
    c, r = 128, 6
    off = torch.tensor([0, 3, 3, 4, 5, 6, 6], dtype=torch.int32)
    u, res = torch.randn(r, c), torch.randn(r, c)
    for kw in (dict(stream_out=u, gate=u), dict(normed_out=u, gate=u), dict(stream_out=res, gate=res)):
        with pytest.raises(ValueError, match="shares memory"):
            block_join(u, res, row_off=off, **kw)
    assert not calls
    block_join(u, res, row_off=off, gate=u)                                # outputs of their own
    block_join(u, res, row_off=off, gate=torch.rand(r, c), stream_out=u)
    block_join(u, res, gate=u, stream_out=u)                               # a gate per row is read where it is written
    block_join(u, res, gate=res, stream_out=res, normed_out=u)
    block_join(u, u, gate=u, stream_out=u)
    assert len(calls) == 5


def test_one_affine_vector_is_passed_on_alone(calls, monkeypatch):
    """scale without shift, or the other way: no vector is made up for the missing one (an allocation and a launch a call)."""
    a, w, out = operand(5, 256), operand(16, 256), torch.zeros(5, 16)
    s = torch.randn(16)
    for name in ("ones", "zeros", "full", "empty"):
        monkeypatch.setattr(torch, name, None)
    for kw, want in ((dict(scale=s), (s.data_ptr(), None)), (dict(shift=s), (None, s.data_ptr())), (dict(scale=s, shift=s), 2 * (s.data_ptr(),)),
                     (dict(), (None, None))):
        block_fp8_linear(a, w, out=out, **kw)
        name, args = calls[-1]
        assert name == "sugar_fp8_linear" and args[11:13] == want and args[13] == (2 if kw else 0)


# ------------------------------------------------------------------------------------------------ the same on a GPU
def rows_of(seed, r, c, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(r, c, generator=g) * torch.exp(spread * torch.randn(c, generator=g))


@gpu
@pytest.mark.parametrize("r,n,k", [(3, 40, 300), (600, 600, 300), (301, 1536, 1536), (1204, 1530, 1536), (12000, 300, 1030), (9000, 1400, 100),
                                   (12001, 536, 528), (60000, 511, 512), (52016, 1000, 200), (23000, 1536, 1152), (44000, 776, 1400),
                                   (100001, 264, 1024)])
def test_one_affine_vector_is_the_same_as_two(r, n, k):
    """Every kernel of the product: a missing scale is 1 and a missing shift 0, bit for bit, and columns around
    the output are left alone."""
    a, w = quantize_block_fp8(rows_of(r, r, k).cuda()), quantize_block_fp8(rows_of(r + 1, n, k).cuda() / k ** 0.5)
    s, t = (rows_of(8 + i, 1, n)[0].cuda() for i in range(2))
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((r, n + 3), 7.0, dtype=dtype, device="cuda")
        for kw, both in ((dict(scale=s), (s, torch.zeros_like(s))), (dict(shift=t, relu=True), (torch.ones_like(t), t))):
            want = block_fp8_linear(a, w, scale=both[0], shift=both[1], relu=kw.get("relu", False), out_dtype=dtype)
            block_fp8_linear(a, w, out=out[:, 1:n + 1], **kw)
            assert torch.equal(out[:, 1:n + 1], want), (dtype, sorted(kw))
            assert (out[:, 0] == 7).all() and (out[:, n + 1:] == 7).all()


@gpu
def test_calls_with_their_outputs_passed_in_allocate_nothing():
    r, c, n = 300, 512, 264
    x, res = rows_of(1, r, c).bfloat16().cuda(), rows_of(2, r, c).bfloat16().cuda()
    w, s = quantize_block_fp8(rows_of(3, n, c).cuda()), rows_of(4, 1, n)[0].cuda()
    q, y, back = BlockFP8.empty(r, c, "cuda"), torch.empty(r, n, device="cuda"), torch.empty_like(x)
    norm, gate, off = RowNorm("layer", rows_of(5, 1, c)[0].cuda()), torch.rand(2, c).cuda(), torch.tensor([0, 9, r], dtype=torch.int32).cuda()
    stream, z = torch.empty_like(x), torch.empty_like(x)

    def run():
        quantize_block_fp8(x, out=q)
        q.dequantize(out=back)
        for kw in (dict(), dict(scale=s), dict(shift=s), dict(scale=s, shift=s)):
            block_fp8_linear(q, w, out=y, **kw)
        block_join(x, res, post=norm, gate=gate, row_off=off, pre=norm, stream_out=stream, normed_out=z, quantized_out=q)
    run()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    run()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


@gpu
def test_the_widest_operands():
    """2^24 - 1 columns, the most that the documentation allows; a launch of the product takes 255 such rows.  Ones, zeros and twos:
    sums below 2^24 are exact in float32, and in the 8-bit instruction too (products of 1, 2 and 4)."""
    k, r, n = (1 << 24) - 1, 300, 5
    x = torch.zeros(2, k, device="cuda", dtype=torch.bfloat16)
    x[0, ::3], x[1, -1], x[1, 7] = 1.5, -448.0, 0.25
    assert torch.equal(quantize_block_fp8(x).dequantize(torch.bfloat16), x)
    one, two = 0x38, 0x40                                                  # 1.0 and 2.0
    a, w = BlockFP8.empty(r, k, "cuda"), BlockFP8.empty(n, k, "cuda")
    for q in (a, w):
        q.data.view(torch.uint8).zero_()
        q.exponent.fill_(127)
    ab, wb = a.data.view(torch.uint8), w.data.view(torch.uint8)
    ab[:, :1 << 23] = one
    rows = torch.arange(r, device="cuda")
    ab[rows, 1000 * rows] = two
    ab[:, k - 1] = one
    ab[::2, k - 1] = two
    wb[0, :k] = one                                                        # sums of rows
    wb[1, k - 1] = one                                                     # the last column
    wb[2, 255 * 1000] = one                                                # the column of row 255, the second launch's first
    wb[3, :1 << 22] = two
    last = torch.where(rows % 2 == 0, 2.0, 1.0).double()
    want = torch.stack([(1 << 23) + 1 + last, last, 1.0 + (rows == 255), 2.0 * ((1 << 22) + (1000 * rows < 1 << 22)), 0 * last], 1)
    assert torch.equal(block_fp8_linear(a, w, out_dtype=torch.float32).double(), want)
    assert torch.equal(block_fp8_linear(a, w), want.to(torch.bfloat16))
    assert torch.equal(block_fp8_linear(a[253:257], w, out_dtype=torch.float32).double(), want[253:257])
    with pytest.raises(ValueError, match="too large"):                     # weights of 4 GiB and more
        block_fp8_linear(w, a)


@gpu
@pytest.mark.parametrize("n,k", [(5, 100), (700, 300)])
def test_row_strides_of_many_megabytes(n, k):
    """Rows 32 MiB apart: a launch takes 127 of them (32-bit offsets), by the direct kernel or in tiles.  The same rows behind one
    another, handed over in the same portions, give the same bits."""
    r, step = 300, 1 << 25
    raw = torch.zeros(r, step, dtype=torch.uint8, device="cuda")
    q = quantize_block_fp8(rows_of(1, r, k).cuda())
    width = q.data.shape[1]
    raw[:, 64:64 + width] = q.data.view(torch.uint8)
    raw[:, 4096:4100] = q.exponent
    far = BlockFP8(raw[:, 64:64 + width].view(torch.float8_e4m3fn), raw[:, 4096:4100], k)
    w = quantize_block_fp8(rows_of(2, n, k).cuda() / k ** 0.5)
    for dtype in (torch.bfloat16, torch.float32):
        want = torch.cat([block_fp8_linear(q[lo:min(lo + 127, r)], w, out_dtype=dtype) for lo in range(0, r, 127)])
        assert torch.equal(block_fp8_linear(far, w, out_dtype=dtype), want)
        assert torch.equal(far.dequantize(dtype), q.dequantize(dtype))
    raw.zero_()
    quantize_block_fp8(rows_of(1, r, k).cuda(), out=far)
    assert torch.equal(far.data.view(torch.uint8), q.data.view(torch.uint8)) and torch.equal(far.exponent, q.exponent)
