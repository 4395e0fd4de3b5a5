"""Norm on the GPU against 64 bits: widths on both sides of every kernel form, each norm before and after, gates, parts, rows
with gaps at any address, 8-bit output, rows that no norm can scale."""
import math

import pytest
import torch

import layer_refs as ref
from layer_refs import E, TORCH
from test_gpu_linear import rows

pytestmark = pytest.mark.gpu

COLS = [1, 7, 8, 9, 200, 511, 512, 513, 1024, 1025, 2048, 2056, 4095, 4097, 8193, 16385, 32769, 65536]
KINDS = [E.NORM_NONE, E.NORM_RMS, E.NORM_LAYER]


class Case:
    def __init__(self, m, cols, dtype, out=None, post=E.NORM_NONE, pre=E.NORM_RMS, parts=1, gate=None, residual=True, affine=True, gap=0,
                 shift=0, offset=0.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(m * 7919 + cols)
        t = TORCH[dtype]
        self.d = E.make_norm_desc(cols, data_type=dtype, output_type=out, parts=parts, post=post, pre=pre, rows_per_gate=gate or 0,
                                  block_scale=0.75, residual_scale=0.5)
        self.m = m
        self.y, _ = rows(g, m * parts, cols, t, gap, shift)
        self.y += offset
        self.r = rows(g, m, cols, t, gap, shift)[0] if residual else None
        self.g = None if gate is None else rows(g, -(-m // gate) if gate else 1, cols, t, gap, shift)[0]
        self.pw = torch.rand((m, parts), generator=g, device="cuda") if parts > 1 else None
        vec = lambda: torch.randn(cols, generator=g, device="cuda") if affine else None  # noqa: E731
        self.w1, self.b1, self.w2, self.b2 = vec(), vec(), vec(), vec()
        self.sum, self.sum_room = rows(g, m, cols, t, gap, shift)
        self.out, self.out_room = rows(g, m, cols, TORCH[self.d.output_type], gap, shift)
        self.sum_room.fill_(-77)
        self.out_room.fill_(-77)
        self.scale = torch.full((m,), -1.0, device="cuda")
        self.h = E.Norm(self.d)

    def strides(self):
        s = lambda t: t.stride(0) if t is not None and t.shape[0] > 1 else 0  # noqa: E731
        return {"output_stride": s(self.out), "sum_stride": s(self.sum), "block_stride": s(self.y), "residual_stride": s(self.r),
                "gate_stride": s(self.g)}

    def run(self, **kw):
        args = dict(output_scale=self.scale if self.d.output_type == E.S8 else None, sum=self.sum, residual=self.r, gate=self.g,
                    part_weights=self.pw, post_weight=self.w1, post_bias=self.b1, pre_weight=self.w2, pre_bias=self.b2, **self.strides())
        args.update(kw)
        self.h.execute(self.out, self.y, self.m, **args)

    def reference(self):
        return ref.norm(self.d, self.m, self.y, self.r, self.g, self.pw, self.w1, self.b1, self.w2, self.b2)

    def check(self):
        torch.cuda.synchronize()
        (h, eh), (o, eo) = self.reference()
        ref.close(self.sum, h, eh)
        if self.d.output_type != E.S8:
            ref.close(self.out, o, eo)
        else:
            check_codes(self.out, self.scale, o, eo)
        self.sum.fill_(-77)
        self.out.fill_(-77)
        assert (self.sum_room == -77).all() and (self.out_room == -77).all(), "written outside of the output"


def check_codes(codes, scale, o, eo):
    most = o.abs().amax(1)
    off = eo.amax(1) / 127 + 2 * ref.EPS32 * most
    assert ((scale.double() - most / 127).abs() <= off + 1e-45).all()
    # half a step from rounding, what the value itself may be off, and the code's own product in f32
    step = scale.double()[:, None]
    assert ((codes.double() * step - o).abs() <= 0.5 * step + 2 * eo + 254 * ref.EPS32 * step + 127 * off[:, None]).all()
    assert (codes != -128).all()


@pytest.mark.parametrize("dtype", [E.BF16, E.F16, E.F32])
@pytest.mark.parametrize("cols", COLS)
def test_widths(cols, dtype):
    c = Case(3, cols, dtype, post=E.NORM_RMS, pre=E.NORM_LAYER, gate=2, gap=3, shift=1)
    c.run()
    c.check()


@pytest.mark.parametrize("post", KINDS)
@pytest.mark.parametrize("pre", KINDS)
@pytest.mark.parametrize("gate, residual, parts, affine", [(None, True, 1, True), (0, False, 3, True), (1, True, 8, False), (3, True, 1, True)])
def test_kinds(post, pre, gate, residual, parts, affine):
    for dtype in (E.BF16, E.F32):
        c = Case(10, 328, dtype, post=post, pre=pre, gate=gate, residual=residual, parts=parts, affine=affine)
        c.run()
        c.check()


@pytest.mark.parametrize("dtype", [E.BF16, E.F16, E.F32])
@pytest.mark.parametrize("cols", [1, 9, 512, 700, 1433, 5000, 20000])
@pytest.mark.parametrize("pre", KINDS)
def test_codes(cols, dtype, pre):
    c = Case(5, cols, dtype, out=E.S8, pre=pre, gap=3, shift=1)
    c.run()
    c.check()


@pytest.mark.parametrize("m", [1, 2, 5, 300, 1030])
def test_rows(m):
    for cols in (64, 600, 3000):
        c = Case(m, cols, E.BF16, post=E.NORM_LAYER)
        c.run()
        c.check()


def test_a_mean_far_above_the_spread():
    """two passes over the registers: the variance of values around 1000 is not lost in their squares"""
    c = Case(4, 777, E.F32, pre=E.NORM_LAYER, residual=False, offset=1000.0)
    c.run()
    c.check()


def test_parts_of_weight_zero_are_not_read():
    c = Case(6, 200, E.BF16, parts=4)
    c.pw[:, 2] = 0
    c.pw[3] = 0   # a token that no expert took
    c.y.view(6, 4, 200)[:, 2] = math.nan
    c.y.view(6, 4, 200)[3] = math.nan
    c.run()
    c.check()


@pytest.mark.parametrize("cols", [200, 900, 3000])
@pytest.mark.parametrize("dtype", [E.BF16, E.F32])
def test_a_single_part_has_its_weight(cols, dtype):
    c = Case(9, cols, dtype, post=E.NORM_NONE, gap=3)
    w = torch.rand((9, 1), device="cuda") + 1.5
    w[4] = 0   # a row that nothing wrote: not read
    c.y[4] = math.nan
    c.run(part_weights=w)
    torch.cuda.synchronize()
    # the product that the weight makes, off by one rounding, in the block's place
    c.y[4] = 0
    p = w.double() * c.y.double()
    (h, eh), (o, eo) = ref.norm(c.d, 9, p, c.r, None, None, c.w1, c.b1, c.w2, c.b2)
    off = 2 * ref.EPS32 * c.d.block_scale * p.abs()
    ref.close(c.sum, h, eh + off)
    ref.close(c.out, *ref.one_norm(h, eh + off, c.d.pre, c.d.pre_eps, c.w2, c.b2))


def test_rows_of_zeros_and_of_what_is_no_number():
    c = Case(5, 300, E.F32, out=E.S8, pre=E.NORM_NONE, residual=False)
    c.y[0] = 0
    c.y[1, 7] = math.nan
    c.y[2, 9] = math.inf
    c.y[3] = torch.linspace(-1e-38, 1e-38, 300)
    c.run(gate=None)
    torch.cuda.synchronize()
    assert (c.out[0] == 0).all() and c.scale[0] == 0
    assert torch.isnan(c.scale[1]) and torch.isinf(c.scale[2])
    assert (c.out[3, 0], c.out[3, -1]) == (-127, 127) and (c.out[3, 150].abs() <= 1)
    (_, _), (o, eo) = c.reference()
    check_codes(c.out[4:], c.scale[4:], o[4:], eo[4:])
    # a norm of zeros is the bias; a NaN stays in its row
    c = Case(3, 300, E.F32, pre=E.NORM_RMS, residual=False)
    c.y[0] = 0
    c.y[1, 3] = math.nan
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(c.out[0], c.b2) and torch.isnan(c.out[1]).all() and torch.isfinite(c.out[2]).all()


@pytest.mark.parametrize("cols", [100, 1000, 2500])
def test_in_place(cols):
    c = Case(9, cols, E.BF16, post=E.NORM_RMS)
    (h, eh), (o, eo) = c.reference()
    c.h.execute(c.y, c.y, 9, sum=c.r, residual=c.r, post_weight=c.w1, post_bias=c.b1, pre_weight=c.w2, pre_bias=c.b2)
    ref.close(c.r, h, eh)
    ref.close(c.y, o, eo)


def test_either_output_alone():
    c = Case(4, 130, E.F16)
    c.run(sum=None)
    ref.close(c.out, *c.reference()[1])
    assert (c.sum_room == -77).all()
    c = Case(4, 130, E.F16)
    c.h.execute(None, c.y, 4, sum=c.sum, residual=c.r)
    ref.close(c.sum, *c.reference()[0])
    c.h.execute(None, None, 0)


def test_rows_past_32_bits():
    m, cols, stride = 20, 100, (1 << 32) // 10 // 2 + 3
    d = E.make_norm_desc(cols)
    room = torch.zeros(m * stride, dtype=torch.bfloat16, device="cuda").view(m, stride)
    room[:, :cols] = torch.randn(m, cols, device="cuda")
    y = room[:, :cols].clone()
    E.Norm(d).execute(room, room, m, output_stride=stride, block_stride=stride)
    ref.close(room[:, :cols], *ref.norm(d, m, y)[1])


def test_stream_and_graph():
    c = Case(33, 1500, E.BF16, post=E.NORM_RMS, gate=0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    c.run(stream=s.cuda_stream)
    s.synchronize()
    c.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        c.y.copy_(torch.randn_like(c.y))
        g.replay()
        c.check()


def test_more_rows_than_a_launch_has_threads():
    """64 threads a row: 2^26 rows and more go out in two launches"""
    m = (1 << 26) + 70
    x = torch.empty(m, dtype=torch.bfloat16, device="cuda").random_(1, 200)
    out = torch.zeros_like(x)
    E.Norm(E.make_norm_desc(1, pre=E.NORM_NONE, block_scale=0.5)).execute(out, x, m)
    assert torch.equal(out, x * 0.5)
