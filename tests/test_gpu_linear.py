"""Linear and the experts' products on the GPU against 64 bits: every kernel, type and epilogue at the sizes where a tile, a
chunk of K or a vector ends, rows with gaps, any alignment.  What lies around the tensors is NaN or a mark, so that a read or a
write past an edge shows."""
import ctypes
import math

import pytest
import torch

import layer_refs as ref
from layer_refs import E, TORCH

pytestmark = pytest.mark.gpu

# rows x inputs x outputs: one of everything; the last chunk of K whole, ragged by a 16-byte part and by an element; the last
# column alone; both sides of the row counts at which another kernel takes over
SIZES = [(1, 1, 1), (1, 64, 64), (2, 33, 17), (15, 200, 31), (16, 512, 130), (17, 63, 65), (32, 520, 64), (33, 129, 33), (64, 1000, 200),
         (65, 257, 40), (129, 96, 300), (193, 64, 257), (257, 328, 70), (300, 129, 513), (515, 640, 1000)]
TYPES = [E.BF16, E.F16, E.S8]


def rows(g, m, n, dtype, gap, shift, scale=1.0):
    """m rows of n values in a buffer that is NaN (8 bits: 99) elsewhere: `gap` values between rows, from element `shift` on"""
    if dtype == torch.int8:
        v = torch.randint(-127, 128, (m, n), generator=g, device="cuda").to(torch.int8)
    else:
        v = (torch.randn((m, n), generator=g, device="cuda") * scale).to(dtype)
    room = torch.full((shift + m * (n + gap) + 64,), 99 if dtype == torch.int8 else math.nan, dtype=dtype, device="cuda")
    t = room[shift:shift + m * (n + gap)].view(m, n + gap)[:, :n]
    t.copy_(v)
    return t, room


class Case:
    def __init__(self, m, ic, oc, itype, otype, activation=E.ACT_NONE, gated=False, bias=False, residual=False, experts=1, gap=0, shift=0,
                 seed=0, in_rows=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed * 1000003 + m * 10007 + ic * 101 + oc)
        self.d = E.make_linear_desc(ic, oc, experts=experts, input_type=itype, output_type=otype, activation=activation, gated=gated,
                                    with_bias=bias, with_residual=residual, residual_scale=0.5)
        n2 = oc * (2 if gated else 1)
        self.m, self.gap, self.shift, self.otype = m, gap, shift, TORCH[otype]
        n_in = m if in_rows is None else in_rows
        self.x, self.x_room = rows(g, n_in, ic, TORCH[itype], gap, shift)
        self.w, _ = rows(g, experts * n2, ic, TORCH[itype], 0, 0, ic ** -0.5)
        self.xs = self.ws = self.b = self.r = None
        if itype == E.S8:
            self.xs = torch.rand(n_in, generator=g, device="cuda") / 64
            self.ws = torch.rand(experts * n2, generator=g, device="cuda") / 64 * ic ** -0.5
        if bias:
            self.b = torch.randn(experts * n2, generator=g, device="cuda")
        if residual:
            self.r, _ = rows(g, m, oc, self.otype, gap, shift)
        self.out, self.out_room = rows(g, m, oc, self.otype, gap, shift)
        self.out_room.fill_(-77)
        self.h = E.Linear(self.d)
        self.h.prepare(self.w, bias=self.b, scale=self.ws)

    def run(self, out=None, stream=0):
        self.h.execute(self.out if out is None else out, self.x, self.m, input_scale=self.xs, residual=self.r,
                       output_stride=self.out.stride(0) if self.m > 1 else 0, input_stride=self.x.stride(0) if self.m > 1 else 0,
                       residual_stride=0 if self.r is None or self.m == 1 else self.r.stride(0), stream=stream)

    def check(self):
        torch.cuda.synchronize()
        ref.close(self.out, *ref.linear(self.x, self.w, self.d, self.b, self.xs, self.ws, self.r))
        self.out.fill_(-77)
        assert (self.out_room == -77).all(), "written outside of the output"


@pytest.mark.parametrize("itype", TYPES)
@pytest.mark.parametrize("m, ic, oc", SIZES)
def test_product(m, ic, oc, itype):
    c = Case(m, ic, oc, itype, E.F32)
    c.run()
    c.check()


@pytest.mark.parametrize("itype, otype", [(E.BF16, E.BF16), (E.BF16, E.F16), (E.F16, E.F16), (E.S8, E.BF16), (E.S8, E.F16)])
@pytest.mark.parametrize("m, ic, oc", SIZES[2:])
def test_rows_with_gaps_at_any_address(m, ic, oc, itype, otype):
    c = Case(m, ic, oc, itype, otype, bias=True, residual=True, gap=5, shift=3)
    c.run()
    c.check()


@pytest.mark.parametrize("activation", [E.ACT_NONE, E.ACT_RELU, E.ACT_GELU, E.ACT_SILU])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m, ic, oc", [(1, 96, 35), (20, 200, 64), (50, 130, 129), (200, 96, 35), (260, 264, 300)])
def test_epilogues(m, ic, oc, gated, activation):
    for itype, otype, bias, residual in ((E.BF16, E.F32, True, True), (E.S8, E.BF16, True, False), (E.F16, E.F16, False, True)):
        c = Case(m, ic, oc, itype, otype, activation=activation, gated=gated, bias=bias, residual=residual, gap=3)
        c.run()
        c.check()


@pytest.mark.parametrize("form", range(9))
@pytest.mark.parametrize("itype", TYPES)
@pytest.mark.parametrize("m, ic, oc, gap", [(7, 520, 70, 0), (70, 704, 150, 8), (140, 333, 77, 3), (290, 1280, 260, 0)])
def test_every_form(m, ic, oc, gap, itype, form, monkeypatch):
    """the kernel forms at sizes that the choice would not give them; rows at multiples of 16 bytes and others"""
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    for gated in (False, True):
        c = Case(m, ic, oc, itype, E.BF16 if gated else E.F32, activation=E.ACT_GELU, gated=gated, bias=True, residual=True, gap=gap)
        c.run()
        c.check()


@pytest.mark.parametrize("form", range(9))
def test_experts_in_every_form(form, monkeypatch):
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    test_experts(400, 5, 2, 264, 130, E.BF16, "up")
    test_experts(60, 9, 3, 96, 48, E.S8, "down")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_residual_in_place(m):
    c = Case(m, 192, 100, E.BF16, E.BF16, residual=True, gap=4)
    c.out.copy_(c.r)
    before = c.out.clone()
    c.h.execute(c.out, c.x, m, residual=c.out, output_stride=104, input_stride=196, residual_stride=104)
    ref.close(c.out, *ref.linear(c.x, c.w, c.d, residual=before))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_infinities_and_nan_stay_in_their_rows(m):
    c = Case(m, 100, 48, E.BF16, E.F32)
    c.x[0, 5] = math.nan
    c.x[m - 1, 99] = math.inf
    c.run()
    torch.cuda.synchronize()
    assert torch.isnan(c.out[0]).all()
    assert (torch.isinf(c.out[m - 1]) | torch.isnan(c.out[m - 1]) | (c.w[:, 99] == 0)).all()
    ref.close(c.out[1:m - 1], *ref.linear(c.x[1:m - 1], c.w, c.d))


def test_no_rows_is_no_call():
    c = Case(1, 8, 8, E.BF16, E.BF16)
    c.h.execute(None, None, 0)
    assert (c.out_room == -77).all()


@pytest.mark.parametrize("m", [20, 300])
def test_rows_past_32_bits(m):
    """the last rows start more than 2^32 bytes behind the first"""
    ic, oc, stride = 64, 40, (1 << 32) // (m - 10) // 2 + 8
    d = E.make_linear_desc(ic, oc)
    x = torch.zeros(m * stride, dtype=torch.bfloat16, device="cuda").view(m, stride)
    out = torch.zeros(m * stride, dtype=torch.bfloat16, device="cuda").view(m, stride)
    x[:, :ic] = torch.randn(m, ic, device="cuda")
    w = torch.randn(oc, ic, device="cuda").bfloat16()
    h = E.Linear(d)
    h.prepare(w)
    h.execute(out, x, m, output_stride=stride, input_stride=stride)
    ref.close(out[:, :oc], *ref.linear(x[:, :ic], w, d))


def test_streams_and_graph():
    """executes of one handle on two streams at once, and a captured one replayed on new inputs"""
    cases = [Case(m, 256, 192, E.BF16, E.BF16, bias=True, activation=E.ACT_SILU, gated=True, seed=s) for s, m in enumerate((5, 48, 400))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in cases:
        outs = [torch.empty_like(c.out) for _ in streams]
        for _ in range(8):
            for s, o in zip(streams, outs):
                c.run(out=o, stream=s.cuda_stream)
        c.run()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o.view(torch.int16), c.out.contiguous().view(torch.int16))
        c.check()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run(stream=torch.cuda.current_stream().cuda_stream)
        for i in range(3):
            c.x.copy_(torch.randn_like(c.x.float()).to(c.x.dtype))
            g.replay()
            c.check()


def plan(g, tokens, experts, topk, empty=(), dropped=0):
    """ids of a routing, its slots in expert order (-1 behind the last) and offsets"""
    ids = torch.stack([torch.randperm(experts, generator=g)[:topk] for _ in range(tokens)]).reshape(-1)
    ids = torch.where(torch.tensor([int(i) in empty for i in ids]), torch.tensor(-1), ids)
    ids[:dropped] = -1
    key = torch.where(ids < 0, experts, ids)
    order = key.argsort(stable=True)
    live = int((ids >= 0).sum())
    slots = order.clone()
    slots[live:] = -1
    offsets = torch.searchsorted(key[order], torch.arange(experts + 1))
    return slots.int().cuda(), offsets.int().cuda(), ids


@pytest.mark.parametrize("itype", TYPES)
@pytest.mark.parametrize("tokens, experts, topk, ic, oc", [(1, 4, 2, 64, 40), (16, 8, 3, 200, 65), (50, 3, 2, 129, 100), (400, 70, 4, 96, 48),
                                                           (700, 3, 2, 264, 130), (600, 2, 1, 100, 70)])
@pytest.mark.parametrize("side", ["up", "down"])
def test_experts(tokens, experts, topk, ic, oc, itype, side):
    g = torch.Generator()
    g.manual_seed(tokens)
    slots, offsets, _ = plan(g, tokens, experts, topk, empty=(1,), dropped=topk)
    count = tokens * topk
    up = side == "up"
    c = Case(count, ic, oc, itype, E.BF16 if itype != E.F16 else E.F16, activation=E.ACT_SILU if up else E.ACT_NONE, gated=up, bias=True,
             experts=experts, in_rows=tokens if up else count, gap=3)
    c.h.execute_experts(c.out, c.x, slots, offsets, count, topk, input_scale=c.xs, input_rows=E.ROWS_TOKEN if up else E.ROWS_SORTED,
                        output_rows=E.ROWS_SORTED if up else E.ROWS_SLOT, output_stride=c.out.stride(0), input_stride=c.x.stride(0))
    torch.cuda.synchronize()
    n2, ends = c.w.shape[0] // experts, offsets.tolist()
    for e in range(experts):
        p = torch.arange(ends[e], ends[e + 1], device="cuda")
        if not len(p):
            continue
        s = slots[p].long()
        x = s // topk if up else p
        o = p if up else s
        part = slice(e * n2, (e + 1) * n2)
        ref.close(c.out[o], *ref.linear(c.x[x], c.w[part], c.d, c.b[part], None if c.xs is None else c.xs[x], None if c.ws is None else c.ws[part]))
        c.out[o] = -77
    assert (c.out_room == -77).all(), "a row was written that no position leads to"


def test_experts_with_slots_out_of_range():
    """slots and offsets come from memory: what is out of range is neither read nor written"""
    experts, tokens, topk, ic, oc = 3, 8, 2, 64, 48
    c = Case(16, ic, oc, E.BF16, E.BF16, experts=experts)
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    slots[2], slots[7] = -5, 1 << 30
    offsets = torch.tensor([-4, 6, 3, 1 << 20], dtype=torch.int32, device="cuda")
    c.h.execute_experts(c.out, c.x, slots, offsets, 16, topk, input_rows=E.ROWS_SLOT, output_rows=E.ROWS_SLOT)
    torch.cuda.synchronize()
    assert (c.out[2] == -77).all() and (c.out[7] == -77).all()
    ref.close(c.out[:2], *ref.linear(c.x[:2], c.w[:oc], c.d))
    ref.close(c.out[8:], *ref.linear(c.x[8:], c.w[2 * oc:], c.d))
    c.out.fill_(-77)
    assert (c.out_room == -77).all()


def test_calls_are_checked_before_a_launch():
    h = E.Linear(E.make_linear_desc(64, 32, input_type=E.S8, with_bias=True, with_residual=True))
    with pytest.raises(E.EulerHipError, match="not prepared"):
        h.execute(256, 256, 4)
    w, s = torch.zeros((32, 64), dtype=torch.int8, device="cuda"), torch.zeros(32, device="cuda")
    for kw, match in (({"bias": s}, "scale per row"), ({"scale": s}, "no bias"), ({"scale": s.data_ptr() + 2, "bias": s}, "multiple")):
        with pytest.raises(E.EulerHipError, match=match):
            h.prepare(w, **kw)
    h.prepare(w, scale=s, bias=s)
    for args, kw, match in (((256, 256, 4), {"input_scale": 256}, "null"), ((256, 256, 4), {"residual": 256}, "null"),
                            ((256, 256, -1), {}, "rows"), ((256, 256, 1 << 31), {}, "rows"), ((256, 256, 4), {"input_stride": 63}, "stride"),
                            ((257, 256, 4), {"input_scale": 256, "residual": 256}, "multiple")):
        with pytest.raises(E.EulerHipError, match=match):
            h.execute(*args, **kw)
    h = E.Linear(E.make_linear_desc(64, 32, experts=2))
    h.prepare(torch.zeros((2, 32, 64), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(E.EulerHipError, match="offsets"):
        h.execute(256, 256, 4)
    for args, kw, match in (((256, 256, 256, 256, 5, 2), {}, "topk"), ((256, 256, 256, 256, 4, 0), {}, "topk"), ((256, 256, None, 256, 4, 2), {}, "null"),
                            ((256, 256, 256, 256, 4, 2), {"input_rows": 3}, "input rows"), ((256, 256, 256, 256, 4, 2), {"output_rows": 1}, "output rows"),
                            ((256, 256, 256, 256, 1 << 30, 2), {}, "2\\^30"), ((256, 256, 258, 256, 4, 2), {}, "multiple")):
        with pytest.raises(E.EulerHipError, match=match):
            h.execute_experts(*args, **kw)
    torch.cuda.synchronize()


def test_tensors_without_a_use_are_refused():
    """not left out without a word"""
    w, v = torch.zeros((32, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros(32, device="cuda")
    x, out = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((4, 32), dtype=torch.bfloat16, device="cuda")
    plain = E.Linear(E.make_linear_desc(64, 32))
    for kw, match in (({"bias": v}, "not with_bias"), ({"scale": v}, "s8 weights")):
        with pytest.raises(E.EulerHipError, match=match):
            plain.prepare(w, **kw)
    plain.prepare(w)
    for kw, match in (({"residual": out}, "not with_residual"), ({"input_scale": v}, "s8 rows")):
        with pytest.raises(E.EulerHipError, match=match):
            plain.execute(out, x, 4, **kw)
    experts = E.Linear(E.make_linear_desc(64, 32, experts=2))
    experts.prepare(torch.zeros((2, 32, 64), dtype=torch.bfloat16, device="cuda"))
    slots, offsets = torch.arange(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(E.EulerHipError, match="s8 rows"):
        experts.execute_experts(out, x, slots, offsets, 4, 2, input_scale=v)

    class Args(ctypes.Structure):   # ehip_linear_args_t: what the Python call has no names for
        _fields_ = [(k, ctypes.c_void_p) for k in ("output", "input", "input_scale", "residual", "slots", "offsets")] + [
            (k, ctypes.c_int64) for k in ("rows", "output_stride", "input_stride", "residual_stride")] + [
            (k, ctypes.c_int32) for k in ("topk", "input_rows", "output_rows")]

    for kw in ({"slots": slots.data_ptr()}, {"offsets": offsets.data_ptr()}):
        args = Args(output=out.data_ptr(), input=x.data_ptr(), rows=4, **kw)
        assert E.lib.ehip_linear_execute(plain._h, ctypes.byref(args), None) == E.EHIP_GENERAL_ERROR
    args = Args(output=out.data_ptr(), input=x.data_ptr(), rows=4, residual=out.data_ptr(), slots=slots.data_ptr(), offsets=offsets.data_ptr(), topk=2)
    assert E.lib.ehip_linear_execute_experts(experts._h, ctypes.byref(args), None) == E.EHIP_GENERAL_ERROR
    plain.execute(out, x, 4)
    torch.cuda.synchronize()


FORMS = ["k_linear_split<1x1>", "k_linear_split<2x1>", "k_linear_split<4x1>", "k_linear_split<2x2>", "k_linear_split<4x2>", "k_linear_split<4x4>",
         "k_linear_tile<128x128>", "k_linear_tile<128x128, deep>", "k_linear_tile<256x256>"]


@pytest.mark.parametrize("otype, residual, gated", [(E.F32, True, False), (E.BF16, False, False), (E.F32, True, True), (E.BF16, True, True)])
@pytest.mark.parametrize("m, ic, oc", [(2048, 256, 512), (853, 704, 3392), (16, 1024, 512), (40, 512, 4096), (300, 1001, 640)])
def test_the_name_is_of_the_kernel_that_runs(m, ic, oc, otype, residual, gated, monkeypatch):
    """forms that share K out differently add in another order: the bits are those of the form that the name says"""
    monkeypatch.delenv("EHIP_LINEAR_FORM", raising=False)
    c = Case(m, ic, oc, E.BF16, otype, residual=residual, gated=gated)
    c.run()
    name = c.h.kernel_name(m)
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(FORMS.index(name)))
    named = Case(m, ic, oc, E.BF16, otype, residual=residual, gated=gated)
    named.run()
    torch.cuda.synchronize()
    assert named.h.kernel_name(m) == name
    assert torch.equal(named.out, c.out), name
    c.check()
    if ic % 8:   # rows that end at other bytes than multiples of 16
        assert name != "k_linear_tile<128x128, deep>"


@pytest.mark.parametrize("form, m", [(5, (1 << 29) + 70), (6, (1 << 31) - 1), (8, (1 << 31) - 1)])
def test_more_rows_than_a_launch_has_threads(form, m, monkeypatch):
    """a launch's threads are counted in 32 bits: more workgroups than that go out in several"""
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    h = E.Linear(E.make_linear_desc(1, 1))
    h.prepare(torch.full((1,), 0.5, dtype=torch.bfloat16, device="cuda"))
    x = torch.empty(m, dtype=torch.bfloat16, device="cuda").random_(1, 200)
    out = torch.zeros_like(x)
    h.execute(out, x, m)
    assert torch.equal(out, x * 0.5)


def test_more_weights_than_a_launch_has_threads():
    """64 GiB of packed weights: a thread packs 16 bytes of them"""
    experts, oc = 32, 1 << 24
    w = torch.empty((experts, oc), dtype=torch.bfloat16, device="cuda").random_(1, 200)
    h = E.Linear(E.make_linear_desc(1, oc, experts=experts))
    h.prepare(w)
    x = torch.tensor([[0.5], [2.0], [1.0]], dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((3, oc), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0] + [1] * 30 + [2, 3], dtype=torch.int32, device="cuda")   # experts 0, 30 and 31
    h.execute_experts(out, x, slots, offsets, 3, 1)
    torch.cuda.synchronize()
    for i, e in enumerate((0, 30, 31)):
        assert torch.equal(out[i], w[e] * x[i])
    h.close()


def act_alone(d, kind, otype):
    """(value, error) of an activation by itself, relative to the value also where that is tiny.  Units are 2^-24.
    GELU max(v, 0) - t: f32 results, t off by 16 + 2 v^2 units of itself (fit 1, Horner's last steps 2, t's argument and its reciprocal
    3, counted 2.3 times, the exponential 2, products 3; the exponent 2.5, v^2 / 2 times); 16-bit results, by the fit's 1.3e-4 of
    itself and no more than 3.3 units of |v|, and by 14 (1 + v^2) units (the partial sums of the exponent's polynomial, carried on,
    and the exponential's 2); one subtraction.
    SiLU: 8 + 2 |v| units (the exponential 2, a sum, its reciprocal 2, a product; the exponent 1.5, |v| times).
    Exponentials and reciprocals below 2^-126 are 0."""
    u, least = ref.EPS32, 2.0 ** -125 * d.abs().clamp(max=100)
    if kind == E.ACT_GELU:
        t = 0.5 * d.abs() * torch.erfc(d.abs() * math.sqrt(0.5))
        want = d.clamp(min=0) - t
        own = (16 + 2 * d * d) * u * t if otype == E.F32 else torch.minimum(1.3e-4 * t, 3.3 * u * d.abs()) + (2 + 14 * (1 + d * d)) * u * t
        return want, own + 2 * u * want.abs() + least
    if kind == E.ACT_SILU:
        want = d * torch.sigmoid(d)
        return want, (8 + 2 * d.abs()) * u * want.abs() + least
    return (d.clamp(min=0) if kind == E.ACT_RELU else d), torch.zeros_like(d)


@pytest.mark.parametrize("form", [1, 5, 7, 8])
@pytest.mark.parametrize("otype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", [E.ACT_NONE, E.ACT_RELU, E.ACT_GELU, E.ACT_SILU])
def test_activations_keep_their_digits(activation, gated, otype, form, monkeypatch):
    """the function by itself, on biases: an output a value; gated, with partners that lift tiny values to about 1"""
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    v = torch.cat([torch.linspace(-16, 16, 20011), torch.linspace(-60, 60, 2001), torch.linspace(-0.3, 0.3, 3001), torch.logspace(-30, 0, 400),
                   -torch.logspace(-30, 0, 400), torch.tensor([0.0, -100.0, 1e30, -1e30, 3e38, -3e38])]).cuda()
    n = len(v)
    want, off = act_alone(v.double(), activation, otype)
    bias = v
    if gated:
        partner = torch.where(want.abs() > 1e-34, 1 / want, torch.ones_like(want)).clamp(-1e35, 1e35).float()
        bias = torch.cat([v, partner])
        want, off = want * partner.double(), off * partner.double().abs() + 2 * ref.EPS32 * (want * partner.double()).abs()
    h = E.Linear(E.make_linear_desc(1, n, output_type=otype, activation=activation, gated=gated, with_bias=True))
    h.prepare(torch.ones((len(bias), 1), dtype=torch.bfloat16, device="cuda"), bias=bias)
    x, out = torch.zeros((3, 1), dtype=torch.bfloat16, device="cuda"), torch.full((3, n), math.nan, dtype=TORCH[otype], device="cuda")
    h.execute(out, x, 3)
    torch.cuda.synchronize()
    # (past the largest f16 values are infinite)
    fits = want.abs() < (65504 if otype == E.F16 else 3e38)
    for row in out:
        ref.close(row[fits], want[fits], off[fits])


def exact_rows(g, *shape, dtype=torch.bfloat16):
    """small whole numbers: every sum of their products is exact in f32 and s32, in any order"""
    return torch.randint(-4, 5, shape, generator=g, device="cuda").to(dtype)


# Runs of 128-byte steps of K for each of eight waves: the loops of every form in several turns with every remainder; waves with
# fewer steps than others, with none; a part of a step behind the last
@pytest.mark.parametrize("form", range(9))
@pytest.mark.parametrize("itype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("steps, tail", [(33, 0), (40, 5), (41, 0), (48, 16), (50, 1), (56, 0), (61, 8), (64, 63), (72, 3), (77, 0)])
def test_every_step_of_a_long_sum_counts_once(steps, tail, gated, itype, form, monkeypatch):
    """bit for bit: a step that is dropped, repeated or taken from another's registers cannot hide in a bound"""
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    g = torch.Generator(device="cuda")
    g.manual_seed(steps * 100 + tail)
    ic, m, oc = steps * (128 if itype == E.S8 else 64) + tail, 37, 70
    n2 = 2 * oc if gated else oc
    x, w = exact_rows(g, m, ic, dtype=TORCH[itype]), exact_rows(g, n2, ic, dtype=TORCH[itype])
    ones = torch.ones(max(m, n2), device="cuda") if itype == E.S8 else None
    h = E.Linear(E.make_linear_desc(ic, oc, input_type=itype, output_type=E.F32, gated=gated))
    h.prepare(w, scale=ones)
    out = torch.full((m, oc), math.nan, device="cuda")
    h.execute(out, x, m, input_scale=ones)
    a = x.double() @ w.double().t().contiguous()
    want = a[:, :oc] * a[:, oc:] if gated else a
    assert torch.equal(out, want.float())


@pytest.mark.parametrize("form", range(9))
@pytest.mark.parametrize("itype", TYPES)
@pytest.mark.parametrize("steps, tail", [(36, 0), (45, 7), (70, 0)])
def test_every_step_of_the_experts_long_sums_counts_once(steps, tail, itype, form, monkeypatch):
    monkeypatch.setenv("EHIP_LINEAR_FORM", str(form))
    g = torch.Generator()
    g.manual_seed(steps)
    tokens, experts, topk, oc = 60, 5, 2, 70
    slots, offsets, ids = plan(g, tokens, experts, topk, empty=(3,))
    g = torch.Generator(device="cuda")
    g.manual_seed(steps)
    ic = steps * (128 if itype == E.S8 else 64) + tail
    for gated in (True, False):
        n2 = 2 * oc if gated else oc
        x, w = exact_rows(g, tokens, ic, dtype=TORCH[itype]), exact_rows(g, experts, n2, ic, dtype=TORCH[itype])
        ones = torch.ones(max(tokens, experts * n2), device="cuda") if itype == E.S8 else None
        h = E.Linear(E.make_linear_desc(ic, oc, experts, itype, E.F32, gated=gated))
        h.prepare(w, scale=ones)
        out = torch.full((tokens * topk, oc), -7.0, device="cuda")
        h.execute_experts(out, x, slots, offsets, tokens * topk, topk, input_scale=ones, input_rows=E.ROWS_TOKEN, output_rows=E.ROWS_SLOT)
        for s, e in enumerate(ids.tolist()):
            if e < 0:
                assert (out[s] == -7).all()
        live = (ids >= 0).cuda()
        at = ids.clamp(min=0).cuda()
        a = torch.zeros((tokens * topk, n2), dtype=torch.float64, device="cuda")
        for e in range(experts):
            here = live & (at == e)
            a[here] = x[torch.arange(tokens * topk, device="cuda")[here] // topk].double() @ w[e].double().t().contiguous()
        want = a[:, :oc] * a[:, oc:] if gated else a
        assert torch.equal(out[live], want[live].float())


@pytest.mark.parametrize("itype, m, ic, oc", [(E.BF16, 1, 4096, 4096), (E.F16, 64, 2048, 1000), (E.S8, 16, 4096, 4096), (E.BF16, 1024, 4096, 1000),
                                              (E.S8, 1500, 4104, 1000), (E.F16, 2100, 4096, 2048)])
def test_products_of_a_models_size(itype, m, ic, oc):
    """the forms that these sizes take, on whole numbers, bit for bit, and on ordinary values within single precision's error"""
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    x, w = exact_rows(g, m, ic, dtype=TORCH[itype]), exact_rows(g, oc, ic, dtype=TORCH[itype])
    ones = torch.ones(max(m, oc), device="cuda") if itype == E.S8 else None
    h = E.Linear(E.make_linear_desc(ic, oc, input_type=itype, output_type=E.F32))
    h.prepare(w, scale=ones)
    out = torch.full((m, oc), math.nan, device="cuda")
    h.execute(out, x, m, input_scale=ones)
    assert torch.equal(out, (x.double() @ w.double().t().contiguous()).float())
    c = Case(m, ic, oc, itype, E.F32, bias=True, residual=True)
    c.run()
    torch.cuda.synchronize()
    if itype != E.S8:
        # at most ic sums, each off by 2^-23 of a partial sum, which is within 6 of its deviation (the root of the products' squares);
        # independent errors add by squares
        want, _ = ref.linear(c.x, c.w, c.d, c.b, None, None, c.r)
        size = ((c.x.double() ** 2) @ (c.w.double() ** 2).t().contiguous()).sqrt() + c.b.double().abs() + c.r.double().abs()
        assert ((c.out.double() - want).abs() / size).max() <= 6 * 2 * ref.EPS32 * math.sqrt(ic)
    c.check()
