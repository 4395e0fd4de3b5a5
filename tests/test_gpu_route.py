"""Route on the GPU against 64 bits: choices and the slots' order exactly, weights to single precision.  Logits are distinct
multiples of a step (so that rounding decides no choice) or ties on purpose."""
import math

import pytest
import torch

import layer_refs as ref
from layer_refs import E, TORCH

pytestmark = pytest.mark.gpu


def logits(tokens, experts, dtype, seed=0, ties=False):
    g = torch.Generator()
    g.manual_seed(seed * 65537 + tokens * 1031 + experts)
    if ties:
        return torch.randint(-2, 3, (tokens, experts), generator=g).to(TORCH[dtype]).cuda()
    # distinct steps of 1 / 64 around 0: exact in bf16 up to 256 of them (|x| <= 2), in f32 always
    step = 64 if dtype != E.BF16 or experts <= 256 else 32
    x = torch.stack([torch.randperm(experts, generator=g) for _ in range(tokens)]).double()
    return ((x - experts // 2) / step).to(TORCH[dtype]).cuda()


def run(d, x, bias=None, stride=0, stream=0, plan=True):
    tokens, k = x.shape[0], d.topk
    h = E.Router(d)
    ids = torch.full((tokens, k), -9, dtype=torch.int32, device="cuda")
    weights = torch.full((tokens, k), math.nan, device="cuda")
    room = torch.full((h.plan_ints(tokens) + 8,), -9, dtype=torch.int32, device="cuda")
    h.execute(ids, weights, room if plan else None, x, tokens, bias=bias, logits_stride=stride, stream=stream)
    torch.cuda.synchronize()
    assert (room[-8:] == -9).all(), "written behind the plan"
    e = d.experts + 1
    return ids, weights, room[:e], room[e:e + tokens * k]


def check(d, x, bias=None, **kw):
    ids, weights, offsets, slots = run(d, x, bias, **kw)
    rids, rweights, roffsets, rslots = ref.route(d, x, bias)
    assert ids.tolist() == rids
    assert offsets.tolist() == roffsets
    assert slots.tolist() == rslots
    # a score is right to some ulp (exp, a sum, a division), a weight is a quotient of such a score and a sum of them
    w = torch.tensor(rweights, dtype=torch.float64)
    assert ((weights.double().cpu() - w).abs() <= 64 * ref.EPS32 * w.abs() + 1e-37).all()


# both sides of every form: experts of a lane, tokens of a workgroup
@pytest.mark.parametrize("score", [E.SCORE_SOFTMAX, E.SCORE_SIGMOID])
@pytest.mark.parametrize("tokens, experts, topk", [(1, 1, 1), (1, 5, 5), (3, 64, 1), (128, 65, 6), (129, 128, 8), (2, 129, 32), (300, 256, 4),
                                                   (130, 257, 2), (5, 512, 8), (140, 513, 3), (7, 1024, 16), (257, 1024, 2)])
def test_topk(tokens, experts, topk, score):
    for dtype in (E.F32, E.F16) if experts > 256 else (E.F32, E.F16, E.BF16):
        check(E.make_route_desc(experts, topk, logits_type=dtype, score=score, scale=1.5), logits(tokens, experts, dtype))


@pytest.mark.parametrize("experts, topk, groups, opened", [(8, 2, 4, 1), (24, 3, 3, 2), (256, 8, 8, 4), (96, 6, 32, 5), (64, 4, 64, 7), (60, 5, 5, 5),
                                                           (1000, 9, 50, 3), (36, 12, 3, 1)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("bias", [False, True])
def test_groups(experts, topk, groups, opened, best, bias):
    d = E.make_route_desc(experts, topk, score=E.SCORE_SIGMOID, groups=groups, open_groups=opened, group_best=best, renormalize=not bias)
    g = torch.Generator()
    g.manual_seed(experts)
    b = (torch.randint(-3, 4, (experts,), generator=g) * 0.3).cuda() if bias else None
    for tokens in (9, 200):
        x = logits(tokens, experts, E.F32)
        x = x / x.abs().max() * 4 if experts > 500 else x   # sigmoid stays apart in single precision
        x = x + 0.5   # around 0, sigmoid(a) + sigmoid(-a) would be a tie of groups that rounding breaks
        check(d, x, b)


@pytest.mark.parametrize("tokens", [6, 500])
@pytest.mark.parametrize("groups, opened", [(1, 1), (8, 3)])
def test_ties_go_to_the_lowest_index(tokens, groups, opened):
    for score in (E.SCORE_SOFTMAX, E.SCORE_SIGMOID):
        d = E.make_route_desc(72, 7, logits_type=E.BF16, score=score, groups=groups, open_groups=opened)
        check(d, logits(tokens, 72, E.BF16, ties=True))


@pytest.mark.parametrize("tokens", [5, 150])
@pytest.mark.parametrize("score", [E.SCORE_SOFTMAX, E.SCORE_SIGMOID])
def test_closed_experts(tokens, score):
    x = logits(tokens, 40, E.F32)
    x[0] = -math.inf                       # no expert at all
    x[1, 3:] = math.nan                    # fewer than topk
    x[2, :39] = -math.inf
    x[3, 7] = math.inf
    x[4] = torch.finfo(torch.float32).min  # the type's lowest value closes nothing
    x[4, 11] = -math.inf
    for groups, opened in ((1, 1), (4, 2)):
        check(E.make_route_desc(40, 6, score=score, groups=groups, open_groups=opened, group_best=2), x)
    b = torch.zeros(40, device="cuda")
    b[5], b[6] = -math.inf, math.nan       # closed to every token
    check(E.make_route_desc(40, 6, score=score), x, b)


def test_rows_with_gaps_and_no_plan():
    room = torch.full((200, 37), math.nan, dtype=torch.float16, device="cuda")
    room[:, :33] = logits(200, 33, E.F16)
    d = E.make_route_desc(33, 4, logits_type=E.F16)
    check(d, room[:, :33], stride=37)
    ids, weights, offsets, _ = run(d, room[:, :33], stride=37, plan=False)
    rids, _, _, _ = ref.route(d, room[:, :33])
    assert ids.tolist() == rids and (offsets == -9).all()


def test_no_tokens_is_an_empty_plan():
    h = E.Router(E.make_route_desc(8, 2))
    plan = torch.full((h.plan_ints(0),), -9, dtype=torch.int32, device="cuda")
    h.execute(None, None, plan, None, 0)
    assert plan.tolist() == [0] * 9
    h.execute(None, None, None, None, 0)


def test_many_tokens_streams_and_graph():
    d = E.make_route_desc(64, 4, logits_type=E.BF16)
    x = logits(5000, 64, E.BF16)
    check(d, x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    check(d, x, stream=s.cuda_stream)
    h = E.Router(d)
    for tokens in (100, 1000):
        x = logits(tokens, 64, E.BF16)
        ids = torch.empty((tokens, 4), dtype=torch.int32, device="cuda")
        w, plan = torch.empty((tokens, 4), device="cuda"), torch.empty(h.plan_ints(tokens), dtype=torch.int32, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h.execute(ids, w, plan, x, tokens, stream=torch.cuda.current_stream().cuda_stream)
        for i in range(3):
            x.copy_(logits(tokens, 64, E.BF16, seed=i + 1))
            plan.fill_(-9)
            g.replay()
            torch.cuda.synchronize()
            rids, _, roffsets, rslots = ref.route(d, x)
            assert ids.tolist() == rids and plan[:65].tolist() == roffsets and plan[65:65 + 4 * tokens].tolist() == rslots
