"""What linear, norm, route and experts refuse, and how their calls take arguments: host logic, no GPU."""
import ctypes

import numpy as np
import pytest

from layer_refs import E


def refuses(cls, desc, code, match):
    with pytest.raises(E.EulerHipError, match=match) as e:
        cls(desc)
    assert e.value.code == code


@pytest.mark.parametrize("kw, code, match", [
    (dict(ic=0), E.EHIP_GENERAL_ERROR, "ic and oc"), (dict(oc=(1 << 24) + 1), E.EHIP_GENERAL_ERROR, "ic and oc"),
    (dict(experts=0), E.EHIP_GENERAL_ERROR, "experts"), (dict(experts=1025), E.EHIP_GENERAL_ERROR, "experts"),
    (dict(input_type=E.F32), E.EHIP_UNIMPLEMENTED, "input"), (dict(input_type=E.U8), E.EHIP_UNIMPLEMENTED, "input"),
    (dict(output_type=E.S8), E.EHIP_UNIMPLEMENTED, "output"), (dict(activation=9), E.EHIP_UNIMPLEMENTED, "activation"),
    (dict(gated=2), E.EHIP_GENERAL_ERROR, "flags"), (dict(experts=2, with_residual=True), E.EHIP_UNIMPLEMENTED, "residual"),
    (dict(input_type=E.S8, ic=131072), E.EHIP_UNIMPLEMENTED, "131071"), (dict(ic=1 << 24, oc=1 << 24, experts=1024), E.EHIP_UNIMPLEMENTED, "too large")])
def test_linear_descriptors(kw, code, match):
    refuses(E.Linear, E.make_linear_desc(**{"ic": 64, "oc": 64, **kw}), code, match)


@pytest.mark.parametrize("kw, code, match", [
    (dict(cols=0), E.EHIP_GENERAL_ERROR, "cols"), (dict(cols=65537), E.EHIP_UNIMPLEMENTED, "65536"), (dict(parts=0), E.EHIP_GENERAL_ERROR, "parts"),
    (dict(parts=65), E.EHIP_UNIMPLEMENTED, "parts"), (dict(data_type=E.U8), E.EHIP_UNIMPLEMENTED, "data"),
    (dict(output_type=E.F32), E.EHIP_UNIMPLEMENTED, "output"), (dict(post=3), E.EHIP_UNIMPLEMENTED, "kind"), (dict(pre=-1), E.EHIP_UNIMPLEMENTED, "kind"),
    (dict(rows_per_gate=-1), E.EHIP_GENERAL_ERROR, "rows_per_gate"), (dict(pre_eps=-1.0), E.EHIP_GENERAL_ERROR, "eps"),
    (dict(post_eps=float("nan")), E.EHIP_GENERAL_ERROR, "eps")])
def test_norm_descriptors(kw, code, match):
    refuses(E.Norm, E.make_norm_desc(**{"cols": 64, **kw}), code, match)


@pytest.mark.parametrize("kw, code, match", [
    (dict(topk=0), E.EHIP_GENERAL_ERROR, "topk"), (dict(topk=65), E.EHIP_GENERAL_ERROR, "topk"), (dict(topk=33), E.EHIP_UNIMPLEMENTED, "32 choices"),
    (dict(experts=1025), E.EHIP_UNIMPLEMENTED, "1024"), (dict(groups=5), E.EHIP_GENERAL_ERROR, "groups"), (dict(groups=4, open_groups=5), E.EHIP_GENERAL_ERROR, "groups"),
    (dict(experts=130, groups=65), E.EHIP_UNIMPLEMENTED, "64 groups"), (dict(group_best=3), E.EHIP_UNIMPLEMENTED, "group_best"),
    (dict(logits_type=E.S8), E.EHIP_UNIMPLEMENTED, "logits"), (dict(score=2), E.EHIP_UNIMPLEMENTED, "score"), (dict(renormalize=3), E.EHIP_GENERAL_ERROR, "flags")])
def test_route_descriptors(kw, code, match):
    refuses(E.Router, E.make_route_desc(**{"experts": 64, "topk": 2, **kw}), code, match)


def test_descriptors_mirror_the_header():
    assert ctypes.sizeof(E.LinearDesc) == 40 and ctypes.sizeof(E.NormDesc) == 44 and ctypes.sizeof(E.RouteDesc) == 36


def test_norm_calls_are_checked_before_a_launch():
    h = E.Norm(E.make_norm_desc(64))
    for args, kw, match in (((256, None, 4), {}, "null"), ((None, 256, 4), {}, "null"), ((256, 256, -1), {}, "rows"), ((256, 256, 1 << 31), {}, "rows"),
                            ((256, 256, 4), {"block_stride": 63}, "stride"), ((256, 256, 4), {"output_stride": -64}, "stride"),
                            ((257, 256, 4), {}, "multiple"), ((256, 256, 4), {"pre_weight": 2}, "multiple")):
        with pytest.raises(E.EulerHipError, match=match):
            h.execute(*args, **kw)
    with pytest.raises(E.EulerHipError, match="null"):
        E.Norm(E.make_norm_desc(64, parts=2)).execute(256, 256, 4)          # no weights of the parts
    with pytest.raises(E.EulerHipError, match="null"):
        E.Norm(E.make_norm_desc(64, output_type=E.S8)).execute(256, 256, 4)   # no place for the scales
    h.execute(None, None, 0)


def test_route_calls_are_checked_before_a_launch():
    h = E.Router(E.make_route_desc(64, 4))
    assert h.plan_ints(0) == 65 and h.plan_ints(10) >= 65 + 40
    for tokens in (-1, 1 << 28, 1 << 62):
        with pytest.raises(ValueError):
            h.plan_ints(tokens)
    for args, kw, match in (((256, 256, 256, None, 4), {}, "null"), ((None, 256, 256, 256, 4), {}, "null"), ((256, 256, 256, 256, -1), {}, "tokens"),
                            ((256, 256, 256, 256, 1 << 28), {}, "tokens"), ((256, 256, 256, 256, 4), {"logits_stride": 5}, "stride"),
                            ((256, 256, 258, 256, 4), {}, "multiple")):
        with pytest.raises(E.EulerHipError, match=match):
            h.execute(*args, **kw)
    h.execute(None, None, None, None, 0)


@pytest.mark.parametrize("base", ["LinearBase", "NormBase", "RouterBase"])
def test_argument_lists(base):
    cls = getattr(E._ehip_call, base)
    h = cls.__new__(cls)   # a handle that is null, as after close()
    n = {"LinearBase": 3, "NormBase": 3, "RouterBase": 5}[base]
    with pytest.raises(E.EulerHipError, match="null argument"):
        h.execute(*[256] * n)
    for args, kw in (([256] * (n - 1), {}), ([256] * n, {"nothing": 1}), ([256] * n, {"stream": 1.0}), ([256] * 40, {})):
        with pytest.raises(TypeError):
            h.execute(*args, **kw)
    if base != "RouterBase":
        with pytest.raises(TypeError):
            h.execute(256, 256, 1.5)
        with pytest.raises(E.EulerHipError, match="null argument"):
            h.execute(256, 256, np.int64(4))
        with pytest.raises(OverflowError):
            h.execute(256, 256, 1 << 70)


@pytest.mark.parametrize("kind", [E.F32, E.F16, E.BF16])
def test_scales_without_codes_are_refused(kind):
    h = E.Norm(E.make_norm_desc(64, data_type=kind))
    for rows in (0, 4):
        with pytest.raises(E.EulerHipError, match="s8 rows"):
            h.execute(256, 256, rows, output_scale=256)


def test_route_counts_tokens_that_a_launch_can_have():
    """8 threads a token, and a launch's are counted in 32 bits"""
    h = E.Router(E.make_route_desc(2, 1))
    assert h.plan_ints((1 << 29) - 128) > 0
    for tokens in ((1 << 29) - 127, (1 << 30) - 1):
        with pytest.raises(ValueError):
            h.plan_ints(tokens)
        with pytest.raises(E.EulerHipError, match="tokens"):
            h.execute(256, 256, 256, 256, tokens)
