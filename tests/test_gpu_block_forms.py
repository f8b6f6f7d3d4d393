"""The gated residual norm on the GPU in every form: each requested gradient is
there, by name, and rows of every width class in calls where a workgroup takes
more than one row."""
import pytest
import torch

from .test_gpu_block_norm import BF16, F16, F32, KINDS, run

pytestmark = pytest.mark.gpu
IDS = dict(ids=lambda k: "-".join(map(str, k)))


def wanted(post, pre, gate):
    names = ["x", "y"] + ["gate"] * (gate is not None)
    for which, kind in (("post", post), ("pre", pre)):
        names += [f"{which}_weight"] * (kind != "none") + [f"{which}_bias"] * (kind == "layer")
    return set(names)


def check(M, D, dt, st, kinds, **kw):
    _, _, _, grads = run(M, D, dt, st, *kinds, **kw)  # holds each gradient that is there to its bound
    names = wanted(*kinds[:3]) if kw.get("wrt") is None else set(kw["wrt"])
    assert set(grads) == names
    assert [n for n, g in grads.items() if g is None] == []
    return grads


@pytest.mark.parametrize("kinds", KINDS, **IDS)
@pytest.mark.parametrize("M,D", [(5, 40), (3, 5), (33, 400), (3, 1537), (2, 4097)])
def test_every_gradient_is_there(M, D, kinds):
    check(M, D, BF16, F32, kinds)


@pytest.mark.parametrize("use", [("r",), ("h",)])
@pytest.mark.parametrize("kinds", KINDS, **IDS)
def test_every_gradient_is_there_with_one_output_used(use, kinds):
    """An input that the used output does not depend on has a gradient of zeros."""
    grads = check(9, 72, F32, F32, kinds, use=use)
    if use == ("r",):
        assert all((grads[n] == 0).all() for n in grads if n.startswith("pre_"))


@pytest.mark.parametrize("gate", ["channel", "row", "full"])
def test_one_gradient_at_a_time(gate):
    kinds = ("layer", "layer", gate, "sigmoid", 0.2)
    for name in wanted(*kinds[:3]):
        check(9, 72, F32, F32, kinds, wrt=(name,))


@pytest.mark.parametrize("dt,st", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("kinds", KINDS, **IDS)
@pytest.mark.parametrize("M,D", [(1100, 300), (530, 2600), (530, 5120), (530, 9001)])
def test_more_rows_than_workgroups(M, D, kinds, dt, st):
    """Past 512 workgroups each takes rows in turn and holds their column sums."""
    check(M, D, dt, st, kinds)


@pytest.mark.parametrize("kinds", [KINDS[1], KINDS[3]], ids=["channel", "full"])
def test_widest_rows(kinds):
    check(515, 16384, F16, F32, kinds)
