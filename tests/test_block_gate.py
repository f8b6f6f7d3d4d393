"""residual_norm without a gate: gate=None beside a gate_act is a block whose
optional gate is absent; a gate_act with the gate left out is refused."""
import numpy as np
import pytest
import torch

import paddlebox_amd.fluid as fluid
from paddlebox_amd.ops.residual import residual_norm


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("post,p", [("none", 0.0), ("rms", 0.25)])
def test_an_absent_gate_has_nothing_to_activate(device, post, p):
    g = torch.Generator().manual_seed(0)
    x, y, go = (torch.randn(7, 40, generator=g).to(device) for _ in range(3))
    w = (torch.rand(40, generator=g) + 0.5).to(device)
    got = []
    for act in ("none", "sigmoid"):
        a, b, v = (t.clone().requires_grad_() for t in (x, y, w))
        r, h = residual_norm(a, b, y_scale=0.5, gate=None, gate_act=act, post=post, post_weight=v if post != "none" else None,
                             pre="rms", pre_weight=v, p=p, seed=3)
        got.append((r, h) + torch.autograd.grad((r, h), (a, b, v), (go, go)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_an_activation_with_the_gate_left_out_is_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="without a gate"):
        residual_norm(x, x, pre="rms", pre_weight=w, gate_act="sigmoid")
    with pytest.raises(ValueError, match="gate_act"):
        residual_norm(x, x, pre="rms", pre_weight=w, gate=None, gate_act="tanh")
    main, startup = fluid.Program(), fluid.Program()
    with fluid.program_guard(main, startup), fluid.unique_name.guard():
        v = fluid.layers.data("x", shape=[8], dtype="float32")
        r, _ = fluid.contrib.layers.fused_residual_norm(v, v, gate_act="sigmoid", name="r")
    scope, exe = fluid.Scope(), fluid.Executor(fluid.CPUPlace())
    exe.run(startup, scope=scope)
    with pytest.raises(ValueError, match="without a gate"):
        exe.run(main, feed={"x": np.zeros((3, 8), np.float32)}, fetch_list=[r], scope=scope)
