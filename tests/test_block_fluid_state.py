"""The (seed, step) state of the fluid layers' dropout masks: where it lives,
that it moves on wherever it came from, and what each rank draws from it."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import paddlebox_amd.fluid as fluid
from paddlebox_amd.fluid import kernels
from paddlebox_amd.ops.dropout import keep_mask
from paddlebox_amd.ps.box_wrapper import BoxWrapper
from paddlebox_amd.utils.flags import set_flags

from .test_block_fluid import _build
from .test_collective_modes import _port
from .test_fluid import S, _files

STATES = ("b0.mask_state", "b1.mask_state", "drop.mask_state")


def _pass(path, device, *, startup, restore=None, save=None, graph=False, k=0, passes=1):
    """Passes of 10 batches on `device`.  startup: the place that startup runs on, None: it does not run.
    Returns the scope's parameters and states on the host, and where the states were."""
    path.mkdir(parents=True, exist_ok=True)
    set_flags({"FLAGS_padbox_train_steps_per_graph": k})
    box = fluid.core.BoxWrapper(8, device=device, new=True)
    try:
        box.cfg.sgd.mf_create_thresholds = 0.0
        box.initialize_gpu_and_load_model(slot_vector=list(range(S)), max_keys=200000,
                                          model_path=str(restore / "sparse") if restore else None)
        scope = fluid.Scope()
        main, start, slots, label, dense, loss = _build()
        main._pipeline_opt = dict(main._pipeline_opt or {}, use_graph=graph)
        exe = fluid.Executor(fluid.CPUPlace() if device == "cpu" else fluid.CUDAPlace(0))
        if startup is not None:
            fluid.Executor(startup).run(start, scope=scope)
        if restore:
            fluid.io.load_persistables(exe, str(restore / "dense"), main, scope=scope)
        ds = fluid.DatasetFactory().create_dataset("PadBoxSlotDataset")
        ds.set_use_var([label] + slots + [dense])
        ds.set_batch_size(64)
        ds.set_filelist(_files(path, 2, 320))
        ds.disable_shuffle()
        fluid.core.BoxPS(ds).read_ins_into_memory()
        boxps = fluid.core.BoxPS(ds)
        replays = 0
        for i in range(passes):
            boxps.begin_pass()
            stats = exe.train_from_dataset(main, ds, scope=scope, fetch_list=[loss], print_period=1000)
            replays += stats.get("graph_replays", 0)
            boxps.end_pass()
            if save and i == 0:
                box.save_base(str(save / "sparse"), str(save / "xbox"), "20240101")
                fluid.io.save_persistables(exe, str(save / "dense"), main, scope=scope)
        assert (replays > 0) == graph
        names = [p.name for p in main.all_parameters()] + list(STATES)
        return ({n: scope.get(n).detach().cpu().numpy().copy() for n in names}, {scope.get(n).device for n in STATES})
    finally:
        set_flags({"FLAGS_padbox_train_steps_per_graph": 0})
        BoxWrapper._instance = None


def test_a_state_that_moves_is_the_scopes():
    """The tensor that a layer reads and counts up is the one that the scope holds and a save writes."""
    main, startup = fluid.Program(), fluid.Program()
    with fluid.program_guard(main, startup), fluid.unique_name.guard():
        x = fluid.layers.data("x", shape=[4], dtype="float32")
        fluid.contrib.layers.counter_dropout(x, 0.5, seed=3, name="d")
    scope = fluid.Scope()
    fluid.Executor(fluid.CPUPlace()).run(startup, scope=scope)
    op = next(o for o in main.global_block().ops if o.type == "counter_dropout")

    class Ctx:
        group = None

    Ctx.scope = scope
    st = kernels._mask_state(Ctx, op, torch.device("meta"))
    assert st.device.type == "meta" and scope.get("d.mask_state") is st
    assert kernels._mask_state(Ctx, op, torch.device("meta")) is st


def _resume(tmp_path, device, **kw):
    ck = tmp_path / "ck"
    want, _ = _pass(tmp_path / "a", device, startup=fluid.CPUPlace() if device == "cpu" else fluid.CUDAPlace(0), passes=2,
                    save=ck)
    got, where = _pass(tmp_path / "b", device, startup=None, restore=ck, **kw)
    assert {d.type for d in where} == {torch.device(device).type}
    for n in want:
        if n in STATES:
            assert got[n][1] == 20 and (got[n] == want[n]).all(), n
        else:
            # the bounds of test_block_fluid.py: the CPU's sums alone, the GPU's atomics and codes at a rounding border
            np.testing.assert_allclose(got[n], want[n], rtol=1e-5 if device == "cpu" else 0,
                                       atol=1e-6 if device == "cpu" else 1e-4, err_msg=n)


def test_resume_without_startup(tmp_path):
    _resume(tmp_path, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(graph=True, k=1), dict(graph=True, k=4)], ids=["eager", "captured", "captured4"])
def test_resume_without_startup_gpu(tmp_path, kw):
    """A checkpoint loaded into an empty scope: its states are host tensors until the first step."""
    _resume(tmp_path, "cuda:0", **kw)


@pytest.mark.gpu
def test_startup_on_the_host_gpu(tmp_path):
    """Startup by a host executor, training on the GPU: the masks of a run that started there."""
    want, _ = _pass(tmp_path / "a", "cuda:0", startup=fluid.CUDAPlace(0))
    got, where = _pass(tmp_path / "b", "cuda:0", startup=fluid.CPUPlace())
    assert {d.type for d in where} == {"cuda"}
    for n in STATES:
        assert got[n][1] == 10 and (got[n] == want[n]).all(), n


def _masks(rank, steps=3, ckpt=None, save=None):
    """What `rank` draws for the same rows: a kept-or-not mask of counter_dropout and of fused_residual_norm a step."""
    main, startup = fluid.Program(), fluid.Program()
    with fluid.program_guard(main, startup), fluid.unique_name.guard():
        x = fluid.layers.data("x", shape=[16], dtype="float32")
        d = fluid.contrib.layers.counter_dropout(x, 0.5, seed=5, name="d")
        r, _ = fluid.contrib.layers.fused_residual_norm(x, x, x_scale=0.0, dropout_prob=0.25, seed=7, pre_norm="none", name="r")
        loss = fluid.layers.reduce_mean(fluid.layers.fc(d, 1, name="f"))
        fluid.optimizer.SGD(learning_rate=0.0).minimize(loss)
    scope, exe = fluid.Scope(), fluid.Executor(fluid.CPUPlace())
    exe.run(startup, scope=scope)
    if ckpt:
        fluid.io.load_persistables(exe, ckpt, main, scope=scope)
    out = []
    for _ in range(steps):
        out += [v != 0 for v in exe.run(main, feed={"x": np.ones((9, 16), np.float32)}, fetch_list=[d, r], scope=scope)]
    if save and rank == 0:
        fluid.io.save_persistables(exe, save, main, scope=scope)
    return out, [scope.get(n).tolist() for n in ("d.mask_state", "r.mask_state")]


def _rank_worker(rank, port, path, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        first = _masks(rank, save=path)
        dist.barrier()
        q.put((rank, first, _masks(rank, steps=2, ckpt=path)))
    finally:
        dist.barrier()
        dist.destroy_process_group()


def _defined(rank, step):
    at = step + (rank << 32)
    return [keep_mask((9, 16), thr, None, seed, at, torch.device("cpu")).numpy() for thr, seed in ((32768, 5), (16384, 7))]


def test_each_rank_draws_its_own_masks(tmp_path):
    """Two data-parallel ranks on the same rows: masks of (seed, step, rank), one state that a checkpoint of rank 0 gives
    to both, and a resumed run that goes on with each rank's masks."""
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _port()
    ps = [ctx.Process(target=_rank_worker, args=(r, port, str(tmp_path / "ck"), q)) for r in range(2)]
    for p in ps:
        p.start()
    got = {r: v for r, *v in (q.get(timeout=120) for _ in ps)}
    for p in ps:
        p.join(timeout=60)
    for rank, ((first, state), (then, after)) in got.items():
        assert state == [[5, 3], [7, 3]] and after == [[5, 5], [7, 5]]  # the same on every rank
        want = [m for step in range(5) for m in _defined(rank, step)]
        for a, b in zip(first + then, want):
            np.testing.assert_array_equal(a, b)
    assert all((a != b).any() for a, b in zip(got[0][0][0], got[1][0][0]))


def test_one_process_draws_the_masks_of_rank_0():
    out, state = _masks(0)
    assert state == [[5, 3], [7, 3]]
    for a, b in zip(out, [m for step in range(3) for m in _defined(0, step)]):
        np.testing.assert_array_equal(a, b)


@pytest.mark.gpu
def test_a_later_rank_captured_gpu(tmp_path, monkeypatch):
    """Rank 1's masks in captured steps are those of its eager steps, and not rank 0's."""
    zero, _ = _pass(tmp_path / "z", "cuda:0", startup=fluid.CUDAPlace(0))
    monkeypatch.setattr(kernels, "_mask_rank", lambda ctx: 1)
    eager, _ = _pass(tmp_path / "e", "cuda:0", startup=fluid.CUDAPlace(0))
    graphed, _ = _pass(tmp_path / "g", "cuda:0", startup=fluid.CUDAPlace(0), graph=True, k=4)
    for n in eager:
        if n in STATES:
            assert (graphed[n] == eager[n]).all() and (zero[n] == eager[n]).all() and eager[n][1] == 10, n
        else:
            np.testing.assert_allclose(graphed[n], eager[n], rtol=0, atol=1e-4, err_msg=n)  # as in test_block_fluid.py
    assert np.abs(zero["w1"] - eager["w1"]).max() > 1e-3  # other masks train another model


def test_layer_seeds():
    """Any whole number is a seed, as for ops.dropout (64 bits of it count); what is not one is refused when the layer is built."""
    def build(seed):
        main, startup = fluid.Program(), fluid.Program()
        with fluid.program_guard(main, startup), fluid.unique_name.guard():
            x = fluid.layers.data("x", shape=[4], dtype="float32")
            fluid.contrib.layers.counter_dropout(x, 0.5, seed=seed, name="d")
            fluid.contrib.layers.fused_residual_norm(x, x, dropout_prob=0.5, seed=seed, name="r")
        scope = fluid.Scope()
        fluid.Executor(fluid.CPUPlace()).run(startup, scope=scope)
        return [scope.get(n).tolist() for n in ("d.mask_state", "r.mask_state")]

    for seed, held in ((0, 0), (-5, -5), (np.int64(7), 7), ((1 << 62) + 12345, (1 << 62) + 12345), (1 << 63, -(1 << 63)),
                       ((1 << 64) + 3, 3)):
        assert build(seed) == [[held, 0]] * 2
    for seed in (1.5, "7", True):
        with pytest.raises(TypeError, match="whole number"):
            build(seed)
