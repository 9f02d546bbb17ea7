"""Clipping of the gradients by their norm in a training step: on the host executor, and on the GPU where there is one."""
import copy
import math
from types import SimpleNamespace

import pytest
import torch

from flexflow_train_b200 import _ffcore as core
from flexflow_train_b200 import api
from flexflow_train_b200.frontend import AdamOptimizer, SGDOptimizer
from flexflow_train_b200.frontend.keras import optimizers as keras_optimizers
from flexflow_train_b200.runtime.executor import ExecConfig, Executable, OptimizerConfig

MLP = {"batch_size": 16, "input_dim": 24}
gpu = pytest.mark.gpu


def batch(classes, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return {"input": torch.randn(16, 24, generator=g) * scale}, torch.randint(0, classes, (16,), generator=g, dtype=torch.int32)


def classes_of(model):
    return int(model.graph.shape(model.executable.loss_value).sizes[-1])


@pytest.mark.parametrize("kind", ["sgd", "adam"])
def test_host_step_is_the_step_of_scaled_gradients(kind):
    make = lambda c: api.compile("mlp", MLP, optimizer=OptimizerConfig(kind=kind, lr=0.1, max_grad_norm=c), device="cpu")  # noqa: E731
    plain = make(0.0)
    x, y = batch(classes_of(plain))
    start = plain.state_dict()
    plain.train_step(x, y)
    grads = {k: v.clone() for k, v in plain.executable.named_gradients()}
    norm = math.sqrt(sum((v.double() ** 2).sum().item() for v in grads.values()))
    for limit in (norm * 0.25, norm * 4):
        m = make(limit)
        m.load_state_dict(start)
        m.train_step(x, y)
        assert abs(m.executable.grad_norm.item() - norm) <= 1e-6 * norm
        scale = min(1.0, limit / norm)
        for k, p in m.executable.named_parameters():
            w, g = start["params"][k], grads[k] * scale
            if kind == "adam":
                g = g / (g.abs() + 1e-8 / math.sqrt(1 - 0.999))          # first step: m / sqrt(v) with both corrected
            assert torch.allclose(p, w - 0.1 * g, rtol=1e-5, atol=1e-6), k


def test_frontends_pass_the_limit_on():
    assert SGDOptimizer(None, 0.1, max_grad_norm=2.0).config.max_grad_norm == 2.0
    assert AdamOptimizer(None, max_grad_norm=0.5).config.max_grad_norm == 0.5
    assert keras_optimizers.SGD(0.1, global_clipnorm=3.0).config.max_grad_norm == 3.0
    assert keras_optimizers.Adam().config.max_grad_norm == 0.0


@pytest.mark.parametrize("limit", [-1.0, float("inf"), float("nan")])
def test_limits_that_are_refused(limit):
    with pytest.raises(ValueError):
        api.compile("mlp", MLP, optimizer=OptimizerConfig(kind="sgd", max_grad_norm=limit), device="cpu")


def test_several_ranks_are_refused():
    from flexflow_train_b200.parallel.dist_executor import DistExecutable
    with pytest.raises(NotImplementedError, match="one device"):
        DistExecutable(core.build_model("mlp", MLP), ExecConfig(optimizer=OptimizerConfig(max_grad_norm=1.0)), SimpleNamespace(world_size=2))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["sgd", "adam"])
def test_step_on_the_gpu(dtype, kind):
    """The clipped step is the step of the gradients it left in the arena, scaled; captured or not."""
    def make(limit, graph=False):
        return api.compile("mlp", MLP, config=api.FFConfig(compute_dtype=dtype, use_cuda_graph=graph),
                           optimizer=OptimizerConfig(kind=kind, lr=0.5, epsilon=0.1, max_grad_norm=limit))

    plain = make(0.0)
    x, y = batch(classes_of(plain))
    state = copy.deepcopy(plain.state_dict())          # the dict holds the live tensors
    plain.train_step(x, y)
    norm = math.sqrt((plain.executable.grads.double() ** 2).sum().item())
    for limit in (norm / 3, norm * 3):
        m = make(limit)
        m.load_state_dict(state)
        before = m.executable.master.double().clone()
        m.train_step(x, y)
        ex = m.executable
        assert torch.equal(ex.grads, plain.executable.grads)             # left as they are: the optimizer scales them
        assert abs(ex.grad_norm.item() - norm) <= 3e-7 * norm
        g = ex.grads.double() * min(1.0, limit / norm)
        if kind == "adam":
            first, second = 0.1 * g, 0.001 * g * g
            g = math.sqrt(1 - 0.999) / (1 - 0.9) * first / (second.sqrt() + 0.1)
        want = before - 0.5 * g
        # the step in 32 bits: a few 2^-24 of the weight and some 1e-6 of the step (the approximate square root and quotient)
        assert ((ex.master.double() - want).abs() <= 2.0 ** -22 * before.abs() + 4e-6 * (0.5 * g).abs() + 1e-9).all()
    eager, replayed = make(norm / 3), make(norm / 3, graph=True)
    replayed.load_state_dict(eager.state_dict())
    for step in range(4):
        x, y = batch(classes_of(plain), seed=step)
        assert eager.train_step(x, y) == replayed.train_step(x, y)
        assert torch.equal(eager.executable.grad_norm, replayed.executable.grad_norm)
    assert torch.equal(eager.executable.master, replayed.executable.master)


@gpu
def test_a_limit_changed_after_the_build():
    """Taken away, the step does not clip; brought in, it is refused."""
    make = lambda limit: api.compile("mlp", MLP, config=api.FFConfig(compute_dtype="fp32", use_cuda_graph=False),  # noqa: E731
                                     optimizer=OptimizerConfig(kind="sgd", lr=0.5, max_grad_norm=limit))
    plain, other = make(0.0), make(1e-3)
    other.load_state_dict(copy.deepcopy(plain.state_dict()))
    x, y = batch(classes_of(plain))
    other.executable.cfg.optimizer.max_grad_norm = 0.0
    plain.train_step(x, y)
    other.train_step(x, y)
    assert torch.equal(plain.executable.master, other.executable.master)
    plain.executable.cfg.optimizer.max_grad_norm = 1.0
    with pytest.raises(ValueError, match="max_grad_norm"):
        plain.train_step(x, y)


@gpu
def test_tables_are_part_of_the_norm():
    """Plain SGD keeps embedding tables out of the arena; with clipping they are in it."""
    cfg = {"batch_size": 64, "embedding_dim": 16, "embedding_bag_size": 1, "embedding_size": [500, 300],
           "dense_arch_layer_sizes": [13, 32, 16], "over_arch_layer_sizes": [48, 32, 1], "arch_interaction_op": "DOT",
           "final_activation": "SIGMOID", "embedding_data_type": "FLOAT"}
    g = core.build_model("dlrm", cfg)
    limit = Executable(g, ExecConfig(loss="mean_squared_error_avg_reduce", optimizer=OptimizerConfig(kind="sgd", lr=0.1, max_grad_norm=1.0)))
    plain = Executable(g, ExecConfig(loss="mean_squared_error_avg_reduce", optimizer=OptimizerConfig(kind="sgd", lr=0.1)))
    assert plain.sparse_weight_nodes() and not limit.sparse_weight_nodes()
    assert limit.num_params > plain.num_params
