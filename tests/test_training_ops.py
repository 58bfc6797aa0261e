"""Refusals of the training operators that need no GPU: every C entry point returns a status, never a crash."""
import pytest
import torch

import compactlogic_b200 as cl
from compactlogic_b200 import _lib as L


def test_public_names():
    for name in ("LogicDropout", "LogicLayerNorm", "action_log_probs", "policy_loss"):
        assert name in cl.__all__
    assert "dropout" not in cl.__all__ and "layer_norm" not in cl.__all__ and callable(cl.dropout) and callable(cl.layer_norm)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: cl.dropout(x, 0.5, seed=1), lambda: cl.layer_norm(x), lambda: cl.LogicDropout(0.5)(x),
                 lambda: cl.LogicLayerNorm(8)(x), lambda: cl.action_log_probs(x, torch.zeros(4, dtype=torch.int64)),
                 lambda: cl.policy_loss(x, torch.zeros(4, dtype=torch.int64), torch.zeros(4), torch.zeros(4))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("p", [-0.5, 1.5, float("nan")])
def test_dropout_rates_are_checked(p):
    with pytest.raises(ValueError):
        cl.LogicDropout(p)
    with pytest.raises(ValueError):
        cl.dropout(torch.zeros(2, 2), p, seed=0)
    assert L.lib().clb_dropout(0, 16, 4, 4, 4, 0, p, 1, 0, 0, None, 16, 4, None) == L.CLB_ERR_INVALID


def test_dropout_module_state():
    m = cl.LogicDropout(0.5, seed=123)
    assert m.state_dict()["rng_state"].tolist() == [123, 0]
    x = torch.zeros(2, 2)
    assert m.eval()(x) is x and cl.LogicDropout(0.0)(x) is x
    for seed in (-1, 1 << 63):
        with pytest.raises(ValueError):
            cl.LogicDropout(0.5, seed=seed)
    torch.manual_seed(3)
    a = cl.LogicDropout(0.5).rng_state.tolist()
    torch.manual_seed(3)
    assert a == cl.LogicDropout(0.5).rng_state.tolist()


def test_c_entry_points_refuse_without_a_gpu():
    lib = L.lib()
    assert lib.clb_dropout(9, 16, 4, 4, 4, 0, 0.5, 1, 0, 0, None, 16, 4, None) == L.CLB_ERR_DTYPE
    assert lib.clb_dropout(0, None, 4, 4, 4, 0, 0.5, 1, 0, 0, None, 16, 4, None) == L.CLB_ERR_INVALID
    assert lib.clb_dropout(0, 16, 4, -1, 4, 0, 0.5, 1, 0, 0, None, 16, 4, None) == L.CLB_ERR_INVALID
    assert lib.clb_dropout(0, 16, 4, 4, (1 << 32) + 1, 0, 0.5, 1, 0, 0, None, 16, 4, None) == L.CLB_ERR_INVALID
    assert lib.clb_dropout(0, None, 0, 0, 4, 0, 0.5, 1, 0, 0, None, None, 0, None) == L.CLB_OK  # nothing to do
    assert lib.clb_dropout_advance(None, 16, None) == L.CLB_ERR_INVALID
    norm = [0, 16, 8, 4, 8, 0, None, None, 1e-5, 16, 8, None, None, None, 0, None]
    for at, value, status in [(0, 7, L.CLB_ERR_DTYPE), (1, None, L.CLB_ERR_INVALID), (3, -1, L.CLB_ERR_INVALID),
                              (4, 0, L.CLB_ERR_INVALID), (2, 7, L.CLB_ERR_INVALID), (8, -1.0, L.CLB_ERR_INVALID),
                              (8, float("nan"), L.CLB_ERR_INVALID), (3, 0, L.CLB_OK)]:
        a = list(norm)
        a[at] = value
        assert lib.clb_layer_norm_forward(*a) == status, (at, value)
    back = [0, 16, 8, 16, 8, 4, 8, 0, None, 16, 16, 16, 8, None, None, None, 0, None]
    for at, value, status in [(0, 7, L.CLB_ERR_DTYPE), (3, None, L.CLB_ERR_INVALID), (9, None, L.CLB_ERR_INVALID),
                              (12, 7, L.CLB_ERR_INVALID)]:
        a = list(back)
        a[at] = value
        assert lib.clb_layer_norm_backward(*a) == status, (at, value)
    logp = [0, 16, 8, 4, 8, 0, 16, None, 1.0, 16, None, None]
    for at, value, status in [(0, 7, L.CLB_ERR_DTYPE), (1, None, L.CLB_ERR_INVALID), (2, 7, L.CLB_ERR_INVALID),
                              (4, 0, L.CLB_ERR_INVALID), (6, None, L.CLB_ERR_INVALID), (8, 0.0, L.CLB_ERR_INVALID),
                              (9, None, L.CLB_ERR_INVALID), (3, 0, L.CLB_OK)]:
        a = list(logp)
        a[at] = value
        assert lib.clb_action_logp(*a) == status, (at, value)
    grad = [0, 16, 8, 4, 8, 0, 16, None, 1.0, 16, None, None, 16, 0, 1, 16, 8, None]
    for at, value, status in [(9, None, L.CLB_ERR_INVALID), (12, None, L.CLB_ERR_INVALID), (13, 1, L.CLB_ERR_INVALID),
                              (15, None, L.CLB_ERR_INVALID), (16, 7, L.CLB_ERR_INVALID)]:
        a = list(grad)
        a[at] = value
        assert lib.clb_logit_grad(*a) == status, (at, value)


def test_entry_points_run_on_their_inputs_gpu(monkeypatch):
    """Where another GPU is the current one, the input's is made current around the call, and its stream is taken."""
    from compactlogic_b200 import training as T
    calls, entered = [], []

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *error):
            entered.append(None)

    class Lib:
        def clb_probe(self, *args):
            calls.append((args, list(entered)))
            return self.status

    class Input:
        def get_device(self):
            return 1

    fake = Lib()
    fake.status = L.CLB_OK
    monkeypatch.setattr(T, "_stream", lambda index: 100 + index)
    monkeypatch.setattr(T.torch.cuda, "device", On)
    monkeypatch.setattr(T.L, "lib", lambda: fake)
    for current in (0, 1):
        monkeypatch.setattr(T, "_device", lambda: current)
        T._run("clb_probe", Input(), 7, 8)
    assert calls == [((7, 8, 101), [1]), ((7, 8, 101), [1, None])] and entered == [1, None]
    fake.status = L.CLB_ERR_INVALID
    fake.clb_last_error = lambda: b"no"
    with pytest.raises(RuntimeError, match="clb_probe"):
        T._run("clb_probe", Input())
