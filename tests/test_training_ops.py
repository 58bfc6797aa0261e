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


def test_public_calls_start_over_on_their_inputs_gpu(monkeypatch):
    """Where another GPU is the current one, the input's is made current around the whole call: for a stand-in of a tensor of
    GPU 1, the launch comes with that one current, and the other is current again afterwards."""
    from compactlogic_b200 import training as T
    log = []

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            log.append(("enter", self.index))
            self.before, state.current = state.current, self.index

        def __exit__(self, *error):
            state.current = self.before

    class Far(torch.Tensor):  # on the CPU, says that it is on GPU 1
        is_cuda = True
        device = torch.device("cuda", 1)

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            with torch._C.DisableTorchFunctionSubclass():
                out = func(*args, **(kwargs or {}))
            return out.as_subclass(Far) if isinstance(out, torch.Tensor) else out

        def get_device(self):
            return 1

    class state:
        current = 0

    class Launched(Exception):
        pass

    def launch(*args):
        log.append(("launch", state.current))
        raise Launched

    monkeypatch.setattr(T, "_device", lambda: state.current)
    monkeypatch.setattr(T.torch.cuda, "device", On)
    for name in ("_drop", "_norm_forward", "_logp_forward", "_policy"):
        monkeypatch.setattr(T, name, launch)
    x, one = torch.zeros(4, 8).as_subclass(Far), torch.zeros(4).as_subclass(Far)
    act = torch.zeros(4, dtype=torch.int64).as_subclass(Far)
    m = cl.LogicDropout(0.5)
    m.rng_state = m.rng_state.as_subclass(Far)
    monkeypatch.setattr(m, "_draw", lambda t: log.append(("draw", state.current)))
    for call in (lambda: cl.dropout(x, 0.5, seed=1), lambda: cl.layer_norm(x), lambda: cl.action_log_probs(x, act),
                 lambda: cl.policy_loss(x, act, one, one), lambda: m(x)):
        for current in (0, 1):
            state.current = current
            log.clear()
            with pytest.raises(Launched):
                call()
            assert log[-1] == ("launch", 1) and state.current == current
            assert [e for e in log if e[0] == "enter"] == ([] if current else [("enter", 1)])
            assert all(at == 1 for what, at in log if what == "draw")
