"""What the torch face of the token operators (csrc/torch_tokens.cpp) refuses by itself, on CPU tensors: every refusal comes before a device is asked
for."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fw

ROWS, DIM, TOP = 5, 8, 3


def face():
    from omnihd_amd._lib import torch_ops
    return torch_ops()


def tensors():
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen)
    return dict(table=r(6, DIM), x=r(ROWS, DIM), y=r(ROWS, DIM), post=r(DIM), gate=r(DIM), next=r(DIM), z=r(ROWS, DIM), t=r(ROWS, TOP), w=torch.ones(ROWS), avg=torch.ones(()))


CALLS = {
    "token_embedding": (("table",), lambda f, m: f.token_embedding(torch.zeros(ROWS, dtype=torch.int64), m["table"], 1.0, -1, torch.float32)),
    "block_norm": (("x", "next"), lambda f, m: f.block_join(m["x"], None, None, None, m["next"], 1.0, 1e-6, 0, 1, torch.float32)),
    "block_join": (("x", "y", "post", "gate", "next"), lambda f, m: f.block_join(m["x"], m["y"], m["post"], m["gate"], m["next"], 1.0, 1e-6, 1, ROWS, torch.float32)),
    "topk_distill_loss": (("z", "t", "w", "avg"), lambda f, m: f.topk_distill(m["z"], m["t"], torch.zeros(ROWS, TOP, dtype=torch.int64), m["w"], m["avg"], 1.0, 1.0, False)),
}
NAMED = [(call, name) for call, (names, _) in CALLS.items() for name in names]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("wants", [True, False])
@pytest.mark.parametrize("call,name", NAMED)
def test_dual_tensors_are_refused(call, name, wants, grad):
    """A tangent that the kernel does not carry on would make the directional derivative zero without a word."""
    with fw.dual_level(), contextlib.nullcontext() if grad else torch.no_grad():
        m = tensors()
        m[name] = fw.make_dual(m[name].requires_grad_(wants), torch.ones_like(m[name]))
        with pytest.raises(NotImplementedError, match=f"{call}: forward-mode"):
            CALLS[call][1](face(), m)


@pytest.mark.filterwarnings("ignore")                     # (torch's own, about the trace)
@pytest.mark.parametrize("call,name", NAMED)
def test_traces_are_refused(call, name):
    """A trace would hold the output's allocation alone."""
    from torch.fx.experimental.proxy_tensor import make_fx
    m = tensors()
    body = lambda v: CALLS[call][1](face(), {**m, name: v})
    with pytest.raises(NotImplementedError, match=f"{call}: cannot be traced"):
        torch.jit.trace(body, (m[name],))
    with pytest.raises(NotImplementedError, match=f"{call}: cannot be traced"):
        make_fx(body)(m[name])


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the wrappers' argument checks run on it."""
    is_cuda = True


def test_numbers_that_want_a_gradient_are_refused(monkeypatch):
    """They would be taken for constants; under no_grad, and as numbers or plain tensors, they are what they were."""
    from omnihd_amd import ops
    from omnihd_amd.ops import misc, norm
    seen = []

    class Face:
        def __getattr__(self, name):
            return lambda *args: (seen.append([a for a in args if type(a) is float]), [None, None])[1]
    monkeypatch.setattr(misc, "torch_ops", Face)
    monkeypatch.setattr(norm, "torch_ops", Face)
    m = {k: v.as_subclass(OnDevice) for k, v in tensors().items()}
    ids = torch.zeros(ROWS, TOP, dtype=torch.int64).as_subclass(OnDevice)
    calls = {
        "scale": lambda v: ops.token_embedding(ids, m["table"], scale=v), "eps": lambda v: ops.block_norm(m["x"], m["next"], eps=v),
        "residual_scale": lambda v: ops.block_join(m["x"], m["y"], residual_scale=v), "temperature": lambda v: ops.topk_distill_loss(m["z"], m["t"], ids, temperature=v),
        "loss_weight": lambda v: ops.topk_distill_loss(m["z"], m["t"], ids, loss_weight=v, reduction="sum"),
    }
    for name, call in calls.items():
        learnt = torch.tensor(0.5, requires_grad=True)
        with pytest.raises(TypeError, match=f"{name} is a constant"):
            call(learnt)
        with fw.dual_level(), pytest.raises(TypeError, match=f"{name} is a constant"):
            call(fw.make_dual(torch.tensor(0.5), torch.tensor(1.0)))
        assert not seen
        with torch.no_grad():
            call(learnt)
        for value in (0.5, torch.tensor(0.5), torch.tensor([0.5])):
            call(value)
        assert len(seen) == 4 and all(0.5 in floats for floats in seen)
        seen.clear()
