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
