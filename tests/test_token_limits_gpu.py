"""The token operators at the ends of what they accept, and beside other machinery of torch than the backward pass."""
import pytest
import torch

from .token_helpers import bound, check_close

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16


def test_forward_mode_and_traces_are_refused(cuda):
    """Through the public entry points; beside them, in the same dual level, calls without a tangent run as ever."""
    import torch.autograd.forward_ad as fw

    from omnihd_amd import ops
    ids = torch.arange(6, device="cuda")
    x, y, w, t = (torch.randn(*s, device="cuda") for s in ((6, 16), (6, 16), (16,), (6, 2)))
    calls = {
        "token_embedding": lambda v: ops.token_embedding(ids, v), "block_norm": lambda v: ops.block_norm(v, w),
        "block_join": lambda v: ops.block_join(x, v, post_weight=w, gate=w, next_weight=w)[1],
        "topk_distill_loss": lambda v: ops.topk_distill_loss(v, t, ids[:, None].expand(6, 2).contiguous()),
    }
    for name, call in calls.items():
        want = call(x)
        with fw.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                    call(fw.make_dual(y, x))
            assert torch.equal(call(x), want)
            with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                call(fw.make_dual(x.clone().requires_grad_(), y))
        with pytest.raises(NotImplementedError, match=f"{name}: cannot be traced"):
            torch.jit.trace(call, (x,))
        assert torch.equal(call(x), want)


def test_embedding_gradient_of_as_many_ids_as_are_accepted(cuda):
    """2^31 - 1 tokens of one column: the last group of eight positions ends where the next would begin beyond 2^31.  Sums of ones, whole
    numbers under 2^24 all along, are exact in fp32 in any order."""
    from omnihd_amd import ops
    n, vocab = 2 ** 31 - 1, 1000
    ids = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(vocab)
    table = torch.zeros(vocab, 1, device="cuda", requires_grad=True)
    out = ops.token_embedding(ids, table, out_dtype=B)
    grad, = torch.autograd.grad(out, table, torch.ones(n, 1, dtype=B, device="cuda"))
    want = torch.full((vocab, 1), float(n // vocab), device="cuda")
    want[:n % vocab] += 1
    assert torch.equal(grad, want)
