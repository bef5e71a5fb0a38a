"""The token operators together, as a model uses them: tokens in through the embedding, blocks between norms, gates and the residual stream,
logits of the tied table, a teacher's top logits out.

fp32 against the same model in fp64 on the CPU.  The longest chain to a gradient of this model has under 4000 roundings (embedding 2; per block
and direction two norms of 40, two products of 40 and 80 terms and 10 more; the logits 40; the loss 800): values within 4000 * 2^-24 =
2.4e-4 of the largest of their kind."""
import pytest
import torch

pytestmark = pytest.mark.gpu
V, D, HID, LAYERS, B, L, K = 97, 40, 80, 2, 3, 21, 8
TOL = 4000 * 2.0 ** -24


def parameters(seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    p = {"table": 0.5 * r(V, D), "first": 1 + 0.1 * r(D)}
    for i in range(LAYERS):
        p.update({f"in{i}": r(D, HID) / D ** 0.5, f"out{i}": r(HID, D) / HID ** 0.5, f"post{i}": 1 + 0.1 * r(D), f"next{i}": 1 + 0.1 * r(D)})
    p["gate0"], p["gate1"] = 0.5 * r(D), 0.5 * r(B, 1, D)                     # one gate a channel, one a sample
    return p, torch.randint(0, V, (B, L), generator=gen), 3 * r(B, L, K), torch.randint(0, V, (B, L, K), generator=gen)


def model(ops, p, ids):
    x = ops.token_embedding(ids, p["table"], scale=D ** 0.5, padding_idx=0)
    h = ops.block_norm(x, p["first"])
    for i in range(LAYERS):
        y = torch.tanh(h @ p[f"in{i}"]) @ p[f"out{i}"]
        x, h = ops.block_join(x, y, post_weight=p[f"post{i}"], gate=p[f"gate{i}"], residual_scale=0.9, next_weight=p[f"next{i}"])
    return h @ p["table"].t()


def step(ops, p, ids, t, tid, weight):
    loss = ops.topk_distill_loss(model(ops, p, ids), t, tid, temperature=2.0, row_weight=weight)
    return [loss.detach(), *torch.autograd.grad(loss, list(p.values()))]


class Plain:
    """The operators' definitions, for fp64 tensors."""

    @staticmethod
    def token_embedding(ids, table, scale, padding_idx):
        rows = table[ids]
        pad = (ids == padding_idx)[..., None]
        return scale * torch.where(pad, rows.detach(), rows)

    @staticmethod
    def block_norm(x, w, eps=1e-6):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w

    @classmethod
    def block_join(cls, x, y, post_weight, gate, residual_scale, next_weight):
        x = residual_scale * x + gate * cls.block_norm(y, post_weight)
        return x, cls.block_norm(x, next_weight)

    @staticmethod
    def topk_distill_loss(z, t, tid, temperature, row_weight):
        p, lq = torch.softmax(t / temperature, -1), torch.log_softmax(z / temperature, -1)
        return (temperature ** 2 * row_weight * (p * (p.log() - lq.gather(-1, tid))).sum(-1)).mean()


def test_training_step(cuda):
    from omnihd_amd import ops
    p, ids, t, tid = parameters(1)
    weight = (torch.rand(B, L, generator=torch.Generator().manual_seed(2)) < 0.8).float()
    ids[0, :3] = 0
    want = step(Plain, {k: v.double().requires_grad_() for k, v in p.items()}, ids, t.double(), tid, weight.double())
    q = {k: v.cuda().requires_grad_() for k, v in p.items()}
    args = (ids.cuda(), t.cuda(), tid.cuda(), weight.cuda())
    got = step(ops, q, *args)
    for name, a, b in zip(["loss", *p], got, want):
        off = (a.double().cpu() - b).abs().max().item()
        assert off <= TOL * b.abs().max().item(), (name, off, b.abs().max().item())
    # captured: replays with other inputs, the program's own eager steps between them
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ops, q, *args)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        held = step(ops, q, *args)
    gen = torch.Generator().manual_seed(3)
    for _ in range(4):
        args[0].copy_(torch.randint(0, V, (B, L), generator=gen))
        with torch.no_grad():
            for v in q.values():
                v.add_(0.01 * torch.randn(v.shape, generator=gen).cuda())
        graph.replay()
        torch.cuda.synchronize()
        now = step(ops, q, *args)
        for name, a, b in zip(["loss", *p], held, now):
            assert (a - b).abs().max().item() <= TOL * b.abs().max().item(), name          # (the library's products need not repeat bit for bit)


def test_single_tokens_give_the_batch_rows(cuda):
    """The serving form: what a token's row is does not depend on the rows beside it, bit for bit (the blocks' products left out)."""
    from omnihd_amd import ops
    p, ids, _, _ = parameters(4)
    q, ids = {k: v.cuda() for k, v in p.items()}, ids.cuda()
    y = torch.randn(B, L, D, generator=torch.Generator().manual_seed(5)).cuda()
    one_gate = q["gate0"]

    def run(ids, y):
        x = ops.token_embedding(ids, q["table"], scale=2.0)
        h = ops.block_norm(x, q["first"])
        return (x, h, *ops.block_join(x, y, post_weight=q["post0"], gate=one_gate, next_weight=q["next0"]))
    whole = run(ids, y)
    for b, l in ((0, 0), (1, 7), (2, L - 1)):
        one = run(ids[b:b + 1, l:l + 1], y[b:b + 1, l:l + 1])
        for a, c in zip(whole, one):
            assert torch.equal(a[b:b + 1, l:l + 1], c)


def test_bf16_model_runs_and_learns_from_the_same_graph_twice(cuda):
    """bf16 activations around an fp32 stream and fp32 parameters; retained graph, two backward passes, gradients add up."""
    from omnihd_amd import ops
    p, ids, t, tid = parameters(6)
    q = {k: v.cuda().requires_grad_() for k, v in p.items()}
    x = ops.token_embedding(ids.cuda(), q["table"], scale=2.0)
    h = ops.block_norm(x, q["first"], out_dtype=torch.bfloat16)
    y = torch.tanh(h @ q["in0"].bfloat16()) @ q["out0"].bfloat16()
    x, h = ops.block_join(x, y, post_weight=q["post0"], gate=q["gate0"], next_weight=q["next0"])
    assert x.dtype == torch.float32 and h.dtype == torch.bfloat16
    loss = ops.topk_distill_loss(h @ q["table"].bfloat16().t(), t.cuda(), tid.cuda(), reduction="mean")
    used = [q[k] for k in ("table", "first", "in0", "out0", "post0", "gate0", "next0")]
    once = torch.autograd.grad(loss, used, retain_graph=True)
    twice = torch.autograd.grad(loss, used)
    for a, b, v in zip(once, twice, used):
        assert a.dtype == v.dtype and bool(a.isfinite().all()) and torch.equal(a, b)


def test_occupancy_head_distils(cuda):
    """BEVOCCHead2Dv2.distill_loss: each voxel's kept classes, unknown voxels left out; values and gradients against fp64."""
    from projects.mmdet3d_plugin.bevfusion.dense_heads.bev_occ_head import BEVOCCHead2Dv2
    gen = torch.Generator().manual_seed(7)
    shape, classes, top = (2, 6, 5, 4), 12, 4
    z = torch.randn(*shape, classes, generator=gen)
    full = 2 * torch.randn(*shape, classes, generator=gen)
    t, tid = full.topk(top, -1)
    known = torch.rand(*shape, generator=gen) < 0.7
    ref = z.double().requires_grad_()
    p, lq = torch.softmax(t.double() / 1.5, -1), torch.log_softmax(ref / 1.5, -1)
    want = 0.5 * (1.5 ** 2 * known * (p * (p.log() - lq.gather(-1, tid))).sum(-1)).sum() / known.sum()
    want.backward()
    zc = z.cuda().requires_grad_()
    got = BEVOCCHead2Dv2.distill_loss(None, zc, t.cuda(), tid.cuda(), known=known.cuda(), temperature=1.5, loss_weight=0.5)["loss_occ_distill"]
    got.backward()
    assert abs(got.item() - want.item()) <= 1000 * 2.0 ** -24 * want.item() * 4
    assert (zc.grad.double().cpu() - ref.grad).abs().max() <= 1000 * 2.0 ** -24 * ref.grad.abs().max()
    none = BEVOCCHead2Dv2.distill_loss(None, zc, t.cuda(), tid.cuda(), known=torch.zeros(shape, device="cuda"))["loss_occ_distill"]
    assert none.item() == 0


def test_two_streams_at_once(cuda):
    """Two training steps on two streams, work of both in flight: each as it is alone (workspaces belong to their call)."""
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(11)
    sets = []
    for k in range(2):
        n, vocab, dim = 3000 + 500 * k, 2000, 264
        table = torch.randn(vocab, dim, generator=gen).cuda().requires_grad_()
        w = torch.rand(dim, generator=gen).cuda().requires_grad_()
        y = torch.randn(n, dim, generator=gen).cuda().requires_grad_()
        sets.append((torch.randint(0, vocab, (n,), generator=gen).cuda(), table, w, y, torch.randn(n, 5, generator=gen).cuda(), torch.randint(0, dim, (n, 5), generator=gen).cuda()))

    def one(ids, table, w, y, t, tid):
        x = ops.token_embedding(ids, table)
        x, h = ops.block_join(x, y, post_weight=w, gate=w, next_weight=w)
        loss = ops.topk_distill_loss(h, t, tid) + x.square().mean()
        return [loss.detach(), *torch.autograd.grad(loss, (table, w, y))]
    alone = [one(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(one(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert all(torch.equal(u, v) for u, v in zip(a[1:], b[1:]))


def test_saved_tensors_elsewhere_and_recomputed(cuda):
    """What the operators keep for the backward may be moved to the host in between, or computed again (checkpointing): the same gradients."""
    from torch.utils.checkpoint import checkpoint

    from omnihd_amd import ops
    p, ids, t, tid = parameters(9)
    q = {k: v.cuda().requires_grad_() for k, v in p.items()}
    args = (ids.cuda(), t.cuda(), tid.cuda(), torch.ones(B, L, device="cuda"))
    want = step(ops, q, *args)
    with torch.autograd.graph.save_on_cpu():
        got = step(ops, q, *args)
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= TOL * b.abs().max()
    loss = ops.topk_distill_loss(checkpoint(lambda i: model(ops, q, i), args[0], use_reentrant=False), args[1], args[2], temperature=2.0, row_weight=args[3])
    for a, b in zip(torch.autograd.grad(loss, list(q.values())), want[1:]):
        assert (a - b).abs().max() <= TOL * b.abs().max()
