"""The token operators at the ends of what they accept, and beside other machinery of torch than the backward pass."""
import pytest
import torch

from . import test_block_norm_gpu as norm
from . import test_topk_distill_gpu as distill
from .token_helpers import bound, check_close

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.filterwarnings("ignore")                     # (torch's own, about the trace)
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


MANY = [
    # samples of few rows: more gate rows than blocks on the card, fewer rows than a block has places for, one block sum or several a gate row
    ((1500, 2, 16), F, F, F, True, True), ((700, 3, 333), B, F, F, True, True), ((300, 5, 2048), B, B, B, True, True), ((260, 2, 4100), F, F, F, True, True),
    ((2000, 2, 8), H, H, H, False, True), ((1100, 3, 72), B, B, F, True, False), ((300, 70, 64), F, F, F, True, True), ((900, 40, 40), B, F, H, False, False),
    ((30, 40, 2, 24), F, F, F, True, True), ((300, 2, 9001), B, B, F, True, True), ((900, 2, 1), F, F, F, True, True),
]


@pytest.mark.parametrize("shape,act,stream,weights,post,nxt", MANY)
def test_many_gate_rows(cuda, shape, act, stream, weights, post, nxt):
    from omnihd_amd import ops
    x, y, pw, _, nw, gx, gh = norm.inputs(shape, act, stream, weights, "none", post, nxt, sum(shape))
    gen = torch.Generator().manual_seed(sum(shape) + 1)
    gate = (0.7 * torch.randn(*shape[:-2], 1, shape[-1], generator=gen)).to(weights).cuda().requires_grad_()
    assert ops._gate_layout(gate, shape) == (ops._GATE_ROWS, shape[-2])
    got = norm.run_join(ops, x, y, pw, gate, 0.75, nw, gx, gh)
    want, terms = norm.reference(x, y, pw, gate, 0.75, nw, gx, gh)
    norm.compare(got, want, terms, norm.rows_of(shape))
    again = norm.run_join(ops, x, y, pw, gate, 0.75, nw, gx, gh)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("samples,rows,dim", [(16384, 4, 4096), (2 ** 24 + 5, 2, 8)])
def test_more_gate_rows_than_one_launch_takes(cuda, samples, rows, dim):
    """A block for each gate row and 16 columns, or for each gate row alone, would be 2^32 threads and more.  Only the first and last samples have
    an upstream gradient, so the weights' gradients are theirs, and the samples' own are compared there."""
    from omnihd_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=B)
    x, y, gate = r(samples, rows, dim).requires_grad_(), r(samples, rows, dim).requires_grad_(), r(samples, 1, dim).requires_grad_()
    pw, nw = (torch.rand(dim, generator=gen, device="cuda").add_(0.5).requires_grad_() for _ in range(2))
    assert ops._gate_layout(gate, x.shape) == (ops._GATE_ROWS, rows)
    ends = torch.cat([torch.arange(30), torch.arange(samples - 30, samples)]).cuda()
    gx, gh = torch.zeros_like(x), torch.zeros_like(x)
    for g in (gx, gh):
        g[ends] = r(60, rows, dim)
    got = norm.run_join(ops, x, y, pw, gate, 0.75, nw, gx, gh)
    pick = lambda t: t.detach()[ends]
    want, terms = norm.reference(pick(x), pick(y), pw, pick(gate), 0.75, nw, pick(gx), pick(gh))
    for k in ("g_x", "g_y", "g_gate"):
        assert not got[k][samples // 2].any()
    norm.compare({k: v.detach() if k in ("g_post", "g_next") else pick(v) for k, v in got.items()}, want, terms, 60 * rows)


@pytest.mark.parametrize("vocab", [9, 12, 50, 300, 1500, 9001, 40000, 70003, 120001])
def test_distillation_of_values_far_from_zero(cuda, vocab):
    """Only differences count, however far from 0 the values lie: whole rows under a mask of -1e10 or of the type's lowest value, half rows, a
    temperature of 1e-6; the teacher's slots likewise.  (A row of equal values has q = 1 / V exactly, up to the quotient's rounding.)"""
    from omnihd_amd import ops
    low = torch.finfo(F).min
    z, t, ids, gen = distill.inputs(9, vocab, 5, F, F, vocab)
    z[0], z[1], z[2, ::2], z[3, 1::2] = -1e10, low, -1e10, low
    ids[3] -= ids[3] % 2                                   # (what the lowest value masks is not wanted: 3e38 times log2(e) is infinite)
    z[4] = -1e10 + 1024 * torch.randint(0, 3, (vocab,), generator=gen).cuda()          # (1024: a step of fp32 there)
    z[5] = 3e9 + 256 * torch.randint(-1, 2, (vocab,), generator=gen).cuda()
    t[0], t[1], t[2, 1:], t[3], t[4, ::2] = -1e10, low, low, 5e9, -1e10
    z[6], t[6] = low, low
    for reduction in ("sum", "none"):
        loss, grad = distill.check(ops, z, t, ids, 1.0, reduction=reduction)
        assert bool(loss.isfinite().all() and grad.isfinite().all())
    for far in (torch.full_like(z, 5000.0), 5000 + 2.0 ** -10 * torch.randint(0, 2, z.shape, generator=gen).cuda()):
        loss, grad = distill.check(ops, far.float(), 3000 + 0 * t, ids, 1e-6, reduction="none")
        assert bool(loss.isfinite().all() and grad.isfinite().all())
    half = z.clamp(-6e4, 6e4).half()                       # a lowest value among 16-bit logits
    half[1], half[3, 1::2] = torch.finfo(H).min, torch.finfo(H).min
    wide = z.bfloat16()
    wide[1], wide[3, 1::2], wide[6] = torch.finfo(B).min, torch.finfo(B).min, torch.finfo(B).min
    for v in (half, wide):
        loss, grad = distill.check(ops, v, t, ids, 2.0, reduction="none")
        assert bool(loss.isfinite().all() and grad.isfinite().all())


def test_distillation_holds_no_gradient_that_hooks_or_capture_do_not_see(cuda):
    """Device memory of a summed loss between forward and backward: one gradient beside the logits in a plain step, none where saved tensors go
    elsewhere or are computed again, none once its backward is captured; values and gradients are the same bits everywhere."""
    from torch.utils.checkpoint import checkpoint

    from omnihd_amd import ops
    rows, vocab = 512, 32000
    size, small = rows * vocab * 4, 4 << 20
    z, t, ids, _ = distill.inputs(rows, vocab, 6, F, F, 1)
    z.requires_grad_()
    call = lambda v: ops.topk_distill_loss(v, t, ids, temperature=2.0)
    want, = torch.autograd.grad(call(z), z)
    value = call(z.detach())

    def held(forward):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = forward()
        between = torch.cuda.memory_allocated() - before
        torch.cuda.reset_peak_memory_stats()
        grad, = torch.autograd.grad(loss, z)
        peak = torch.cuda.max_memory_allocated() - before
        assert torch.equal(loss, value) and torch.equal(grad, want)
        return between, peak

    def moved():
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v):
            return call(z)
    between, peak = held(lambda: call(z))
    assert size <= between < size + small and peak < size + small
    for forward in (lambda: checkpoint(call, z, use_reentrant=False), moved):
        between, peak = held(forward)
        assert between < small and peak < size + small
    with torch.autograd.graph.save_on_cpu():
        loss = call(z)
    grad, = torch.autograd.grad(loss, z)
    assert torch.equal(grad, want)
    del loss, grad
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    up = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = call(z)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grad, = torch.autograd.grad(loss, z, up, retain_graph=True)
    assert torch.cuda.memory_allocated() - before < size + small           # the captured backward's own
    for factor in (1.0, 2.0, 1.0):
        up.fill_(factor)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, factor * want)
        assert torch.equal(torch.autograd.grad(loss, z, up, retain_graph=True)[0], grad)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="asks for the state of a second device's stream")
def test_capture_on_another_device_than_the_current_one(cuda):
    """The forward captured on the logits' device while another one is current: every replay's gradient follows the logits."""
    from omnihd_amd import ops
    other = torch.device("cuda:1")
    z, t, ids = (v.to(other) for v in distill.inputs(20, 900, 6, F, F, 1)[:3])
    z.requires_grad_()

    def step():
        with torch.cuda.device(0):
            return torch.autograd.grad(ops.topk_distill_loss(z, t, ids), z)[0]
    with torch.cuda.device(other):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for _ in range(3):
            with torch.no_grad():
                z.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, step())


@pytest.mark.parametrize("n", [50, 150000])
@pytest.mark.parametrize("padding", [-1, 40, 2 ** 31 - 1, 2 ** 32 + 3, 2 ** 40 + 3, -2 ** 32 + 3, 3])
def test_padding_outside_the_table(cuda, n, padding):
    """At the C entry, which takes 64 bits: only a row of the table is left out."""
    from omnihd_amd._lib import lib
    L, vocab, dim = lib(), 40, 8
    ids = torch.arange(n, device="cuda") % vocab
    g, grad = torch.ones(n, dim, device="cuda"), torch.empty(vocab, dim, device="cuda")
    ws = torch.empty(L.omnihd_token_embed_bwd_workspace_bytes(n, vocab, dim), dtype=torch.uint8, device="cuda")
    assert L.omnihd_token_embed_bwd(ids.data_ptr(), 1, n, g.data_ptr(), 0, dim, vocab, dim, 1.0, padding, grad.data_ptr(), 0, ws.data_ptr(), ws.numel(),
                                    torch.cuda.current_stream().cuda_stream) == 0
    want = torch.bincount(ids, minlength=vocab).float()
    if 0 <= padding < vocab:
        want[padding] = 0
    assert torch.equal(grad, want[:, None].expand(vocab, dim))


@pytest.mark.parametrize("amp", [False, True])
def test_occupancy_head_trains_from_a_teacher(cuda, amp):
    """The built head, from features to its parameters' gradients, with a teacher head's best four classes a voxel: the loss's own gradient against the
    definition, and every parameter gets what the head passes on of it."""
    from omnihd_amd.mm.registry import HEADS, build_from_cfg
    from projects.mmdet3d_plugin.bevfusion.dense_heads import bev_occ_head  # noqa: F401
    cfg = dict(type="BEVOCCHead2Dv2", in_dim=16, out_dim=16, Dz=4, num_classes=12, loss_occ=dict(type="CrossEntropyLoss", ignore_index=255, loss_weight=1.0))
    student, teacher = (build_from_cfg(cfg, HEADS).cuda() for _ in range(2))
    feats = torch.randn(2, 16, 6, 5, device="cuda")
    with torch.no_grad():
        t, tid = teacher([feats]).mul(3).topk(4, -1)
    known = torch.rand(t.shape[:-1], device="cuda") < 0.7
    with torch.autocast("cuda", torch.bfloat16, enabled=amp):
        pred = student([feats])
    assert pred.shape == (2, 5, 6, 4, 12) and pred.dtype == (B if amp else F)
    loss = student.distill_loss(pred, t, tid, known=known, temperature=1.5, loss_weight=0.5)["loss_occ_distill"]
    grad, = torch.autograd.grad(loss, pred, retain_graph=True)
    flat = lambda v: v.reshape(-1, v.shape[-1])
    count = float(known.sum())
    _, _, dz, terms = distill.reference(flat(pred), flat(t), flat(tid), 1.5, known.reshape(-1).float(), 0.5 / count)
    check_close(flat(grad), dz, bound(dz, pred.dtype, terms, distill.ROUNDINGS), "gradient")
    for g in torch.autograd.grad(loss, list(student.parameters())):
        assert bool(g.isfinite().all()) and bool(g.any())


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("vocab", [9, 12, 50, 300, 1500, 9001, 40000, 70003, 140001])
def test_distillation_of_rows_without_a_finite_maximum(cuda, vocab, dtype):
    """Nothing but -inf, an infinity, a NaN: the row is NaN as its softmax is, unless it has no weight; the rows beside it are what they are alone."""
    from omnihd_amd import ops
    z, t, ids, _ = distill.inputs(12, vocab, 4, dtype, F, vocab)
    inf = float("inf")
    weight = torch.ones(12, device="cuda")
    z[1], z[3, vocab // 2], z[5, vocab - 1], z[7], z[8] = -inf, inf, float("nan"), -inf, inf
    t[9, 1], t[10] = inf, -inf
    weight[7], weight[8] = 0, 0
    z.requires_grad_()
    loss = ops.topk_distill_loss(z, t, ids, row_weight=weight, reduction="none")
    grad, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    bad, none, fine = [1, 3, 5, 9], [7, 8, 10], [0, 2, 4, 6, 11]
    named = torch.zeros(vocab, dtype=torch.bool, device="cuda").index_fill_(0, ids[9], True)     # dz = q - sum of p: p is NaN, q is not
    assert bool(loss[bad].isnan().all()) and bool(grad[bad[:3]].isnan().all()) and torch.equal(grad[9].isnan(), named)
    assert not loss[none].any() and not grad[none].any()
    want, terms, dz, dz_terms = distill.reference(z[fine], t[fine], ids[fine], 1.0, None, 1.0)
    check_close(loss[fine], want, bound(want, F, terms, distill.ROUNDINGS), "row losses")
    check_close(grad[fine], dz, bound(dz, dtype, dz_terms, distill.ROUNDINGS) + 2.0 ** -126, "gradient")
