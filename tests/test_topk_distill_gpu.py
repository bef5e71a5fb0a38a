"""ops.topk_distill_loss (csrc/topk_distill.hip) against its definition in fp64 on the CPU.

Chains: exp2 of a difference d (one rounding of d * c, two of c) is off by a few steps of 2^-24 and by 3 * 2^-24 * |d| relative; a row sum passes
up to 300 additions in a lane and 10 across; the quotient and products add 6.  So q, p are off by at most (320 + 3 * |d|max) * 2^-24 of
themselves, with |d|max <= 130 here (beyond it they vanish in fp32): 800 roundings of T * k * (q + p) for the gradient.  A row's loss is
T^2 * sum p * (ln p - ln q): 800 roundings of p * (|ln p| + |ln q| + 1) (the 1: p's own relative error, and ln of a sum that is off relatively).
The sum over rows adds a rounding a row of a block, in fp32.

exp2 gives 0 for what is under 2^-126, the smallest normal fp32 number: e = exp2(..) is off by up to 2^-126 more, and the gradient
T * k * (e / sum - p) with sum >= 1 by up to T * |k| * 2^-126 more (a loss, of terms p * ln p with p >= 2^-126 lost or not, by K * 2^-126 * 130
* T^2 * |k|: far under its own bound)."""
import math

import pytest
import torch

from .token_helpers import bound, check_close

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16
ROUNDINGS = 800


def reference(z, t, ids, temperature, weight, k):
    """Row losses, gradient (k: what multiplies row r's loss in the result), and the absolute terms of both; rows without mass or weight are 0."""
    z, t, ids = z.detach().double().cpu(), t.detach().double().cpu(), ids.long().cpu()
    N, V = z.shape
    w = torch.ones(N, dtype=torch.float64) if weight is None else weight.double().cpu()
    k = torch.as_tensor(k, dtype=torch.float64).expand(N)
    rows, row_terms = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    dz, dz_terms = torch.zeros(N, V, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    hole = ids < 0
    tt = (t / temperature).masked_fill(hole, -math.inf)
    live = (w != 0) & (tt != -math.inf).any(1)
    if live.any():
        zl, tl, il = z[live] / temperature, tt[live], ids[live].clamp_min(0)
        p = torch.softmax(tl, 1)
        lq = torch.log_softmax(zl, 1)
        lqk = lq.gather(1, il)
        each = torch.where(p > 0, p * (p.clamp_min(1e-300).log() - lqk), torch.zeros_like(p))
        mag = torch.where(p > 0, p * (p.clamp_min(1e-300).log().abs() + lqk.abs() + 1), torch.zeros_like(p))
        rows[live], row_terms[live] = temperature ** 2 * each.sum(1) * w[live], temperature ** 2 * mag.sum(1) * w[live].abs()
        q = lq.exp()
        f = (temperature * w * k)[live][:, None]
        dz[live] = f * q.scatter_add(1, il, -p)
        dz_terms[live] = f.abs() * q.scatter_add(1, il, p)
    return rows * k, row_terms * k.abs(), dz, dz_terms


def inputs(rows, vocab, top, z_t, t_t, seed, scale=2.0, ids_t=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    z = (scale * torch.randn(rows, vocab, generator=gen)).to(z_t).cuda()
    t = (scale * torch.randn(rows, top, generator=gen)).to(t_t).cuda()
    ids = torch.randint(0, vocab, (rows, top), generator=gen).to(ids_t).cuda()           # (the same id twice in a row now and then)
    return z, t, ids, gen


def check(ops, z, t, ids, temperature=1.0, weight=None, reduction="mean", avg=None, loss_weight=1.0, up=None):
    z = z.detach().requires_grad_()
    N = z.shape[0]
    loss = ops.topk_distill_loss(z, t, ids, temperature=temperature, row_weight=weight, reduction=reduction, avg_factor=avg, loss_weight=loss_weight)
    k = loss_weight
    if reduction == "mean":
        k = loss_weight / (max(N, 1) if avg is None else float(avg))
    rows, row_terms, _, _ = reference(z, t, ids, temperature, weight, k)
    assert loss.dtype == F
    if reduction == "none":
        check_close(loss, rows, bound(rows, F, row_terms, ROUNDINGS), "row losses")
        up = torch.ones(N, device="cuda") if up is None else up
    else:
        check_close(loss, rows.sum(), bound(rows.sum(), F, row_terms.sum(), ROUNDINGS + N), "loss")
    grad, = torch.autograd.grad(loss, z, up, retain_graph=True)
    _, _, dz, dz_terms = reference(z, t, ids, temperature, weight, k if up is None else k * up.double().cpu())
    flushed = temperature * 2.0 ** -126 * float(torch.as_tensor(k, dtype=torch.float64).abs().max()) * (1 if weight is None else float(weight.abs().max()))
    check_close(grad, dz, bound(dz, z.dtype, dz_terms, ROUNDINGS) + flushed * (1 if up is None else float(up.abs().max())), "gradient")
    with torch.no_grad():
        assert torch.equal(ops.topk_distill_loss(z, t, ids, temperature=temperature, row_weight=weight, reduction=reduction, avg_factor=avg,
                                                 loss_weight=loss_weight), loss)
    again, = torch.autograd.grad(loss, z, up)
    assert torch.equal(grad, again)
    return loss, grad


CASES = [
    # rows, vocab, top, logits, teacher, temperature: every geometry of the kernels, its largest and its next size
    (1, 1, 1, F, F, 1.0), (3, 2, 5, B, F, 2.0), (1000, 12, 4, F, F, 1.0), (513, 16, 9, H, H, 0.5), (300, 17, 3, B, B, 1.0), (257, 32, 40, F, F, 3.0),
    (70, 33, 7, F, F, 1.0), (70, 33, 7, B, F, 1.0), (33, 64, 8, H, F, 2.0), (40, 65, 200, B, F, 1.0), (50, 128, 3, F, F, 1.0), (17, 250, 64, B, B, 1.5),
    (9, 256, 65, F, F, 1.0), (9, 257, 256, F, H, 1.0), (20, 512, 16, H, H, 1.0), (20, 513, 16, B, F, 1.0), (6, 1024, 16, F, F, 4.0), (6, 2048, 33, B, F, 1.0),
    (6, 2049, 33, B, F, 1.0), (5, 4096, 100, F, F, 1.0), (5, 8192, 20, B, B, 1.0), (5, 8193, 20, H, F, 0.7), (4, 16384, 256, B, F, 1.0), (4, 16387, 5, F, F, 1.0),
    (3, 32000, 20, B, F, 2.0), (3, 32771, 20, B, F, 2.0), (3, 65536, 50, H, F, 1.0), (3, 65537, 50, B, F, 1.0), (2, 33001, 50, F, F, 1.0), (2, 150001, 64, B, F, 1.0),
    (2, 262144, 10, F, F, 1.0),
]


@pytest.mark.parametrize("rows,vocab,top,z_t,t_t,temperature", CASES)
def test_loss_and_gradient(cuda, rows, vocab, top, z_t, t_t, temperature):
    from omnihd_amd import ops
    z, t, ids, gen = inputs(rows, vocab, top, z_t, t_t, vocab + top, ids_t=torch.int64 if vocab % 2 else torch.int32)
    check(ops, z, t, ids, temperature)
    up = torch.rand(rows, generator=gen).cuda()
    check(ops, z, t, ids, temperature, reduction="none", up=up, loss_weight=0.3)


@pytest.mark.parametrize("rows,vocab,top", [(200, 12, 6), (60, 100, 20), (40, 3001, 30), (20, 20000, 8), (6, 70001, 100)])
def test_holes_masks_and_rows_without_mass(cuda, rows, vocab, top):
    from omnihd_amd import ops
    z, t, ids, gen = inputs(rows, vocab, top, F, F, vocab)
    ids[torch.rand(rows, top, generator=gen).cuda() < 0.3] = -1
    ids[1], ids[3, 1:] = -1, -5                            # no slot; the first slot alone
    t[ids < 0] = float("nan")                              # empty slots may hold anything
    t[4, :] = -math.inf                                    # slots without mass
    t[5, 0] = -math.inf
    weight = (torch.rand(rows, generator=gen) < 0.6).float().cuda() * 1.7
    weight[2], weight[0], weight[3:6] = 0, 2.5, 1
    z[1], z[2], z[4, 0] = float("nan"), float("inf"), float("nan")        # rows that add nothing, whatever they hold
    for reduction in ("mean", "sum", "none"):
        loss, grad = check(ops, z, t, ids, 1.3, weight=weight, reduction=reduction)
        assert bool(loss.isfinite().all()) and not grad[[1, 2, 4]].any()


@pytest.mark.parametrize("rows,vocab,top", [(100, 12, 4), (40, 100, 4), (40, 3001, 4), (10, 20000, 4), (6, 70001, 4)])
def test_infinite_and_bad_values(cuda, rows, vocab, top):
    """A student entry of -inf has no probability; where the teacher wants it the row is infinite.  An id outside the vocabulary makes its row NaN."""
    from omnihd_amd import ops
    z, t, ids, _ = inputs(rows, vocab, top, F, F, vocab + 1)
    z[:, 1] = -math.inf
    ids[ids == 1] = 0
    check(ops, z, t, ids, 1.0)                             # masked entries
    ids[2, 0] = 1
    z = z.requires_grad_()
    loss = ops.topk_distill_loss(z, t, ids, reduction="none")
    assert math.isinf(loss[2].item()) and bool(loss[[0, 1, 3]].isfinite().all())
    grad, = torch.autograd.grad(loss.sum(), z)
    assert bool(grad.isfinite().all())
    ids[2, 0], ids[3, 1], t[4, 0] = 2 ** 31 + 5, vocab, float("nan")
    with torch.no_grad():
        z[5, vocab - 1] = float("nan")
    loss = ops.topk_distill_loss(z, t, ids, reduction="none")
    assert bool(loss[2:6].isnan().all()) and bool(loss[[0, 1]].isfinite().all())
    grad, = torch.autograd.grad(loss.sum(), z)
    assert bool(grad[[2, 3, 5]].isnan().all()) and bool(grad[[0, 1]].isfinite().all())
    assert math.isnan(ops.topk_distill_loss(z.detach(), t, ids).item())


@pytest.mark.parametrize("vocab", [9, 50, 700, 9001, 70003])
def test_far_values(cuda, vocab):
    """Logits around 3e4 and spread over hundreds: only differences count."""
    from omnihd_amd import ops
    z, t, ids, _ = inputs(8, vocab, 5, F, F, vocab, scale=30.0)
    z, t = (z * 4).round() / 4 + 30000, (t * 4).round() / 4 - 20000
    check(ops, z, t, ids, 2.0)


def test_reductions_factors_and_upstreams(cuda):
    from omnihd_amd import ops
    z, t, ids, gen = inputs(64, 500, 10, B, F, 1)
    check(ops, z, t, ids, 1.5, avg=17.0, loss_weight=2.0)
    check(ops, z, t, ids, 1.5, avg=torch.tensor([17.0], device="cuda"), loss_weight=2.0)
    check(ops, z, t, ids, 1.5, reduction="sum")
    for value in (3.0, 0.1, 0.0, -1.0):
        check(ops, z, t, ids, up=torch.tensor(value, device="cuda"))


def test_second_backward_keeps_the_first(cuda):
    """The first backward's tensor is its caller's: a second one, of another upstream, does not write to it."""
    from omnihd_amd import ops
    z, t, ids, _ = inputs(30, 900, 10, F, F, 2)
    z.requires_grad_()
    loss = ops.topk_distill_loss(z, t, ids)
    first, = torch.autograd.grad(loss, z, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, z, torch.tensor(2.0, device="cuda"), retain_graph=True)
    assert torch.equal(first, kept) and torch.equal(second, 2 * kept)
    (loss * 2).backward()
    assert torch.equal(z.grad, 2 * kept) and torch.equal(first, kept)
    one, two = ops.topk_distill_loss(z, t, ids), ops.topk_distill_loss(z * 1.0, t, ids)    # two at once
    total, = torch.autograd.grad(one + 3 * two, z)
    # q - p cancels at the teacher's entries: what 1 and 3 times it are off by is relative to q + p, as for any gradient here
    _, _, dz, dz_terms = reference(z, t, ids, 1.0, None, 4 / 30)
    check_close(total, dz, bound(dz, F, dz_terms, ROUNDINGS), "total")


def test_shapes_strides_and_no_rows(cuda):
    from omnihd_amd import ops
    z, t, ids, _ = inputs(60, 77, 6, B, F, 3)
    flat = ops.topk_distill_loss(z, t, ids, reduction="none")
    assert torch.equal(ops.topk_distill_loss(z.view(3, 4, 5, 77), t.view(3, 4, 5, 6), ids.view(3, 4, 5, 6), reduction="none"), flat.view(3, 4, 5))
    assert ops.topk_distill_loss(z[0], t[0], ids[0]).shape == () and torch.equal(ops.topk_distill_loss(z[0], t[0], ids[0]), flat[0])
    for vocab, pitch, offset in ((77, 80, 0), (77, 93, 3), (80, 81, 1), (12, 20, 0), (12, 13, 1), (3000, 3008, 8), (3001, 3003, 1)):
        z, t, ids, gen = inputs(40, vocab, 6, B, F, vocab)
        wide = torch.zeros(40 * pitch + offset, dtype=B, device="cuda")[offset:].view(40, pitch)
        wide[:, :vocab] = z
        wide[:, vocab:] = 99
        view = wide[:, :vocab].detach().requires_grad_()
        tw, iw = torch.zeros(40, 9, device="cuda")[:, 1:7], torch.zeros(40, 8, dtype=ids.dtype, device="cuda")[:, 2:8]
        tw.copy_(t), iw.copy_(ids)
        got = ops.topk_distill_loss(view, tw, iw)
        grad, = torch.autograd.grad(got, view)
        # which lane adds which entry goes by the row's address: the same bounds as for dense rows, not the same bits
        rows, row_terms, dz, dz_terms = reference(z, t, ids, 1.0, None, 1 / 40)
        check_close(got, rows.sum(), bound(rows.sum(), F, row_terms.sum(), ROUNDINGS + 40), "loss")
        check_close(grad, dz, bound(dz, B, dz_terms, ROUNDINGS), "gradient")
        assert grad.shape == (40, vocab) and bool((wide[:, vocab:] == 99).all())
    z = torch.zeros(0, 50, device="cuda").requires_grad_()
    empty = (torch.zeros(0, 4, device="cuda"), torch.zeros(0, 4, dtype=torch.int64, device="cuda"))
    loss = ops.topk_distill_loss(z, *empty)
    assert loss.item() == 0 and torch.autograd.grad(loss, z)[0].shape == (0, 50)
    assert ops.topk_distill_loss(z, *empty, reduction="none").shape == (0,)


def test_more_rows_than_places(cuda):
    """Blocks that walk over several rows, in each form."""
    from omnihd_amd import ops
    for rows, vocab, top in ((600000, 5, 2), (70000, 40, 3), (9000, 600, 5), (2600, 5000, 5), (700, 20000, 5), (600, 70000, 3)):
        z, t, ids, _ = inputs(rows, vocab, top, B, F, rows)
        z = z.requires_grad_()
        loss = ops.topk_distill_loss(z, t, ids, reduction="none")
        grad, = torch.autograd.grad(loss.sum(), z)
        pick = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:400]
        want, terms, dz, dz_terms = reference(z.detach()[pick.cuda()], t[pick.cuda()], ids[pick.cuda()], 1.0, None, 1.0)
        check_close(loss[pick.cuda()], want, bound(want, F, terms, ROUNDINGS), "row losses")
        check_close(grad[pick.cuda()], dz, bound(dz, B, dz_terms, ROUNDINGS), "gradient")
        total = ops.topk_distill_loss(z.detach(), t, ids, reduction="sum")
        assert abs(total.item() - loss.double().sum().item()) <= rows * 2.0 ** -24 * loss.double().abs().sum().item()


def test_stream_and_graph(cuda):
    """Captured as a whole, and the backward alone: every replay follows the contents, the upstream's too."""
    from omnihd_amd import ops
    z, t, ids, gen = inputs(50, 3000, 12, F, F, 4)
    z.requires_grad_()
    up = torch.ones((), device="cuda")

    def step():
        loss = ops.topk_distill_loss(z, t, ids, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, z, up)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_g, grad_g = step()
    for k, value in enumerate((1.0, 0.25, 1.0, 3.0)):
        with torch.no_grad():
            z.copy_(torch.randn(z.shape, generator=gen).cuda())
        up.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        loss, grad = step()
        assert torch.equal(loss, loss_g) and torch.equal(grad, grad_g), k


def test_second_derivatives_are_refused(cuda):
    from omnihd_amd import ops
    z, t, ids, _ = inputs(5, 40, 3, F, F, 1)
    z.requires_grad_()
    w = torch.ones(40, device="cuda").requires_grad_()
    for value in (ops.topk_distill_loss(z, t, ids), ops.block_norm(z, w).sum(), ops.block_join(z, z, next_weight=w)[1].sum(), ops.token_embedding(ids, z).sum()):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(value, z, create_graph=True)


def test_backward_captured_alone(cuda):
    """An eager forward, its backward in a graph: every replay gives the gradient for what the upstream holds then, 1 among it."""
    from omnihd_amd import ops
    for vocab in (12, 700, 9000):
        z, t, ids, _ = inputs(40, vocab, 6, F, F, vocab)
        z.requires_grad_()
        up = torch.ones((), device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            loss = ops.topk_distill_loss(z, t, ids)
            torch.autograd.grad(ops.topk_distill_loss(z, t, ids), z, up)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            grad, = torch.autograd.grad(loss, z, up, retain_graph=True)
        _, _, dz, dz_terms = reference(z, t, ids, 1.0, None, 1 / 40)
        for value in (2.0, 1.0, -3.0, 1.0):
            up.fill_(value)
            graph.replay()
            torch.cuda.synchronize()
            check_close(grad, value * dz, bound(value * dz, F, abs(value) * dz_terms, ROUNDINGS), (vocab, value))


@pytest.mark.parametrize("vocab,top", [(9, 3), (30, 200), (50, 70), (300, 70), (1500, 130), (3000, 256), (6000, 256), (15000, 64), (30000, 65), (60000, 256), (120001, 200), (140000, 256)])
def test_ids_that_stand_in_a_row_many_times(cuda, vocab, top):
    """All slots the same, pairs side by side, pairs far apart, halves empty: an entry's gradient takes the sum of its slots."""
    from omnihd_amd import ops
    z, t, ids, _ = inputs(6, vocab, top, F, F, vocab + top)
    k = torch.arange(top, device="cuda")
    ids[0] = vocab - 1
    ids[1] = (k // 2) % vocab
    ids[2] = (k % max(1, top // 2)) % vocab
    ids[3] = torch.where(k < top // 2, torch.full_like(k, 2), torch.full_like(k, -1))
    ids[4] = torch.where(k % 3 == 0, torch.full_like(k, -7), (k * 5) % vocab)
    for reduction in ("sum", "none"):
        check(ops, z, t, ids, 2.0, reduction=reduction)
    check(ops, z.bfloat16(), t, ids.int(), 2.0)


@pytest.mark.parametrize("vocab,top,temperature", [(12, 4, 1.0), (40, 6, 2.0), (3000, 20, 1.0)])
def test_differences(cuda, vocab, top, temperature):
    """Directional derivatives by central differences.  In T^2 * ln sum exp(z / T) the third derivative along a unit-normal way is under 3 / T in
    mean, so a step s is off by s^2 / 6 * 3 a row; the losses' rounding by 2^-24 * loss / s.  At s = 1e-2 both are under 1e-4 a row, of
    products q * way whose absolute values sum to 0.5 and more."""
    from omnihd_amd import ops
    z, t, ids, gen = inputs(6, vocab, top, F, F, vocab)
    z.requires_grad_()
    way = torch.randn(z.shape, generator=gen).cuda()
    value = lambda v: ops.topk_distill_loss(v, t, ids, temperature=temperature, reduction="none").double()
    grad, = torch.autograd.grad(ops.topk_distill_loss(z, t, ids, temperature=temperature, reduction="sum"), z)
    with torch.no_grad():
        quotient = (value(z + 1e-2 * way) - value(z - 1e-2 * way)) / 2e-2
    assert bool(((quotient - (grad.double() * way).sum(1)).abs() <= 2e-3).all())


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 logits: the last rows are what they are alone."""
    from omnihd_amd import ops
    vocab = 131072
    rows = 2 ** 31 // vocab + 30
    z = torch.zeros(rows, vocab, dtype=B, device="cuda")
    gen = torch.Generator().manual_seed(3)
    z[-40:] = torch.randn(40, vocab, generator=gen).bfloat16().cuda()
    t, ids = torch.randn(rows, 5, generator=gen).cuda(), torch.randint(0, vocab, (rows, 5), generator=gen).cuda()
    small = z[-40:].clone().requires_grad_()
    loss_s = ops.topk_distill_loss(small, t[-40:], ids[-40:], reduction="none")
    grad_s, = torch.autograd.grad(loss_s.sum(), small)
    z.requires_grad_()
    loss = ops.topk_distill_loss(z, t, ids, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), z)
    assert torch.equal(loss[-40:], loss_s) and torch.equal(grad[-40:], grad_s)
    assert torch.allclose(grad[5].float().sum().cpu(), torch.zeros(()), atol=vocab * 2.0 ** -8 / vocab)      # q sums to 1 as p does, each rounded once
