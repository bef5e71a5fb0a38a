"""The naive sync BatchNorm's fp32 rows on the host (omnihd_amd/mm/sync_bn.py): batch statistics in fp64.

Everything between the fp32 inputs and the fp32 results is done in fp64 (2^-53), so outputs, gradients and running statistics are the
formula's in fp64 after one rounding to fp32, 2^-24 of themselves; the weights' gradients are sums of fp64 values, rounded once as well.  The fp64
reference differs from the module's own fp64 by a few 2^-53 of its terms: 2^-40 of the largest term is allowed for that."""
import pytest
import torch
from torch import nn

STEP, INNER = 2.0 ** -24, 2.0 ** -40


def close(got, want, terms):
    assert got.dtype == torch.float32
    assert bool(((got.detach().double() - want).abs() <= STEP * want.abs() + INNER * terms + 2.0 ** -149).all())


def pair(cls, n, c, seed, **kw):
    gen = torch.Generator().manual_seed(seed)
    bn = cls(c, eps=1e-3, **kw).train()
    with torch.no_grad():
        if bn.affine:
            bn.weight.copy_(1 + 0.3 * torch.randn(c, generator=gen))
            bn.bias.copy_(torch.randn(c, generator=gen))
        bn.running_mean.copy_(torch.randn(c, generator=gen))
        bn.running_var.copy_(1 + torch.rand(c, generator=gen))
    x = 3 * torch.randn(n, c, generator=gen) + torch.randn(c, generator=gen)
    return bn, x, torch.randn(n, c, generator=gen)


@pytest.mark.parametrize("n,c,momentum", [(2, 1, 0.1), (7, 5, 0.01), (1000, 64, 0.01), (70001, 3, 1.0), (300, 33, 0.0)])
def test_rows_gradients_and_running_statistics(n, c, momentum):
    from omnihd_amd.mm.sync_bn import NaiveSyncBatchNorm1d
    bn, x, up = pair(NaiveSyncBatchNorm1d, n, c, n + c, momentum=momentum)
    old_mean, old_var = bn.running_mean.double(), bn.running_var.double()
    x.requires_grad_()
    out = bn(x)
    gx, gw, gb = torch.autograd.grad(out, (x, bn.weight, bn.bias), up)
    d, g, w = x.detach().double(), up.double(), bn.weight.detach().double()
    mean, var = d.mean(0), d.var(0, unbiased=False)
    r = torch.rsqrt(var + 1e-3)
    xh = (d - mean) * r
    close(out, xh * w + bn.bias.detach().double(), (xh * w).abs() + bn.bias.detach().double().abs() + (mean.abs() * r * w.abs()))
    a = g * w
    close(gx, r * (a - a.mean(0) - xh * (a * xh).mean(0)), r * (a.abs() + a.abs().mean(0) + xh.abs() * (a * xh).abs().mean(0)))
    close(gw, (g * xh).sum(0), (g * xh).abs().sum(0) + g.abs().sum(0) * mean.abs() * r)
    close(gb, g.sum(0), g.abs().sum(0))
    close(bn.running_mean, (1 - momentum) * old_mean + momentum * mean, old_mean.abs() + d.abs().mean(0))
    close(bn.running_var, (1 - momentum) * old_var + momentum * var * n / (n - 1), old_var + d.square().mean(0) * n / (n - 1))
    assert bn.num_batches_tracked.item() == 1
    bn(x)
    assert bn.num_batches_tracked.item() == 2


def test_everything_else_takes_the_plain_module():
    """Evaluation, cumulative averages, layers without weights or statistics, 3-d rows and fp64 rows: torch's own, bit for bit."""
    from omnihd_amd.mm.sync_bn import NaiveSyncBatchNorm1d
    for kind, kw in (("eval", {}), ("cumulative", dict(momentum=None)), ("bare", dict(affine=False)), ("three", {}), ("double", {})):
        got, want = (pair(cls, 40, 6, 3, **kw) for cls in (NaiveSyncBatchNorm1d, nn.BatchNorm1d))
        results = []
        for bn, x, _ in (got, want):
            if kind == "eval":
                bn.eval()
            if kind == "three":
                x = x.view(10, 6, 4)
            if kind == "double":
                bn, x = bn.double(), x.double()
            results.append((bn(x), bn.running_mean, bn.running_var, bn.num_batches_tracked))
        for a, b in zip(*results):
            assert torch.equal(a, b), kind
    got, want = (cls(6, track_running_stats=False).train() for cls in (NaiveSyncBatchNorm1d, nn.BatchNorm1d))
    x = pair(nn.BatchNorm1d, 40, 6, 3)[1]
    assert torch.equal(got(x), want(x)) and got.running_mean is None
