"""What the tests of the token operators share.

Tolerances count roundings.  One rounding of a value v to a type is off by at most half_step(type) * |v| (plus half of the smallest
subnormal).  An output computed in fp32 from exact inputs is off by at most `roundings` * 2^-24 * (the same formula with every term
replaced by its absolute value), `roundings` being the longest chain from an input to the output; then it is rounded once to its type."""
import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bound(want, dtype, terms=None, roundings=0):
    """Allowed distance from `want` (fp64): `roundings` fp32 roundings of `terms` and one rounding to `dtype`."""
    inner = torch.zeros_like(want) if terms is None else roundings * F32 * terms
    return inner + half_step(dtype) * (want.abs() + inner) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check_close(got, want, allowed, what):
    got = got.detach().double().cpu()
    want, allowed = want.detach().cpu(), allowed.detach().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~((off <= allowed) | (got == want))
    if bad.any():
        i = int((off / allowed.clamp_min(1e-300)).where(bad, torch.zeros_like(off)).reshape(-1).nan_to_num(1e300).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst at {i}: got {got.reshape(-1)[i]:.9g}, "
                             f"want {want.reshape(-1)[i]:.9g}, allowed {allowed.reshape(-1)[i]:.3g}")
